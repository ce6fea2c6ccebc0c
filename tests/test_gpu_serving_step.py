"""The packed-batch calls together as a serving step uses them: one archive that appends a ragged
batch's K and V to the block-scaled cache, attends over it and over the prompt itself, applies the
requests' rules and picks, run over a prompt, a second chunk and captured decode steps."""
import numpy as np
import pytest

import torch

from conftest import from_dev, to_dev
from hologram_amd import DTYPE_BF16, HipSession
from packed_reference import attend, block_append, bound, decode, encode, process_logits
from test_packed_batch import serving_graph

pytestmark = pytest.mark.gpu

H, KV, D, BUCKET, BLOCK, COLS, HIST, B = 8, 2, 64, 160, 32, 700, 24, 3
DT = DTYPE_BF16


def inputs(rng, rows, pos):
    tokens = sum(rows)
    x = dict(qkv=encode(rng.standard_normal((tokens, (H + 2 * KV) * D)), DT),
             starts=np.concatenate([[0], np.cumsum(rows)]).astype(np.uint32),
             pos=np.array(pos, np.uint32), lens=np.array([p + n for p, n in zip(pos, rows)], np.uint32),
             logits=encode(rng.standard_normal((B, COLS)) * 4, DT),
             history=rng.integers(0, COLS, (B, HIST)).astype(np.int32),
             spans=np.array([[4, 9], [0, 24], [24, 24]], np.uint32),
             params=rng.uniform(1.0, 1.5, (B, 3)).astype(np.float32))
    x["history"][:, ::2] = np.argmax(decode(x["logits"], DT).reshape(B, COLS), 1)[:, None]
    return x


def check(out, x, rows, cache):
    tokens = sum(rows)
    qkv = decode(x["qkv"], DT).reshape(tokens, H + 2 * KV, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
    want = {n: block_append(cache[n], cache[n + "s"], new, rows, x["pos"].tolist(), BLOCK)
            for n, new in (("k", k), ("v", v))}
    for i, n in enumerate("kv"):
        assert np.array_equal(out[i].view(np.int8).reshape(want[n][0].shape), want[n][0])
        assert np.array_equal(out[2 + i].view(np.float32).reshape(want[n][1].shape), want[n][1])
        cache[n], cache[n + "s"] = want[n]
    at = 0
    got, prompt = (decode(o.view(np.uint16), DT).reshape(tokens, H, D) for o in (out[4], out[6]))
    for b, n in enumerate(rows):
        length = int(x["lens"][b])
        of = np.arange(length) // BLOCK
        kk, vv = ((want[c][0][b, :, :length] * want[c][1][b][:, of, None].astype(np.float64)).transpose(1, 0, 2)
                  for c in "kv")
        w, slack, top = attend(q[at:at + n], kk, vv, length - n + 1 + np.arange(n), H, KV, 8.0)
        assert (np.abs(got[at:at + n] - w) <= bound(slack, top, DT)).all()
        w, slack, top = attend(q[at:at + n], k[at:at + n], v[at:at + n], 1 + np.arange(n), H, KV, 8.0)
        assert (np.abs(prompt[at:at + n] - w) <= bound(slack, top, DT)).all()
        at += n
    ruled = process_logits(decode(x["logits"], DT).reshape(B, COLS), x["history"], x["spans"], x["params"],
                           None, None, None)
    ruled = decode(encode(ruled, DT), DT).reshape(B, COLS)
    picks = out[5].view(np.int32)
    # (the f32 value next to a bf16 step may round to either side: within a step of the largest)
    assert (ruled[np.arange(B), picks] >= ruled.max(1) - 2.0 ** -7 * np.abs(ruled.max(1))).all()


def test_prompt_chunk_and_captured_decode(torch_cuda, backend):
    rng = np.random.default_rng(11)
    nb = -(-BUCKET // BLOCK)
    cache = {n: np.zeros((B, KV, BUCKET, D), np.int8) for n in "kv"}
    cache.update({n + "s": np.zeros((B, KV, nb), np.float32) for n in "kv"})
    dev = [to_dev(torch, cache[n]) for n in ("k", "v", "ks", "vs")]      # one cache for all sessions
    pos = [0, 0, 0]

    def session(rows):
        return HipSession(backend, serving_graph(sum(rows), B, H, KV, D, BUCKET, BLOCK, COLS, HIST, DT))

    def bind(s, x):
        held = [to_dev(torch, x[n]) for n in ("qkv", "starts", "pos", "lens")] + dev
        held += [to_dev(torch, x[n]) for n in ("logits", "history", "spans", "params")]
        for i, t in enumerate(held):
            s.bind_input(i, t)
        return held

    for rows in ([40, 1, 90], [7, 33, 2]):
        s = session(rows)
        x = inputs(rng, rows, pos)
        held = bind(s, x)
        torch.cuda.synchronize()
        s.run()
        s.synchronize()
        check([np.frombuffer(s.read_output(i), np.uint8) for i in range(7)], x, rows, cache)
        pos = [p + n for p, n in zip(pos, rows)]
        s.close()
        del held

    s = session([1] * B)
    names = ("qkv", "starts", "pos", "lens", "k", "v", "ks", "vs", "logits", "history", "spans", "params")
    x = inputs(rng, [1] * B, pos)
    held = dict(zip(names, bind(s, x)))
    torch.cuda.synchronize()
    for step in range(5):
        if step == 0:
            s.capture()                  # runs the step, then records it
        else:
            x = inputs(rng, [1] * B, pos)
            for n in names[:4] + names[8:]:
                held[n].copy_(to_dev(torch, x[n]))
            torch.cuda.synchronize()
            s.replay()
        s.synchronize()
        check([np.frombuffer(s.read_output(i), np.uint8) for i in range(7)], x, [1] * B, cache)
        pos = [p + 1 for p in pos]
    assert np.array_equal(from_dev(dev[0], np.int8).reshape(cache["k"].shape), cache["k"])
    s.close()
