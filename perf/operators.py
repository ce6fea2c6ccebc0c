"""The packed-batch serving operators as cases that can be timed and checked.

A packed batch lays the rows of its sequences end to end, `starts[b]` the first row of sequence b
and `starts[batch]` one past the last. Four operators serve it:

  packed   causal attention of whole prompts of different lengths over their own K and V
  append   new K (or V) rows quantized to 8 bits and appended to a cache that holds one scale for
           each block of rows of a sequence and head
  blocks   attention of new rows (one a sequence in decode, many in a prompt's later chunk) over
           that cache
  logits   repetition, frequency and presence penalties, biases and a grammar's mask on logits

`run` computes a case in elementary torch operations where `own` is false, and through the
backend's kernel calls where it is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


def listed():
    return [
        # the smallest prompt pass: a few short questions at once, where latency counts
        dict(name="packed_small", kind="packed", dtype="bf16", batch=4, shortest=1, longest=61,
             heads=32, kv_heads=8, head_dim=64, fused=False),
        # a serving batch of ragged prompts, q, k and v left in one projection's output
        dict(name="packed_ragged", kind="packed", dtype="f16", batch=24, shortest=17, longest=2000,
             heads=32, kv_heads=8, head_dim=128, fused=True),
        # long documents
        dict(name="packed_long", kind="packed", dtype="bf16", batch=3, shortest=4096, longest=16384,
             heads=32, kv_heads=8, head_dim=128, fused=False),
        # an f32 graph's prompts, a head size between the powers of two
        dict(name="packed_f32", kind="packed", dtype="f32", batch=5, shortest=33, longest=1000,
             heads=8, kv_heads=2, head_dim=96, fused=False),
        # one decoded token for each of 32 sequences joins the cache
        dict(name="append_decode", kind="append", dtype="bf16", batch=32, shortest=1, longest=1,
             past=250, kv_heads=8, head_dim=128, bucket=256, block=32),
        # the prompts of 16 sequences join it, most of them starting inside a block
        dict(name="append_prompt", kind="append", dtype="bf16", batch=16, shortest=100,
             longest=1500, past=500, kv_heads=8, head_dim=128, bucket=2048, block=64),
        # decode over short contexts, where latency counts
        dict(name="blocks_small", kind="blocks", dtype="f16", batch=8, shortest=1, longest=1,
             past_short=30, past_long=700, heads=32, kv_heads=8, head_dim=64, bucket=1024, block=16),
        # serving decode: a ragged batch of long contexts, one token each
        dict(name="blocks_decode", kind="blocks", dtype="bf16", batch=32, shortest=1, longest=1,
             past_short=512, past_long=32767, heads=32, kv_heads=8, head_dim=128, bucket=32768,
             block=32),
        # the next chunk of four prompts, over what the cache holds of them
        dict(name="blocks_chunk", kind="blocks", dtype="bf16", batch=4, shortest=301, longest=1024,
             past_short=1, past_long=6000, heads=32, kv_heads=8, head_dim=128, bucket=8192,
             block=64),
        # a chat's next token: one row, a short history
        dict(name="logits_one", kind="logits", dtype="f32", rows=1, cols=32000, history=1024,
             biases=8, mask=False),
        # a batch of structured generations: every row with a grammar's mask and a long history
        dict(name="logits_batch", kind="logits", dtype="bf16", rows=128, cols=128000, history=4096,
             biases=64, mask=True),
    ]


# ------------------------------------------------------------------ draws ----
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 8]), kv


def _draw_packed(rng):
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    heads, kv = _heads(rng)
    longest = _log(rng, 1, 1500 if dtype == "f32" else 6000)
    return dict(kind="packed", dtype=dtype, batch=_log(rng, 1, 16),
                shortest=_log(rng, 1, longest), longest=longest, heads=heads, kv_heads=kv,
                head_dim=rng.choice([64, 128, 128, 80, 96, 256]), fused=rng.random() < 0.4)


def _draw_append(rng):
    longest = rng.choice([1, 1, _log(rng, 2, 1500)])
    past = rng.choice([0, _log(rng, 1, 500)])
    return dict(kind="append", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                batch=_log(rng, 1, 32), shortest=_log(rng, 1, longest), longest=longest, past=past,
                kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 96, 128, 128]),
                bucket=max(256, -(-(longest + past) // 256) * 256),
                block=rng.choice([16, 32, 64, 128]))


def _draw_blocks(rng):
    heads, kv = _heads(rng)
    decode = rng.random() < 0.5
    longest = rng.choice([1, 1, 2, 4]) if decode else _log(rng, 2, 700)
    past = _log(rng, 1, 16000 if decode else 4000)
    return dict(kind="blocks", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                batch=_log(rng, 1, 32 if decode else 4), shortest=_log(rng, 1, longest),
                longest=longest, past_short=_log(rng, 1, past), past_long=past, heads=heads,
                kv_heads=kv, head_dim=rng.choice([64, 128, 128, 96, 256]),
                bucket=-(-(longest + past) // 256) * 256, block=rng.choice([16, 32, 64, 128]))


def _draw_logits(rng):
    return dict(kind="logits", dtype=rng.choice(["bf16", "f32", "f16"]), rows=_log(rng, 1, 96),
                cols=_log(rng, 500, 128000), history=_log(rng, 16, 8192),
                biases=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.5)


def draw(rng):
    return rng.choice([_draw_packed, _draw_packed, _draw_append, _draw_blocks, _draw_blocks,
                       _draw_logits])(rng)


# ---------------------------------------------------------------- lengths ----
def _spread(n, lo, hi):
    """n lengths from lo to hi, even over their logarithm, in a mixed order."""
    if n == 1:
        return [hi]
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    geo = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    return [geo[(i * step + n // 2) % n] for i in range(n)]


def _rows(c):
    return _spread(c["batch"], c["shortest"], c["longest"])


def _past(c):
    if c["kind"] == "append":     # any whole number up to `past`, off the blocks' ends
        return [(37 * i + c["past"]) % (c["past"] + 1) for i in range(c["batch"])]
    return _spread(c["batch"], c["past_short"], c["past_long"])[::-1]


def _starts(rows):
    out = [0]
    for n in rows:
        out.append(out[-1] + n)
    return out


# ----------------------------------------------------------------- inputs ----
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _u32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(g, planes, bucket, d, block):
    """int8 rows of N(0, 1) and each block's power-of-two scale."""
    q = torch.empty((planes, bucket, d), dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // (bucket * d))
    for p in range(0, planes, step):
        x = torch.randn((min(step, planes - p), bucket, d), generator=g, device="cuda")
        q[p:p + step] = (x * 36.0).round_().clamp_(-127, 127).to(torch.int8)
    nb = -(-bucket // block)
    e = torch.randint(-6, -3, (planes, nb), generator=g, device="cuda")
    return q, torch.exp2(e.float())


def _packed_state(c, g):
    rows, d, dt = _rows(c), c["head_dim"], DTYPES[c["dtype"]]
    tokens, h, kv = sum(rows), c["heads"], c["kv_heads"]
    st = {"rows": rows, "starts": _u32(_starts(rows))}
    if c["fused"]:
        st["qkv"] = _randn(g, (tokens, (h + 2 * kv) * d), dt)
        st["q"], st["k"], st["v"] = st["qkv"].split([h * d, kv * d, kv * d], dim=1)
    else:
        st["q"] = _randn(g, (tokens, h * d), dt)
        st["k"] = _randn(g, (tokens, kv * d), dt)
        st["v"] = _randn(g, (tokens, kv * d), dt)
    return st


def _append_state(c, g):
    rows, past, d = _rows(c), _past(c), c["head_dim"]
    planes = c["batch"] * c["kv_heads"]
    # K rows as a model makes them: a few channels much larger than the rest
    x = torch.randn((sum(rows), c["kv_heads"] * d), generator=g, device="cuda")
    big = torch.rand(c["kv_heads"] * d, generator=g, device="cuda") < 0.02
    new = (x * torch.where(big, 20.0, 1.0)).to(DTYPES[c["dtype"]])
    cache, scales = _cache(g, planes, c["bucket"], d, c["block"])
    return {"rows": rows, "past": past, "starts": _u32(_starts(rows)), "pos": _u32(past),
            "new": new, "cache": cache, "scales": scales}


def _blocks_state(c, g):
    rows, past, d = _rows(c), _past(c), c["head_dim"]
    planes = c["batch"] * c["kv_heads"]
    kq, ks = _cache(g, planes, c["bucket"], d, c["block"])
    vq, vs = _cache(g, planes, c["bucket"], d, c["block"])
    lens = [p + n for p, n in zip(past, rows)]
    return {"rows": rows, "len": lens, "starts": _u32(_starts(rows)), "lens": _u32(lens),
            "q": _randn(g, (sum(rows), c["heads"] * d), DTYPES[c["dtype"]]),
            "kq": kq, "ks": ks, "vq": vq, "vs": vs}


def _logits_state(c, g):
    rows, cols, hist, nb = c["rows"], c["cols"], c["history"], c["biases"]
    ri = lambda lo, hi, shape: torch.randint(lo, hi, shape, generator=g, device="cuda",  # noqa: E731
                                             dtype=torch.int32)
    # histories in which some tokens come back often, of different lengths
    history = torch.minimum(ri(0, cols, (rows, hist)), ri(0, cols, (rows, hist)))
    history[:, ::5] = history[:, :1]
    lens = ri(hist // 2, hist + 1, (rows,))
    prompt = (lens.float() * torch.rand(rows, generator=g, device="cuda")).int()
    u = torch.rand((rows, 3), generator=g, device="cuda")
    params = torch.stack([1.0 + 0.5 * u[:, 0], u[:, 1], u[:, 2]], dim=1).contiguous()
    st = {"logits": _randn(g, (rows, cols), DTYPES[c["dtype"]], 4.0), "history": history,
          "spans": torch.stack([prompt, lens], dim=1).contiguous(), "params": params,
          "ids": None, "values": None, "mask": None}
    if nb:      # distinct tokens a row
        st["ids"] = torch.stack([torch.randperm(cols, generator=g, device="cuda")[:nb]
                                 for _ in range(rows)]).int().contiguous()
        st["values"] = _randn(g, (rows, nb), torch.float32, 3.0)
    if c["mask"]:
        words = ri(-2**31, 2**31 - 1, (rows, -(-cols // 32)))
        st["mask"] = words & ri(-2**31, 2**31 - 1, words.shape)
    return st


def prepare(case, seed):
    g = _gen(seed)
    st = {"packed": _packed_state, "append": _append_state, "blocks": _blocks_state,
          "logits": _logits_state}[case["kind"]](case, g)
    st["case"] = case
    if own:
        _bind(st)
    return st


# --------------------------------------------------- the framework's calls ----
def _bind(st):
    """The backend, the bound slots and the calls that a serving program keeps."""
    from hologram_amd import BufferRef, DeviceWorkspace, HipBackend, KernelCall
    from hologram_amd import kernel_call as kc
    c = st["case"]
    dt = {"bf16": kc.DTYPE_BF16, "f16": kc.DTYPE_F16, "f32": kc.DTYPE_F32}[c["dtype"]]
    be = HipBackend(0, torch.cuda.current_stream().cuda_stream)
    ws, calls, refs = DeviceWorkspace(), [], []

    def slot(t):
        if t is None:
            return kc.NO_BUFFER
        refs.append(t)
        ws.bind(len(refs) - 1, t)
        return BufferRef(len(refs) - 1)

    if c["kind"] == "packed":
        h, kv, d, tokens = c["heads"], c["kv_heads"], c["head_dim"], sum(st["rows"])
        st["out"] = torch.empty((tokens, h * d), dtype=DTYPES[c["dtype"]], device="cuda")
        if c["fused"]:
            s, es = slot(st["qkv"]).slot, SIZES[c["dtype"]]
            q, k, v = (BufferRef(s, es * d * at) for at in (0, h, h + kv))
            stride = (h + 2 * kv) * d
            strides = (stride, stride, stride)
        else:
            q, k, v = slot(st["q"]), slot(st["k"]), slot(st["v"])
            strides = (0, 0, 0)
        calls.append(KernelCall.AttentionPacked(kc.AttentionPackedCall(
            q, k, v, slot(st["starts"]), slot(st["out"]), tokens, c["batch"], h, kv, d, *strides,
            0, dt)))
    elif c["kind"] == "append":
        planes, d = c["batch"] * c["kv_heads"], c["head_dim"]
        cache, scales = slot(st["cache"]), slot(st["scales"])
        calls.append(KernelCall.KvBlockAppend(kc.KvBlockAppendCall(
            slot(st["new"]), slot(st["starts"]), slot(st["pos"]), cache, scales, cache, scales,
            sum(st["rows"]), c["batch"], c["kv_heads"], c["bucket"], c["block"], d, 0, dt)))
        # the values that the cache stands for: every one an exact bf16
        st["zeros"] = torch.zeros(st["scales"].numel(), dtype=torch.int32, device="cuda")
        st["values"] = torch.empty(st["cache"].shape, dtype=torch.bfloat16, device="cuda")
        calls.append(KernelCall.Dequantize(kc.DequantizeCall(
            cache, scales, slot(st["zeros"]), slot(st["values"]), planes * c["bucket"] * d,
            st["scales"].numel(), c["block"] * d, kc.DTYPE_I8, kc.DTYPE_BF16)))
    elif c["kind"] == "blocks":
        h, kv, d, tokens = c["heads"], c["kv_heads"], c["head_dim"], sum(st["rows"])
        st["out"] = torch.empty((tokens, h * d), dtype=DTYPES[c["dtype"]], device="cuda")
        calls.append(KernelCall.AttentionI8Blocks(kc.AttentionI8BlocksCall(
            slot(st["q"]), slot(st["kq"]), slot(st["vq"]), slot(st["ks"]), slot(st["vs"]),
            slot(st["starts"]), slot(st["lens"]), slot(st["out"]), tokens, c["batch"], h, kv,
            c["bucket"], c["block"], d, 0, 0, dt)))
    else:
        st["out"] = torch.empty_like(st["logits"])
        calls.append(KernelCall.LogitsProcess(kc.LogitsProcessCall(
            slot(st["logits"]), slot(st["history"]), slot(st["spans"]), slot(st["params"]),
            slot(st["ids"]), slot(st["values"]), slot(st["mask"]), slot(st["out"]), c["rows"],
            c["cols"], c["history"], c["biases"], dt)))
    st["be"], st["ws"], st["calls"] = be, ws, calls


def _run_own(st):
    for call in st["calls"]:
        st["be"].dispatch(call, st["ws"])
    if st["case"]["kind"] == "append":
        return st["values"], st["scales"]
    return st["out"]


# ------------------------------------------------------------- plain forms ----
def _plain_attend(q, k, v, n, past, heads, kv):
    """q [n, heads * d] over k, v [kv, past + n, d], all f32; row i sees past + i + 1 keys."""
    d, g, total = k.shape[-1], heads // kv, past + n
    q = q.view(n, kv, g, d).permute(1, 2, 0, 3).reshape(kv, g * n, d)
    kt = k.transpose(1, 2).contiguous()
    out = torch.empty((kv, g * n, d), device=q.device)
    j, i = torch.arange(total, device=q.device), torch.arange(n, device=q.device).repeat(g)
    for h in range(kv):           # one kv head at a time: the scores of a long prompt are large
        s = (q[h] @ kt[h]) * (1.0 / math.sqrt(d))
        s.masked_fill_(j > (past + i)[:, None], -math.inf)
        s -= s.amax(dim=-1, keepdim=True)
        p = s.exp_()
        out[h] = (p @ v[h]) / p.sum(dim=-1, keepdim=True)
    return out.view(kv, g, n, d).permute(2, 0, 1, 3).reshape(n, heads * d)


def _plain_packed(st):
    c = st["case"]
    d, kv, at = c["head_dim"], c["kv_heads"], 0
    out = torch.empty((sum(st["rows"]), c["heads"] * d), dtype=DTYPES[c["dtype"]], device="cuda")
    for n in st["rows"]:
        q, k, v = (st[x][at:at + n].float() for x in "qkv")
        k, v = (x.reshape(n, kv, d).transpose(0, 1).contiguous() for x in (k, v))
        out[at:at + n] = _plain_attend(q.contiguous(), k, v, n, 0, c["heads"], kv).to(out.dtype)
        at += n
    return out


def _plain_blocks(st):
    c = st["case"]
    d, kv, t, at = c["head_dim"], c["kv_heads"], c["block"], 0
    out = torch.empty((sum(st["rows"]), c["heads"] * d), dtype=DTYPES[c["dtype"]], device="cuda")
    for b, (n, total) in enumerate(zip(st["rows"], st["len"])):
        plane, nb = slice(b * kv, (b + 1) * kv), -(-total // t)
        k, v = (st[x][plane, :total].float()
                * st[s][plane, :nb].repeat_interleave(t, dim=1)[:, :total, None]
                for x, s in (("kq", "ks"), ("vq", "vs")))
        q = st["q"][at:at + n].float()
        out[at:at + n] = _plain_attend(q, k, v, n, total - n, c["heads"], kv).to(out.dtype)
        at += n
    return out


def _plain_append(st):
    """A block's scale is the least power of two 2^e with max|x| <= 127 * 2^e over its new rows,
    and not below the scale of the rows it holds already; those are rounded anew where it grew."""
    c = st["case"]
    kv, d, t, bucket, batch = c["kv_heads"], c["head_dim"], c["block"], c["bucket"], c["batch"]
    nb = bucket // t
    starts, pos = st["starts"].long(), st["pos"].long()
    new = st["new"].float().view(-1, kv, d)
    tok = torch.arange(new.shape[0], device="cuda")
    seq = torch.searchsorted(starts, tok, right=True) - 1
    at = pos[seq] + tok - starts[seq]                       # the row each token takes
    f, e = torch.frexp(new.abs().amax(dim=-1))
    need = torch.exp2((torch.where(f <= 127.0 / 128.0, e - 7, e - 6)).clamp_min(-126).float())
    need = torch.where(f == 0, 0.0, need)                   # [tokens, kv]
    plane = seq[:, None] * kv + torch.arange(kv, device="cuda")
    scales, cache = st["scales"].view(-1), st["cache"]
    block = plane * nb + (at // t)[:, None]
    grown = torch.zeros(batch * kv * nb, device="cuda")
    grown.scatter_reduce_(0, block.view(-1), need.view(-1), "amax")
    touched = torch.zeros(batch * kv * nb, dtype=torch.bool, device="cuda")
    touched[block.view(-1)] = True
    # the block a sequence's first new row falls into keeps the rows before it
    n = starts[1:] - starts[:-1]
    has = ((pos % t != 0) & (n > 0)).repeat_interleave(kv)
    p = torch.arange(batch * kv, device="cuda")
    first = p * nb + (pos // t).clamp_max(nb - 1).repeat_interleave(kv)
    held = torch.where(has, scales[first], torch.zeros_like(scales[first]))
    grown.scatter_reduce_(0, first, held, "amax")
    r = torch.arange(t, device="cuda")
    old_row = ((pos // t) * t).repeat_interleave(kv)[:, None] + r
    keep = has[:, None] & (old_row < pos.repeat_interleave(kv)[:, None])
    old_row = old_row.clamp_max(bucket - 1)
    rows = cache[p[:, None], old_row]
    ratio = torch.where(held > 0, held / grown[first], torch.zeros_like(held))
    again = torch.round(rows.float() * ratio[:, None, None]).to(torch.int8)
    cache[p[:, None], old_row] = torch.where(keep[..., None], again, rows)
    st["scales"].view(-1)[touched] = grown[touched]
    inv = torch.where(grown[block] > 0, 1.0 / grown[block], torch.zeros_like(grown[block]))
    cache[plane, at[:, None]] = torch.round(new * inv[..., None]).to(torch.int8)
    values = cache.view(-1, t, d).float() * st["scales"].view(-1, 1, 1)
    return values.to(torch.bfloat16).view(cache.shape), st["scales"]


def _plain_logits(st):
    c = st["case"]
    rows, cols = c["rows"], c["cols"]
    x = st["logits"].float()
    prompt, length = st["spans"][:, :1], st["spans"][:, 1:]
    j = torch.arange(c["history"], device="cuda")
    ids = st["history"].long()
    count = torch.zeros((rows, cols), device="cuda")
    count.scatter_add_(1, ids, ((j >= prompt) & (j < length)).float())
    seen = torch.zeros((rows, cols), device="cuda")
    seen.scatter_add_(1, ids, (j < length).float())
    rep, freq, pres = (st["params"][:, i:i + 1] for i in range(3))
    x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, x - freq * count - pres, x)
    if st["ids"] is not None:
        x.scatter_add_(1, st["ids"].long(), st["values"])
    if st["mask"] is not None:
        bit = (st["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x = torch.where(bit.view(rows, -1)[:, :cols] == 1, x, -math.inf)
    return x.to(DTYPES[c["dtype"]])


def run(state):
    if own:
        return _run_own(state)
    return {"packed": _plain_packed, "append": _plain_append, "blocks": _plain_blocks,
            "logits": _plain_logits}[state["case"]["kind"]](state)


# ------------------------------------------------------------------- work ----
def _pairs(rows, past):
    return sum(n * p + n * (n + 1) // 2 for n, p in zip(rows, past))


def work(case):
    c, es = case, SIZES[case["dtype"]]
    if c["kind"] == "logits":
        n = c["rows"] * c["cols"]
        aux = c["rows"] * (c["history"] * 4 + c["biases"] * 8 + 20)
        mask = c["rows"] * -(-c["cols"] // 32) * 4 if c["mask"] else 0
        return {"bytes": 2 * n * es + aux + mask, "flops": n}
    rows, d, kv = _rows(c), c["head_dim"], c["kv_heads"]
    tokens = sum(rows)
    if c["kind"] == "append":
        # the new rows in, their int8 out, and the cache's values read and written once
        held = c["batch"] * kv * c["bucket"] * d
        return {"bytes": tokens * kv * d * (es + 1) + held * 3, "flops": tokens * kv * d * 3 + held}
    h = c["heads"]
    if c["kind"] == "packed":
        return {"bytes": tokens * (2 * h + 2 * kv) * d * es,
                "flops": 4 * h * d * _pairs(rows, [0] * len(rows))}
    past = _past(c)
    keys = sum(n + p for n, p in zip(rows, past))
    blocks = sum(-(-(n + p) // c["block"]) for n, p in zip(rows, past))
    return {"bytes": tokens * 2 * h * d * es + kv * (keys * 2 * d + blocks * 8),
            "flops": 4 * h * d * _pairs(rows, past)}


# ------------------------------------------------------------------ exact ----
def _exact_attention(q, k, v, first):
    """One query head, 64 bits: q [n, d] over k, v [m, d], row i over the first + i + 1 keys."""
    n, m = q.shape[0], k.shape[0]
    out = torch.empty((n, v.shape[1]), dtype=torch.float64, device=q.device)
    kt = k.t().contiguous()
    for r in range(0, n, 2048):
        e = min(n, r + 2048)
        s = torch.mm(q[r:e], kt) / math.sqrt(q.shape[1])
        row = torch.arange(r, e, device=q.device)
        s[torch.arange(m, device=q.device)[None, :] >= first + 1 + row[:, None]] = -math.inf
        out[r:e] = torch.mm(torch.softmax(s, dim=1), v)
    return out


def exact(case, seed):
    c = case
    if work(c)["flops"] > 1.5e13:
        return None
    st = {"packed": _packed_state, "append": _append_state, "blocks": _blocks_state,
          "logits": _logits_state}[c["kind"]](c, _gen(seed))
    if c["kind"] == "packed":
        d, g, parts, at = c["head_dim"], c["heads"] // c["kv_heads"], [], 0
        for n in st["rows"]:
            head = lambda x, i: x[at:at + n, i * d:(i + 1) * d].double()  # noqa: E731,B023
            parts.append(torch.cat([_exact_attention(head(st["q"], h), head(st["k"], h // g),
                                                     head(st["v"], h // g), 0)
                                    for h in range(c["heads"])], dim=1))
            at += n
        return torch.cat(parts)
    if c["kind"] == "blocks":
        d, kv, t, parts, at = c["head_dim"], c["kv_heads"], c["block"], [], 0
        for b, (n, total) in enumerate(zip(st["rows"], st["len"])):
            heads = []
            for h in range(c["heads"]):
                p = b * kv + h // (c["heads"] // kv)
                of = torch.arange(total, device="cuda") // t
                k = st["kq"][p, :total].double() * st["ks"][p].double()[of][:, None]
                v = st["vq"][p, :total].double() * st["vs"][p].double()[of][:, None]
                q = st["q"][at:at + n, h * d:(h + 1) * d].double()
                heads.append(_exact_attention(q, k, v, total - n))
            parts.append(torch.cat(heads, dim=1))
            at += n
        return torch.cat(parts)
    if c["kind"] == "append":
        return _exact_append(c, st)
    return _exact_logits(c, st)


def _exact_append(c, st):
    """Block by block: powers of two make every quotient exact, so 64 bits give the same integers
    as any width that holds the inputs."""
    kv, d, t = c["kv_heads"], c["head_dim"], c["block"]
    cache = st["cache"].double().view(c["batch"], kv, -1, t, d)
    scales = st["scales"].double().view(c["batch"], kv, -1).clone()
    at = 0
    for b, (n, p) in enumerate(zip(st["rows"], st["past"])):
        new = st["new"][at:at + n].double().view(n, kv, d).transpose(0, 1)
        at += n
        for j in range(p // t, (p + n - 1) // t + 1):
            lo, hi = max(p, j * t), min(p + n, (j + 1) * t)
            x = new[:, lo - p:hi - p]
            top = x.abs().amax(dim=(1, 2))
            s = torch.exp2(torch.ceil(torch.log2(top / 127.0)))
            s = torch.where(top > 127.0 * s, 2.0 * s, torch.where(top <= 63.5 * s, 0.5 * s, s))
            s = torch.where(top == 0, torch.zeros_like(s), s.clamp_min(2.0 ** -126))
            if lo > j * t:
                before = scales[b, :, j].clone()
                s = torch.maximum(s, before)
                back = torch.where(s > 0, before / s, s)[:, None, None]
                held = cache[b, :, j, :lo - j * t]
                cache[b, :, j, :lo - j * t] = torch.round(held * back)
            scales[b, :, j] = s
            div = torch.where(s > 0, s, torch.ones_like(s))[:, None, None]
            cache[b, :, j, lo - j * t:hi - j * t] = torch.round(x / div)
    return (cache * scales[..., None, None]).view(st["cache"].shape), scales.view(st["scales"].shape)


def _exact_logits(c, st):
    out = st["logits"].double()
    for r in range(c["rows"]):
        prompt, length = st["spans"][r].tolist()
        ids = st["history"][r, :length].long()
        rep, freq, pres = st["params"][r].double()
        said = torch.unique(ids)
        x = out[r, said]
        out[r, said] = torch.where(x > 0, x / rep, x * rep)
        made, times = torch.unique(ids[prompt:], return_counts=True)
        out[r, made] = out[r, made] - (freq * times.double() + pres)
        if st["ids"] is not None:
            ids = st["ids"][r].long()
            out[r, ids] = out[r, ids] + st["values"][r].double()
        if st["mask"] is not None:
            words = st["mask"][r].long() & 0xFFFFFFFF
            allowed = (words[:, None] >> torch.arange(32, device="cuda")) & 1
            out[r, allowed.view(-1)[:c["cols"]] == 0] = -math.inf
    return out
