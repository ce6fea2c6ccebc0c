"""Long-context serving of a packed batch as cases that can be timed and checked.

A packed batch lays the rows of its sequences end to end, `starts[b]` the first row of sequence b
and `starts[batch]` one past the last; `pos[b]` is the position of its first row, `lens[b]` the
keys that its last row sees. Four operators take a step of it from the projections to the attention
over a long int8 cache:

  rotary    each head of q and k normed and rotated by its row's position
  bounds    each cache block's smallest and largest K bytes, brought up to date behind an append
  select    each row's blocks, by the largest score that a block's bounds allow
  selected  attention of each row over the blocks of its list

`run` computes a case in elementary torch operations where `own` is false, and through the
backend's kernel calls where it is true.
"""
import math
import struct

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
EPSILON = 1e-6


def listed():
    return [
        # the next token of 32 chats: one row each, where latency counts
        dict(name="rotary_decode", kind="rotary", dtype="bf16", batch=32, shortest=1, longest=1,
             past_short=10, past_long=32000, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, norms=3, scaled=False, fused=True),
        # ragged prompts left in one projection's output, half of each head rotated, no norms
        dict(name="rotary_prompt", kind="rotary", dtype="f16", batch=16, shortest=100, longest=1500,
             past_short=0, past_long=0, heads=32, kv_heads=8, head_dim=128, rotary_dim=64,
             interleaved=True, norms=0, scaled=False, fused=True),
        # chunks of long documents, far positions under frequencies scaled for them
        dict(name="rotary_far", kind="rotary", dtype="bf16", batch=4, shortest=2048, longest=16384,
             past_short=4096, past_long=900000, heads=32, kv_heads=8, head_dim=128, rotary_dim=128,
             interleaved=False, norms=3, scaled=True, fused=False),
        # one decoded token for each of 32 sequences has joined the cache
        dict(name="bounds_decode", kind="bounds", batch=32, shortest=1, longest=1, past_short=20,
             past_long=4000, kv_heads=8, head_dim=128, bucket=4096, block=32),
        # prompts have joined it, most of them starting inside a block
        dict(name="bounds_prompt", kind="bounds", batch=16, shortest=100, longest=8000,
             past_short=3, past_long=500, kv_heads=8, head_dim=128, bucket=8704, block=64),
        # decode over contexts that are just past the list, where latency counts
        dict(name="select_small", kind="select", dtype="f16", batch=8, shortest=1, longest=1,
             past_short=200, past_long=2000, heads=32, kv_heads=8, head_dim=64, bucket=2048,
             block=16, top=16),
        # serving decode over a ragged batch of long contexts
        dict(name="select_decode", kind="select", dtype="bf16", batch=32, shortest=1, longest=1,
             past_short=2048, past_long=65535, heads=32, kv_heads=8, head_dim=128, bucket=65536,
             block=32, top=64),
        # the next chunk of four prompts, every row with a list of its own
        dict(name="select_chunk", kind="select", dtype="bf16", batch=4, shortest=301, longest=1024,
             past_short=2000, past_long=30000, heads=32, kv_heads=8, head_dim=128, bucket=32768,
             block=64, top=32),
        # the attention of such a short decode step
        dict(name="selected_small", kind="selected", dtype="f16", batch=8, shortest=1, longest=1,
             past_short=200, past_long=2000, heads=32, kv_heads=8, head_dim=64, bucket=2048,
             block=16, top=16),
        # and of serving decode: 2048 keys of each of 32 long contexts
        dict(name="selected_decode", kind="selected", dtype="bf16", batch=32, shortest=1, longest=1,
             past_short=2048, past_long=32767, heads=32, kv_heads=8, head_dim=128, bucket=32768,
             block=64, top=32),
        # drafts of a few tokens, f32 rows, a head size between the powers of two
        dict(name="selected_draft", kind="selected", dtype="f32", batch=8, shortest=2, longest=5,
             past_short=1000, past_long=16000, heads=16, kv_heads=4, head_dim=96, bucket=16384,
             block=32, top=40),
        # a prompt's next chunk
        dict(name="selected_chunk", kind="selected", dtype="bf16", batch=2, shortest=200,
             longest=512, past_short=8000, past_long=30000, heads=32, kv_heads=8, head_dim=128,
             bucket=32768, block=64, top=32),
    ]


# ------------------------------------------------------------------ draws ----
def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8])
    return kv * rng.choice([1, 2, 3, 4, 8]), kv


def _draw_rotary(rng):
    heads, kv = _heads(rng)
    d = rng.choice([64, 128, 128, 80, 96, 256])
    longest = rng.choice([1, _log(rng, 2, 6000), _log(rng, 2, 6000)])
    past = rng.choice([0, _log(rng, 1, 1000000)])
    return dict(kind="rotary", dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                batch=_log(rng, 1, 32 if longest == 1 else 8), shortest=_log(rng, 1, longest),
                longest=longest, past_short=past and _log(rng, 1, past), past_long=past,
                heads=heads, kv_heads=kv, head_dim=d, rotary_dim=rng.choice([d, d, d // 2]),
                interleaved=rng.random() < 0.5, norms=rng.choice([0, 1, 3, 3]),
                scaled=rng.random() < 0.5, fused=rng.random() < 0.5)


def _draw_bounds(rng):
    longest = rng.choice([1, 1, _log(rng, 2, 4000)])
    past = rng.choice([0, _log(rng, 1, 2000)])
    return dict(kind="bounds", batch=_log(rng, 1, 32 if longest == 1 else 16),
                shortest=_log(rng, 1, longest), longest=longest,
                past_short=past and _log(rng, 1, past), past_long=past,
                kv_heads=rng.choice([1, 2, 4, 8]), head_dim=rng.choice([64, 96, 128, 128]),
                bucket=max(256, -(-(longest + past) // 256) * 256),
                block=rng.choice([16, 32, 64, 128]))


def _draw_lists(rng, kind):
    heads, kv = _heads(rng)
    decode, block, top = rng.random() < 0.6, rng.choice([16, 32, 64, 128]), _log(rng, 4, 40)
    longest = rng.choice([1, 1, 2, 4]) if decode else _log(rng, 2, 300)
    # one sequence at least is past what its list holds
    past = _log(rng, 2 * top * block, max(32000 if decode else 8000, 4 * top * block))
    return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                batch=_log(rng, 1, 32 if decode else 2), shortest=_log(rng, 1, longest),
                longest=longest, past_short=_log(rng, 1, past), past_long=past, heads=heads,
                kv_heads=kv, head_dim=rng.choice([64, 128, 128, 96, 256]),
                bucket=-(-(longest + past) // 256) * 256, block=block, top=top)


def draw(rng):
    costs = [work(c) for c in listed()]
    while True:
        case = rng.choice([_draw_rotary, _draw_rotary, _draw_bounds,
                           lambda r: _draw_lists(r, "select"), lambda r: _draw_lists(r, "select"),
                           lambda r: _draw_lists(r, "selected"),
                           lambda r: _draw_lists(r, "selected")])(rng)
        if all(work(case)[x] <= max(w[x] for w in costs) for x in ("bytes", "flops")):
            return case


# ---------------------------------------------------------------- lengths ----
def _spread(n, lo, hi):
    """n lengths from lo to hi, even over their logarithm, in a mixed order."""
    if n == 1 or lo == hi:
        return [hi] * n
    step = next(s for s in (7, 5, 3, 1) if math.gcd(s, n) == 1)
    geo = [int(round(lo * (hi / lo) ** (i / (n - 1)))) for i in range(n)]
    return [geo[(i * step + n // 2) % n] for i in range(n)]


def _rows(c):
    return _spread(c["batch"], c["shortest"], c["longest"])


def _past(c):
    return _spread(c["batch"], c["past_short"], c["past_long"])[::-1]


def _starts(rows):
    out = [0]
    for n in rows:
        out.append(out[-1] + n)
    return out


def _visible(c):
    """The keys that each row sees, sequence by sequence."""
    return [[p + t + 1 for t in range(n)] for n, p in zip(_rows(c), _past(c))]


# ----------------------------------------------------------------- inputs ----
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _u32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _scales(g, shape):
    return torch.exp2(torch.randint(-6, -3, shape, generator=g, device="cuda").float())


def _bytes(g, planes, bucket, d):
    """int8 cache rows of N(0, 1)."""
    q = torch.empty((planes, bucket, d), dtype=torch.int8, device="cuda")
    step = max(1, (1 << 27) // (bucket * d))
    for p in range(0, planes, step):
        x = torch.randn((min(step, planes - p), bucket, d), generator=g, device="cuda")
        q[p:p + step] = (x * 36.0).round_().clamp_(-127, 127).to(torch.int8)
    return q


def _frequencies(c):
    """Radians a position. Scaled for long contexts: those that turn less than once in the trained
    length slow down by a factor, those that turn often stay, the ones between in proportion."""
    half = c["rotary_dim"] // 2
    base = 500000.0 if c["scaled"] else 10000.0
    out = []
    for i in range(half):
        f = base ** (-i / half)
        if c["scaled"]:
            turns = 8192 * f / (2 * math.pi)
            keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            f = f * keep + f / 8.0 * (1.0 - keep)
        out.append(f)
    return torch.tensor(out, dtype=torch.float64).float().cuda()


def _rotary_state(c, g):
    rows, past, d, dt = _rows(c), _past(c), c["head_dim"], DTYPES[c["dtype"]]
    tokens, h, kv = sum(rows), c["heads"], c["kv_heads"]
    st = {"rows": rows, "past": past, "starts": _u32(_starts(rows)), "pos": _u32(past),
          "freqs": _frequencies(c), "gamma_q": None, "gamma_k": None}
    if c["fused"]:
        st["qkv"] = _randn(g, (tokens, (h + 2 * kv) * d), dt)
        st["q"], st["k"], _ = st["qkv"].split([h * d, kv * d, kv * d], dim=1)
    else:
        st["q"] = _randn(g, (tokens, h * d), dt)
        st["k"] = _randn(g, (tokens, kv * d), dt)
    for bit, name in ((1, "gamma_q"), (2, "gamma_k")):
        if c["norms"] & bit:
            st[name] = (1.0 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt)
    return st


def _bounds_state(c, g):
    rows, past, d = _rows(c), _past(c), c["head_dim"]
    planes, nb = c["batch"] * c["kv_heads"], -(-c["bucket"] // c["block"])
    lo = -torch.randint(40, 128, (planes, nb, 1, d), generator=g, device="cuda")
    hi = torch.randint(40, 128, (planes, nb, 1, d), generator=g, device="cuda")
    return {"rows": rows, "past": past, "starts": _u32(_starts(rows)), "pos": _u32(past),
            "cache": _bytes(g, planes, c["bucket"], d), "scales": _scales(g, (planes, nb)),
            "bounds": torch.cat([lo, hi], dim=2).to(torch.int8)}


def _row_state(c, g):
    rows, past = _rows(c), _past(c)
    lens = [p + n for p, n in zip(past, rows)]
    return {"rows": rows, "len": lens, "starts": _u32(_starts(rows)), "lens": _u32(lens),
            "q": _randn(g, (sum(rows), c["heads"] * c["head_dim"]), DTYPES[c["dtype"]])}


def _select_state(c, g):
    st, d = _row_state(c, g), c["head_dim"]
    planes, nb = c["batch"] * c["kv_heads"], -(-c["bucket"] // c["block"])
    # what rows of N(0, 1) leave: bounds of two to three deviations, a few channels wider
    x = torch.randn((2, planes, nb, d), generator=g, device="cuda") * 14.0 + 80.0
    x = x.round_().clamp_(0, 127)
    st["bounds"] = torch.stack([-x[0], x[1]], dim=2).to(torch.int8)
    st["scales"] = _scales(g, (planes, nb)) * torch.exp2(
        -torch.rand((planes, nb), generator=g, device="cuda"))
    return st


def _selected_state(c, g):
    st, d, t, top = _row_state(c, g), c["head_dim"], c["block"], c["top"]
    planes, nb = c["batch"] * c["kv_heads"], -(-c["bucket"] // t)
    for x in "kv":
        st[x + "q"] = _bytes(g, planes, c["bucket"], d)
        st[x + "s"] = _scales(g, (planes, nb))
    # a row's list: its first and last blocks and a random choice between, ascending, -1 behind
    seen = torch.tensor([-(-v // t) for rows in _visible(c) for v in rows], device="cuda")
    u = torch.rand((seen.numel(), c["kv_heads"], nb), generator=g, device="cuda")
    j = torch.arange(nb, device="cuda")
    last = seen[:, None, None] - 1
    u = torch.where((j == 0) | (j == last), 2.0, torch.where(j < last, u, -1.0))
    best = u.topk(min(top, nb), dim=-1)
    ids = torch.where(best.values >= 0, best.indices, nb).sort(dim=-1).values
    ids = torch.where(ids < nb, ids, -1).int()
    pad = torch.full((*ids.shape[:2], top - ids.shape[2]), -1, dtype=torch.int32, device="cuda")
    st["blocks"] = torch.cat([ids, pad], dim=-1).contiguous()
    return st


MAKERS = {"rotary": _rotary_state, "bounds": _bounds_state, "select": _select_state,
          "selected": _selected_state}


def prepare(case, seed):
    st = MAKERS[case["kind"]](case, _gen(seed))
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
    d, kv, tokens = c["head_dim"], c["kv_heads"], sum(st["rows"])
    dt = {"bf16": kc.DTYPE_BF16, "f16": kc.DTYPE_F16, "f32": kc.DTYPE_F32}.get(c.get("dtype"))
    be = HipBackend(0, torch.cuda.current_stream().cuda_stream)
    ws, calls, refs = DeviceWorkspace(), [], []

    def slot(t):
        if t is None:
            return kc.NO_BUFFER
        refs.append(t)
        ws.bind(len(refs) - 1, t)
        return BufferRef(len(refs) - 1)

    if c["kind"] == "rotary":
        h = c["heads"]
        st["q_out"] = torch.empty((tokens, h * d), dtype=DTYPES[c["dtype"]], device="cuda")
        st["k_out"] = torch.empty((tokens, kv * d), dtype=DTYPES[c["dtype"]], device="cuda")
        if c["fused"]:
            s, stride = slot(st["qkv"]).slot, (h + 2 * kv) * d
            q, k = BufferRef(s), BufferRef(s, SIZES[c["dtype"]] * h * d)
        else:
            q, k, stride = slot(st["q"]), slot(st["k"]), 0
        calls.append(KernelCall.QkNormRotary(kc.QkNormRotaryCall(
            q, k, slot(st["gamma_q"]), slot(st["gamma_k"]), slot(st["starts"]), slot(st["pos"]),
            slot(st["freqs"]), slot(st["q_out"]), slot(st["k_out"]), tokens, c["batch"], h, kv, d,
            c["rotary_dim"], stride, stride, struct.unpack("<I", struct.pack("<f", EPSILON))[0], 0,
            c["norms"], int(c["interleaved"]), dt)))
    elif c["kind"] == "bounds":
        bounds, planes = slot(st["bounds"]), c["batch"] * kv
        calls.append(KernelCall.KvBlockBounds(kc.KvBlockBoundsCall(
            slot(st["cache"]), slot(st["starts"]), slot(st["pos"]), bounds, bounds, tokens,
            c["batch"], kv, c["bucket"], c["block"], d)))
        # the values that the bounds stand for: every one an exact bf16
        nb = st["scales"].shape[1]
        st["zeros"] = torch.zeros(planes * nb, dtype=torch.int32, device="cuda")
        st["values"] = torch.empty(st["bounds"].shape, dtype=torch.bfloat16, device="cuda")
        calls.append(KernelCall.Dequantize(kc.DequantizeCall(
            bounds, slot(st["scales"]), slot(st["zeros"]), slot(st["values"]),
            planes * nb * 2 * d, planes * nb, 2 * d, kc.DTYPE_I8, kc.DTYPE_BF16)))
    elif c["kind"] == "select":
        st["out"] = torch.empty((tokens, kv, c["top"]), dtype=torch.int32, device="cuda")
        calls.append(KernelCall.KvBlockSelect(kc.KvBlockSelectCall(
            slot(st["q"]), slot(st["bounds"]), slot(st["scales"]), slot(st["starts"]),
            slot(st["lens"]), slot(st["out"]), tokens, c["batch"], c["heads"], kv, c["bucket"],
            c["block"], d, 0, c["top"], 1, 2, dt)))
    else:
        st["out"] = torch.empty((tokens, c["heads"] * d), dtype=DTYPES[c["dtype"]], device="cuda")
        calls.append(KernelCall.AttentionI8Selected(kc.AttentionI8SelectedCall(
            slot(st["q"]), slot(st["kq"]), slot(st["vq"]), slot(st["ks"]), slot(st["vs"]),
            slot(st["blocks"]), slot(st["starts"]), slot(st["lens"]), slot(st["out"]), tokens,
            c["batch"], c["heads"], kv, c["bucket"], c["block"], d, 0, c["top"], 0, dt)))
    st["be"], st["ws"], st["calls"] = be, ws, calls


def _run_own(st):
    for call in st["calls"]:
        st["be"].dispatch(call, st["ws"])
    kind = st["case"]["kind"]
    if kind == "rotary":
        return st["q_out"], st["k_out"]
    return st["values"] if kind == "bounds" else st["out"]


# ------------------------------------------------------------- plain forms ----
def _plain_rotary(st):
    c = st["case"]
    d, rot, tokens = c["head_dim"], c["rotary_dim"], sum(st["rows"])
    starts = st["starts"].long()
    tok = torch.arange(tokens, device="cuda")
    seq = torch.searchsorted(starts, tok, right=True) - 1
    at = st["pos"].long()[seq] + tok - starts[seq]
    angle = at.double()[:, None] * st["freqs"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    out = []
    for x, gamma in ((st["q"], st["gamma_q"]), (st["k"], st["gamma_k"])):
        x = x.float().reshape(tokens, -1, d)
        if gamma is not None:
            x = x * (1.0 / (x.square().mean(dim=-1, keepdim=True) + EPSILON).sqrt()) * gamma.float()
        if c["interleaved"]:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        out.append(torch.cat([turned, x[..., rot:]], dim=-1).to(DTYPES[c["dtype"]]).view(tokens, -1))
    return tuple(out)


def _plain_bounds(st):
    c = st["case"]
    kv, t, bounds = c["kv_heads"], c["block"], st["bounds"]
    for b, (n, p) in enumerate(zip(st["rows"], st["past"])):
        end, j0 = p + n, p // t
        j1 = -(-end // t)
        x = st["cache"][b * kv:(b + 1) * kv, j0 * t:j1 * t].float()
        x = x.reshape(kv, j1 - j0, t, -1)
        there = torch.arange(j0 * t, j1 * t, device="cuda").view(j1 - j0, t, 1) < end
        bounds[b * kv:(b + 1) * kv, j0:j1, 0] = x.masked_fill(~there, 127).amin(dim=2).to(torch.int8)
        bounds[b * kv:(b + 1) * kv, j0:j1, 1] = x.masked_fill(~there, -128).amax(dim=2).to(torch.int8)
    return (bounds.float() * st["scales"][:, :, None, None]).to(torch.bfloat16)


def _plain_select(st):
    """The first block, the last two that a row sees, and between them those with the largest
    bound of the scores' sum over the heads, q as 8-bit integers. Whole numbers times a scale:
    64 bits hold every score exactly."""
    c = st["case"]
    d, kv, t, top = c["head_dim"], c["kv_heads"], c["block"], c["top"]
    out = torch.full((sum(st["rows"]), kv, top), -1, dtype=torch.int32, device="cuda")
    q = st["q"].float().view(-1, kv, c["heads"] // kv, d)
    f, e = torch.frexp(q.abs().amax(dim=(2, 3), keepdim=True))
    e = torch.where(f <= 127.0 / 128.0, e - 7, e - 6).clamp_min(-126)
    q = torch.round(torch.ldexp(q, -e))
    up, down = (x.sum(dim=2).double() for x in (q.clamp_min(0), q.clamp_max(0)))  # [tokens, kv, d]
    at = 0
    for b, (n, total) in enumerate(zip(st["rows"], st["len"])):
        nb = -(-total // t)
        lo, hi = st["bounds"][b * kv:(b + 1) * kv, :nb].double().permute(2, 0, 3, 1).contiguous()
        score = (torch.bmm(up[at:at + n].transpose(0, 1).contiguous(), hi)
                 + torch.bmm(down[at:at + n].transpose(0, 1).contiguous(), lo))
        score = score * st["scales"][b * kv:(b + 1) * kv, None, :nb].double()  # [kv, n, nb]
        seen = torch.arange(total - n + 1, total + 1, device="cuda")[:, None].add(t - 1) // t
        j = torch.arange(nb, device="cuda")
        score = torch.where((j < 1) | (j >= seen - 2), math.inf, score)
        score = torch.where(j < seen, score, -math.inf)
        order = score.sort(dim=-1, descending=True, stable=True).indices[..., :top]
        ids = torch.where(order < seen, order, nb).sort(dim=-1).values
        ids = torch.where(ids < nb, ids, -1).transpose(0, 1).int()
        out[at:at + n, :, :ids.shape[-1]] = ids
        at += n
    return out


def _plain_selected(st):
    c = st["case"]
    d, kv, t, g = c["head_dim"], c["kv_heads"], c["block"], c["heads"] // c["kv_heads"]
    tokens = sum(st["rows"])
    out = torch.empty((tokens, kv, g, d), dtype=DTYPES[c["dtype"]], device="cuda")
    q = st["q"].float().view(tokens, kv, g, d)
    sees = torch.tensor([v for rows in _visible(c) for v in rows], device="cuda")
    seq = torch.tensor([b for b, n in enumerate(st["rows"]) for _ in range(n)], device="cuda")
    inner = torch.arange(t, device="cuda")
    step = max(1, (1 << 28) // (c["top"] * t * d))
    for h in range(kv):
        for a in range(0, tokens, step):
            e = min(tokens, a + step)
            ids = st["blocks"][a:e, h].long()                       # [rows, top]
            key = (ids.clamp_min(0)[:, :, None] * t + inner).flatten(1)
            there = ((ids >= 0)[:, :, None].expand(-1, -1, t).flatten(1)) & (key < sees[a:e, None])
            key = key.clamp_max(c["bucket"] - 1)
            plane = (seq[a:e] * kv + h)[:, None]
            s = st["ks"][plane, key // t]
            s = (q[a:e, h] @ st["kq"][plane, key].float().transpose(1, 2).contiguous()) * s[:, None]
            s = (s * (1.0 / math.sqrt(d))).masked_fill_(~there[:, None], -math.inf)
            s -= s.amax(dim=-1, keepdim=True)
            p = s.exp_()
            v = st["vq"][plane, key].float() * st["vs"][plane, key // t][..., None]
            out[a:e, h] = ((p @ v) / p.sum(dim=-1, keepdim=True)).to(out.dtype)
    return out.view(tokens, -1)


PLAIN = {"rotary": _plain_rotary, "bounds": _plain_bounds, "select": _plain_select,
         "selected": _plain_selected}


def run(state):
    return _run_own(state) if own else PLAIN[state["case"]["kind"]](state)


# ------------------------------------------------------------------- work ----
def work(case):
    c = case
    rows, past, d, kv = _rows(c), _past(c), c["head_dim"], c["kv_heads"]
    tokens = sum(rows)
    if c["kind"] == "rotary":
        n = tokens * (c["heads"] + kv) * d
        return {"bytes": 2 * n * SIZES[c["dtype"]] + c["rotary_dim"] * 2, "flops": 6 * n}
    t = c["block"]
    if c["kind"] == "bounds":
        # the touched blocks' rows, and the bounds read and their values written once
        held = sum((p + n - p // t * t) for n, p in zip(rows, past)) * kv * d
        all_bounds = c["batch"] * kv * -(-c["bucket"] // t) * 2 * d
        return {"bytes": held + all_bounds * 3, "flops": 2 * held + all_bounds}
    es, h = SIZES[c["dtype"]], c["heads"]
    if c["kind"] == "select":
        blocks = sum(-(-(n + p) // t) for n, p in zip(rows, past))
        pairs = sum(-(-v // t) for seq in _visible(c) for v in seq)
        return {"bytes": tokens * (h * d * es + kv * c["top"] * 4) + blocks * kv * (2 * d + 4),
                "flops": pairs * kv * 4 * d}
    listed_keys = [[min(v, c["top"] * t) for v in seq] for seq in _visible(c)]
    once = sum(min(sum(k), n + p) for k, n, p in zip(listed_keys, rows, past))
    return {"bytes": tokens * (2 * h * d * es + kv * c["top"] * 4) + kv * once * (2 * d) +
            kv * once // t * 8,
            "flops": 4 * h * d * sum(map(sum, listed_keys))}


# ------------------------------------------------------------------ exact ----
def _exact_rotary(c, st):
    d, rot, parts = c["head_dim"], c["rotary_dim"], []
    at = torch.cat([torch.arange(p, p + n, device="cuda") for n, p in zip(st["rows"], st["past"])])
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       at.double()[:, None] * st["freqs"].double())
    for x, gamma in ((st["q"], st["gamma_q"]), (st["k"], st["gamma_k"])):
        y = torch.empty(x.shape, dtype=torch.float64, device="cuda")
        for h in range(x.shape[1] // d):
            v = x[:, h * d:(h + 1) * d].double()
            if gamma is not None:
                v = v / torch.sqrt(torch.sum(v * v, dim=1, keepdim=True) / d + EPSILON)
                v = v * gamma.double()
            pairs = (v[:, :rot].reshape(-1, rot // 2, 2) if c["interleaved"] else
                     v[:, :rot].reshape(-1, 2, rot // 2).transpose(1, 2)).contiguous()
            z = torch.view_as_real(torch.view_as_complex(pairs) * turn)
            y[:, h * d:h * d + rot] = (z if c["interleaved"] else z.transpose(1, 2)).reshape(-1, rot)
            y[:, h * d + rot:(h + 1) * d] = v[:, rot:]
        parts.append(y)
    return tuple(parts)


def _exact_bounds(c, st):
    kv, t = c["kv_heads"], c["block"]
    out = st["bounds"].double()
    for b, (n, p) in enumerate(zip(st["rows"], st["past"])):
        plane = slice(b * kv, (b + 1) * kv)
        for j in range(p // t, (p + n - 1) // t + 1):
            x = st["cache"][plane, j * t:min((j + 1) * t, p + n)]
            out[plane, j, 0], out[plane, j, 1] = (f(x, dim=1).double() for f in (torch.amin, torch.amax))
    return out * st["scales"].double()[:, :, None, None]


def _exact_select(c, st):
    """Row by row and head by head from the definition; whole numbers, so 64 bits are exact."""
    d, kv, t, top = c["head_dim"], c["kv_heads"], c["block"], c["top"]
    g, at = c["heads"] // kv, 0
    out = torch.full((sum(st["rows"]), kv, top), -1, dtype=torch.int32, device="cuda")
    for b, (n, total) in enumerate(zip(st["rows"], st["len"])):
        nb = -(-total // t)
        for h in range(kv):
            q = st["q"][at:at + n, h * g * d:(h + 1) * g * d].double()
            big = q.abs().amax(dim=1, keepdim=True)
            s = torch.exp2(torch.ceil(torch.log2(big / 127.0)))
            s = torch.where(big > 127.0 * s, 2.0 * s, torch.where(big <= 63.5 * s, 0.5 * s, s))
            q = torch.round(q / s.clamp_min(2.0 ** -126)).view(n, g, d)
            bounds = st["bounds"][b * kv + h, :nb].double()
            score = torch.zeros((n, nb), dtype=torch.float64, device="cuda")
            step = max(1, (1 << 25) // (nb * d))
            for r in range(0, n, step):
                for i in range(g):
                    x = q[r:r + step, i, None, :]
                    score[r:r + step] += torch.maximum(x * bounds[:, 0], x * bounds[:, 1]).sum(-1)
            score *= st["scales"][b * kv + h, :nb].double()
            for seen in sorted({-(-(total - n + 1 + r) // t) for r in range(n)}):
                rows = [r for r in range(n) if -(-(total - n + 1 + r) // t) == seen]
                rows = torch.tensor(rows, device="cuda")
                fixed = sorted({0, seen - 2, seen - 1} & set(range(seen)))
                free = [j for j in range(seen) if j not in fixed]
                free = torch.tensor(free, dtype=torch.long, device="cuda")
                more = max(0, min(top - len(fixed), free.numel()))
                # (a stable sort of what is negated: the largest first, of equals the lowest block)
                best = free[torch.sort(-score[rows][:, free], dim=1, stable=True).indices[:, :more]]
                keep = torch.tensor(fixed, device="cuda").expand(rows.numel(), -1)
                ids = torch.cat([best, keep], dim=1).sort(dim=1).values
                out[at + rows, h, :ids.shape[1]] = ids.int()
        at += n
    return out


def _exact_selected(c, st):
    d, kv, t, g = c["head_dim"], c["kv_heads"], c["block"], c["heads"] // c["kv_heads"]
    out = torch.empty((sum(st["rows"]), c["heads"], d), dtype=torch.float64, device="cuda")
    lists, at = st["blocks"].cpu().tolist(), 0
    for b, (n, total) in enumerate(zip(st["rows"], st["len"])):
        for h in range(kv):
            k = st["kq"][b * kv + h, :total].double()
            k *= st["ks"][b * kv + h].double().repeat_interleave(t)[:total, None]
            v = st["vq"][b * kv + h, :total].double()
            v *= st["vs"][b * kv + h].double().repeat_interleave(t)[:total, None]
            q = st["q"][at:at + n].double().view(n, c["heads"], d)[:, h * g:(h + 1) * g]
            step = max(1, (1 << 26) // (total * g))
            for r in range(0, n, step):
                e = min(n, r + step)
                take = torch.zeros((e - r, -(-total // t)), dtype=torch.bool)
                for i in range(r, e):
                    take[i - r, [j for j in lists[at + i][h] if j >= 0]] = True
                take = take.cuda().repeat_interleave(t, dim=1)[:, :total]
                last = total - n + torch.arange(r, e, device="cuda")
                take &= torch.arange(total, device="cuda") <= last[:, None]
                s = torch.mm(q[r:e].reshape(-1, d), k.t().contiguous()).view(e - r, g, total)
                s = torch.where(take[:, None], s / math.sqrt(d), -math.inf)
                p = torch.softmax(s, dim=-1).reshape(-1, total)
                out[at + r:at + e, h * g:(h + 1) * g] = torch.mm(p, v).view(e - r, g, d)
        at += n
    return out.view(out.shape[0], -1)


def exact(case, seed):
    return {"rotary": _exact_rotary, "bounds": _exact_bounds, "select": _exact_select,
            "selected": _exact_selected}[case["kind"]](case, MAKERS[case["kind"]](case, _gen(seed)))
