"""The workloads that the serving operators are measured on.

Four operators: rotary positions, a quantised key/value cache (written and
read back), attention of drafted tokens over that cache, and log
probabilities of given tokens.  ``run`` computes them in plain torch, or,
with ``own`` true, by the calls a user makes of this package.  Shapes are
those of the models the repository's benchmarks use (32 query heads over 8
key/value heads of 64 or 128, 64 over 8 of 128, a vocabulary of 128256).
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GGML = {"q8_0": 8, "q4_0": 2}


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a batch of 16 sequences, far positions under banded scaling
        dict(name="rope_step", op="rope", dtype="bf16", tokens=16, heads=32, kv_heads=8, head_dim=128, rot_dim=128,
             interleaved=False, scaling="llama3", factor=8.0, theta=500000.0, max_pos=131072, inverse=False),
        # the gradient of a training pass, q and k as views of a joint projection
        dict(name="rope_grad", op="rope", dtype="f32", tokens=4099, heads=32, kv_heads=8, head_dim=64, rot_dim=64,
             interleaved=False, scaling="none", factor=1.0, theta=10000.0, max_pos=8192, inverse=True),
        # a long prompt, interleaved pairs over half of each head
        dict(name="rope_prompt", op="rope", dtype="bf16", tokens=16384, heads=64, kv_heads=8, head_dim=128, rot_dim=64,
             interleaved=True, scaling="yarn", factor=4.0, theta=1000000.0, max_pos=65536, inverse=False),
        # one decode step of a batch: a new row of each sequence into the cache, and back
        dict(name="cache_step", op="cache", dtype="f32", cache="q8_0", seqs=40, new=1, ctx=2000, kv_heads=8,
             head_dim=64, page=32),
        # a batch of prompts into a 4-bit cache
        dict(name="cache_prompt4", op="cache", dtype="bf16", cache="q4_0", seqs=5, new=6000, ctx=0, kv_heads=8,
             head_dim=128, page=16),
        # chunked prompts behind earlier ones, 8 bits
        dict(name="cache_chunk8", op="cache", dtype="bf16", cache="q8_0", seqs=9, new=4097, ctx=5000, kv_heads=8,
             head_dim=128, page=64),
        # one sequence, one token: the latency of a decode step
        dict(name="attn_one", op="attn", dtype="f32", cache="q8_0", seqs=1, new=1, ctx=1023, heads=32, kv_heads=8,
             head_dim=64, page=64, tree=False),
        # a decode step of a batch of ragged contexts
        dict(name="attn_batch", op="attn", dtype="bf16", cache="q8_0", seqs=48, new=1, ctx=16000, heads=32, kv_heads=8,
             head_dim=128, page=32, tree=False),
        # trees of up to 64 drafted tokens verified
        dict(name="attn_tree64", op="attn", dtype="bf16", cache="q8_0", seqs=8, new=64, ctx=8190, heads=32, kv_heads=8,
             head_dim=128, page=64, tree=True),
        # small trees over long 4-bit contexts, 8 query heads to a key head
        dict(name="attn_tree13_q4", op="attn", dtype="f16", cache="q4_0", seqs=12, new=13, ctx=30011, heads=64,
             kv_heads=8, head_dim=128, page=16, tree=True),
        # one sampled token scored, with 20 alternatives
        dict(name="logprobs_one", op="logprobs", dtype="f32", rows=1, vocab=128256, tokens=1, top=20),
        # a batch of prompts scored
        dict(name="logprobs_batch", op="logprobs", dtype="bf16", rows=1031, vocab=128256, tokens=1, top=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] + w["flops"] / 100.0


def draw(rng):
    op = rng.choice(["rope", "cache", "attn", "attn", "logprobs"])
    most = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        dt = rng.choice(["f32", "f16", "bf16"])
        heads, kvh = rng.choice([(32, 8), (64, 8), (8, 8), (12, 4), (28, 4), (5, 1)])
        hd = rng.choice([64, 128])
        if op == "rope":
            c = dict(op=op, dtype=dt, tokens=_log(rng, 1, 16384), heads=heads, kv_heads=kvh, head_dim=hd,
                     rot_dim=rng.choice([hd, hd // 2, 32]), interleaved=rng.random() < 0.5,
                     scaling=rng.choice(["none", "linear", "ntk", "yarn", "llama3"]), factor=rng.choice([2.0, 4.0, 8.0]),
                     theta=rng.choice([10000.0, 500000.0]), max_pos=_log(rng, 100, 1000000), inverse=rng.random() < 0.4)
        elif op == "cache":
            c = dict(op=op, dtype=dt, cache=rng.choice(["q8_0", "q4_0"]), seqs=_log(rng, 1, 64), new=_log(rng, 1, 6000),
                     ctx=rng.choice([0, _log(rng, 1, 8000)]), kv_heads=kvh, head_dim=hd, page=rng.choice([16, 32, 64, 128]))
        elif op == "attn":
            c = dict(op=op, dtype=dt, cache=rng.choice(["q8_0", "q4_0"]), seqs=_log(rng, 1, 48),
                     new=rng.choice([1, 1, _log(rng, 2, 64)]), ctx=_log(rng, 1, 30000), heads=heads, kv_heads=kvh,
                     head_dim=hd, page=rng.choice([16, 32, 64, 128]), tree=rng.random() < 0.6)
        else:
            c = dict(op=op, dtype=dt, rows=_log(rng, 1, 1000), vocab=rng.choice([128256, 32000, _log(rng, 64, 200000)]),
                     tokens=rng.choice([1, 1, 4]), top=rng.choice([0, 1, 5, 20, 32]))
        if _cost(c) <= most:
            return c


def _lengths(case):
    """Context lengths and numbers of new tokens of the case's sequences, spread over (1/3 .. 1) of its largest."""
    n = case["seqs"]
    f = (np.arange(n) * 0.6180339887) % 1.0
    ctx = case["ctx"] - np.floor(f * case["ctx"] * 2 / 3).astype(np.int64)
    new = case["new"] - np.floor(((f * 7.0) % 1.0) * case["new"] * 2 / 3).astype(np.int64)
    ctx[0], new[0] = case["ctx"], case["new"]
    return ctx, np.maximum(new, 1)


def work(case):
    op, size = case["op"], SIZE[case["dtype"]]
    if op == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * n * case["head_dim"] * size + 4 * case["tokens"], "flops": 3 * n * case["rot_dim"]}
    if op == "logprobs":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (8 * case["tokens"] + 8 * case["top"] + 4), "flops": 5 * n}
    ctx, new = _lengths(case)
    hd, kvh = case["head_dim"], case["kv_heads"]
    row = 2 * kvh * (hd if case["cache"] == "q8_0" else hd // 2) + 2 * kvh * hd // 16  # K and V codes and scales
    if op == "cache":
        t = int(new.sum())
        return {"bytes": t * (2 * 2 * kvh * hd * size + 2 * row), "flops": t * 6 * kvh * hd}
    length, t = ctx + new, int(new.sum())
    return {"bytes": int(length.sum()) * row + 2 * t * case["heads"] * hd * size,
            "flops": int((4 * new * length).sum()) * case["heads"] * hd}


# ---------------------------------------------------------------- inputs
def _tree_mask(new, rng, words):
    """Ancestor bits of random trees, one row of 32-bit words per drafted token: bit i of row j says that j sees i."""
    rows = []
    for n in new:
        m = np.zeros((n, words * 32), np.uint8)
        for j in range(n):
            if j:
                m[j] = m[rng.randrange(max(0, j - 8), j)]
            m[j, j] = 1
        rows.append(m)
    bits = np.packbits(np.concatenate(rows).reshape(-1, words, 32), axis=-1, bitorder="little")
    return bits.view(np.uint32).reshape(-1, words).view(np.int32)


def _planes(case, pool, pages):
    """Views of the cache pool: K codes, K scales, V codes, V scales of its one layer."""
    kvh, page, hd = case["kv_heads"], case["page"], case["head_dim"]
    cb, nb = (hd if case["cache"] == "q8_0" else hd // 2), hd // 32
    codes, scales = pages * kvh * page * cb, pages * kvh * page * nb * 2
    at, out = 0, []
    for _ in range(2):
        out.append(pool[at:at + codes].view(pages, kvh, page, cb))
        at += codes
        out.append(pool[at:at + scales].view(torch.float16).view(pages, kvh, page, nb))
        at += scales
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = randn(rows, vocab, scale=3.0)
        s["tokens"] = torch.randint(0, vocab, (rows, case["tokens"]), generator=g, device="cuda", dtype=torch.int32)
        return s
    hd, kvh = case["head_dim"], case["kv_heads"]
    if case["op"] == "rope":
        t, h = case["tokens"], case["heads"]
        joint = randn(t, h + kvh, hd)  # the projection's output: q and k side by side in each row
        s["q"], s["k"] = joint[:, :h], joint[:, h:]
        s["positions"] = torch.randint(0, case["max_pos"], (t,), generator=g, device="cuda", dtype=torch.int32)
        if own:
            from m3_avm_b200.attention import Rope

            s["plan"] = Rope(hd, rot_dim=case["rot_dim"], theta=case["theta"], interleaved=case["interleaved"],
                             scaling=case["scaling"], factor=1.0 if case["scaling"] == "none" else case["factor"],
                             orig_ctx=8192)
        return s
    ctx, new = _lengths(case)
    page, n = case["page"], case["seqs"]
    need = -(-(ctx + new) // page)
    most = int(need.max())
    pages = int(need.sum()) + 3
    r = random.Random(seed)
    order = list(range(pages))
    r.shuffle(order)  # a sequence's pages lie anywhere in the pool
    table, at = np.full((n, most), -1, np.int32), 0
    for i in range(n):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
    s["table"] = torch.from_numpy(table).cuda()
    s["ctx"] = torch.from_numpy(ctx.astype(np.int32)).cuda()
    s["start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
    s["total"], s["most_new"], s["most_len"] = int(new.sum()), int(new.max()), int((ctx + new).max())
    cb, nb = (hd if case["cache"] == "q8_0" else hd // 2), hd // 32
    pool = torch.zeros(2 * pages * kvh * page * (cb + 2 * nb), dtype=torch.uint8, device="cuda")
    s["pages"], s["pool"] = pages, pool
    if case["op"] == "cache":
        joint = randn(s["total"], 2 * kvh, hd)
        s["k"], s["v"] = joint[:, :kvh], joint[:, kvh:]
    else:
        for k, plane in enumerate(_planes(case, pool, pages)):
            if k % 2:  # scales of rows of unit size
                u = torch.rand(plane.shape, generator=g, device="cuda")
                plane.copy_((2.0 + u) / (127.0 if case["cache"] == "q8_0" else 7.0))
            elif case["cache"] == "q8_0":
                for i in range(0, pages, 4096):
                    part = plane[i:i + 4096]
                    part.copy_((torch.randn(part.shape, generator=g, device="cuda") * 50.0).round_().clamp_(-127, 127) + 128)
            else:
                for i in range(0, pages, 8192):
                    part = plane[i:i + 8192]
                    lo, hi = ((torch.randn(part.shape, generator=g, device="cuda") * 2.8).round_().clamp_(-8, 7) + 8
                              for _ in range(2))
                    part.copy_(lo + 16 * hi)
        s["q"] = randn(s["total"], case["heads"], hd, scale=1.5)
        s["mask"] = None
        if case["tree"]:
            s["mask"] = torch.from_numpy(_tree_mask(new, r, -(-s["most_new"] // 32))).cuda()
    if own:
        from m3_avm_b200.attention import KvBatch, KvCache

        s["cache"] = KvCache(GGML[case["cache"]], 1, kvh, hd, page, pages, pool=pool)
        s["batch"] = KvBatch(s["start"], s["ctx"], s["table"], s["total"], s["most_new"], s["most_len"])
    return s


# ---------------------------------------------------------------- plain forms
def _frequencies(case):
    """Rotation per position of each pair, in radians (64 bits), and the factor on cos and sin."""
    d, base, factor, mag = case["rot_dim"], case["theta"], case["factor"], 1.0
    i = torch.arange(0, d, 2, dtype=torch.float64, device="cuda")
    orig = 8192
    if case["scaling"] == "ntk":
        base = base * factor ** (d / (d - 2))
    f = base ** (-i / d)
    if case["scaling"] == "linear":
        f = f / factor
    elif case["scaling"] == "yarn":
        def at(turns):
            return d * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), d - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mag = 0.1 * math.log(factor) + 1.0
    elif case["scaling"] == "llama3":
        wave = 2 * math.pi / f
        smooth = ((orig / wave - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = (1 - smooth) * f / factor + smooth * f
    return f, mag


def _plain_rope(s):
    case = s["case"]
    f, mag = _frequencies(case)
    angle = s["positions"].double()[:, None, None] * f
    c, n = (angle.cos() * mag).float(), (angle.sin() * mag).float()
    n = -n if case["inverse"] else n
    d = case["rot_dim"]

    def rotate(x):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:d:2], y[..., 1:d:2]
        else:
            a, b = y[..., :d // 2], y[..., d // 2:d]
        pair = (a * c - b * n, a * n + b * c)
        turned = torch.stack(pair, -1).flatten(-2) if case["interleaved"] else torch.cat(pair, -1)
        return torch.cat((turned, y[..., d:]), -1).to(x.dtype)

    return rotate(s["q"]), rotate(s["k"])


def _slots(s):
    """Page and place in it of every new token."""
    start, page = s["start"].long(), s["case"]["page"]
    t = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(start, t, right=True) - 1
    pos = s["ctx"].long()[seq] + t - start[seq]
    return s["table"].long()[seq, pos // page], pos % page


def _values(codes, scales, kind):
    """Values that codes (..., bytes) with scales (..., blocks) stand for, in f32."""
    if kind == "q8_0":
        c = codes.float() - 128.0
    else:
        b = codes.unflatten(-1, (-1, 16))
        c = torch.cat((b & 15, b >> 4), -1).float() - 8.0
    return (c.reshape(*scales.shape, 32) * scales.float()[..., None]).flatten(-2)


def _codes(x, kind):
    """Codes and scales of rows (..., head_dim), by the rules of the Q8_0 and Q4_0 blocks."""
    b = x.float().unflatten(-1, (-1, 32))
    most = torch.full((), 127.0 if kind == "q8_0" else 7.0, device="cuda")  # a tensor: torch multiplies by a number's inverse
    d = (b.abs().amax(-1) / most).half()
    q = b / d.float()[..., None]  # in f32, as the block format's rule has it
    whole = torch.trunc(q)
    q = whole + torch.sign(q) * ((q - whole).abs() >= 0.5)  # halves away from zero
    q = torch.where(d[..., None] == 0, torch.zeros_like(q), q)
    if kind == "q8_0":
        return (q.clamp(-127, 127) + 128).to(torch.uint8).flatten(-2), d
    q = (q.clamp(-8, 7) + 8).to(torch.uint8)
    return (q[..., :16] | (q[..., 16:] << 4)).flatten(-2), d


def _plain_cache(s):
    case, out = s["case"], []
    kc, ks, vc, vs = _planes(case, s["pool"], s["pages"])
    page, at = _slots(s)
    for x, codes, scales in ((s["k"], kc, ks), (s["v"], vc, vs)):
        codes[page, :, at], scales[page, :, at] = _codes(x, case["cache"])
        out.append(_values(codes[page, :, at], scales[page, :, at], case["cache"]).to(x.dtype))
    return tuple(out)


def _plain_attn(s):
    case = s["case"]
    kvh, hd, n = case["kv_heads"], case["head_dim"], case["seqs"]
    group, new, length = case["heads"] // kvh, s["most_new"], s["most_len"]
    table = s["table"].long().clamp(min=0)
    kc, ks, vc, vs = _planes(case, s["pool"], s["pages"])

    def rows(codes, scales):  # (n, kvh, length, hd), pages in order
        x = _values(codes[table], scales[table], case["cache"])
        return x.transpose(1, 2).reshape(n, kvh, -1, hd)[:, :, :length]

    start = s["start"].long()
    count = start[1:] - start[:-1]
    j = torch.arange(new, device="cuda")
    here = j[None] < count[:, None]
    token = torch.where(here, start[:-1, None] + j, 0)
    q = s["q"][token].float().view(n, new, kvh, group, hd).permute(0, 2, 1, 3, 4).reshape(n, kvh, new * group, hd)
    score = (q @ rows(kc, ks).transpose(-1, -2) * hd ** -0.5).view(n, kvh, new, group, length)
    draft = torch.arange(length, device="cuda")[None] - s["ctx"].long()[:, None]  # of each position; negative: context
    if s["mask"] is None:
        sees = draft[:, None, :] <= j[None, :, None]
    else:
        words = s["mask"][token]
        at = draft.clamp(0, new - 1)
        bits = torch.gather(words, 2, (at >> 5)[:, None, :].expand(n, new, length)) >> (at & 31)[:, None, :]
        sees = (draft < 0)[:, None, :] | ((bits & 1) == 1)
    sees = sees & (draft < count[:, None])[:, None, :]
    score = score.masked_fill(~sees[:, None, :, None, :], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (score - top).exp_()
    del score
    total = p.sum(-1, keepdim=True)
    out = p.view(n, kvh, new * group, length) @ rows(vc, vs)
    out = out / total.view(n, kvh, new * group, 1).clamp(min=1e-38)
    out = out.view(n, kvh, new, group, hd).permute(0, 2, 1, 3, 4).reshape(n, new, kvh * group, hd)
    return out[here].to(s["q"].dtype)


def _plain_logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    y = x - top
    e = y.exp()
    z = e.sum(-1, keepdim=True)
    logz = z.log()
    lp = torch.gather(y, 1, s["tokens"].long()) - logz
    entropy = (logz - (e * y).sum(-1, keepdim=True) / z).squeeze(1)
    out = [lp, entropy]
    if s["case"]["top"]:
        ids = x.sort(dim=-1, descending=True, stable=True)[1][:, :s["case"]["top"]]
        out += [ids.int(), torch.gather(y, 1, ids) - logz]
    return tuple(out)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        if op == "rope":
            return s["plan"].apply(s["positions"], s["q"], s["k"], inverse=s["case"]["inverse"])
        if op == "cache":
            s["cache"].write(0, s["k"], s["v"], s["batch"])
            return s["cache"].read(0, s["batch"], dtype=s["k"].dtype)
        if op == "attn":
            from m3_avm_b200.attention import tree_attention

            return tree_attention(s["q"], s["cache"], 0, s["batch"], mask=s["mask"])
        from m3_avm_b200.logprobs import token_logprobs

        return tuple(x for x in token_logprobs(s["logits"], s["tokens"], n_top=s["case"]["top"], entropy=True)
                     if x is not None)
    return {"rope": _plain_rope, "cache": _plain_cache, "attn": _plain_attn, "logprobs": _plain_logprobs}[op](s)


# ---------------------------------------------------------------- 64 bits
def _exact_rope(s):
    case = s["case"]
    d, half, orig = case["rot_dim"], case["rot_dim"] // 2, 8192.0
    base = case["theta"] * (case["factor"] ** (d / (d - 2.0)) if case["scaling"] == "ntk" else 1.0)
    f, mag = np.empty(half), 1.0
    for i in range(half):
        w = math.exp(-2.0 * i / d * math.log(base))
        if case["scaling"] == "linear":
            w /= case["factor"]
        elif case["scaling"] == "yarn":
            mag = 1.0 + 0.1 * math.log(case["factor"])
            lo, hi = (d / 2.0 * math.log(orig / (2.0 * math.pi * t)) / math.log(base) for t in (32.0, 1.0))
            lo, hi = max(0, math.floor(lo)), min(d - 1, math.ceil(hi))
            r = min(1.0, max(0.0, (i - lo) / max(hi - lo, 0.001)))
            w = r * w / case["factor"] + (1.0 - r) * w
        elif case["scaling"] == "llama3":
            turns = orig * w / (2.0 * math.pi)  # over the original context
            r = min(1.0, max(0.0, (turns - 1.0) / 3.0))
            w = r * w + (1.0 - r) * w / case["factor"]
        f[i] = w
    sign = -1.0 if case["inverse"] else 1.0
    z = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                    sign * s["positions"].double()[:, None] * torch.from_numpy(f).cuda()) * mag
    out = []
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        first, second = (slice(0, d, 2), slice(1, d, 2)) if case["interleaved"] else (slice(0, half), slice(half, d))
        w = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * z[:, None, :]
        y[..., first], y[..., second] = w.real, w.imag
        out.append(y)
    return tuple(out)


def _exact_cache(s):
    """What the cache holds is defined by the block format's rule, f32 quotient and f16 scale included."""
    out, eight = [], s["case"]["cache"] == "q8_0"
    for x in (s["k"], s["v"]):
        b = x.double().reshape(-1, 32)
        big = b.abs().max(1, keepdim=True).values
        d = (big / (127 if eight else 7)).float().half().double()
        q = torch.where(d > 0, b / d, torch.zeros_like(b)).float().double()
        q = torch.where(q < 0, torch.ceil(q - 0.5), torch.floor(q + 0.5))
        q = q.clamp(-127, 127) if eight else q.clamp(-8, 7)
        out.append((q * d).reshape(x.shape))
    return tuple(out)


def _exact_attn(s):
    case = s["case"]
    hd, kvh, page = case["head_dim"], case["kv_heads"], case["page"]
    group = case["heads"] // kvh
    ctx, start = s["ctx"].tolist(), s["start"].tolist()
    out = torch.empty(s["total"], case["heads"], hd, dtype=torch.float64, device="cuda")
    planes = _planes(case, s["pool"], s["pages"])
    for i in range(case["seqs"]):
        a, b = start[i], start[i + 1]
        n, length = b - a, ctx[i] + b - a
        pages = s["table"][i, :-(-length // page)].long()
        held = []
        for codes, scales in (planes[:2], planes[2:]):
            c, d = codes[pages], scales[pages].double()
            if case["cache"] == "q8_0":
                v = c.double() - 128
            else:
                c = c.reshape(*c.shape[:-1], hd // 32, 16)
                v = torch.stack((c % 16, c // 16), -2).double().reshape(*c.shape[:-2], hd) - 8
            v = v * d.repeat_interleave(32, -1)
            held.append(v.permute(1, 0, 2, 3).reshape(kvh, -1, hd)[:, :length])
        sees = torch.ones(n, length, dtype=torch.bool, device="cuda")
        if s["mask"] is None:
            sees[:, ctx[i]:] = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        else:
            for k in range(n):
                sees[:, ctx[i] + k] = ((s["mask"][a:b, k // 32] >> (k % 32)) & 1).bool()
        q = s["q"][a:b].double().view(n, kvh, group, hd)
        for h in range(kvh):
            w = torch.einsum("nge,le->ngl", q[:, h], held[0][h]) / math.sqrt(hd)
            w = torch.softmax(w.masked_fill(~sees[:, None], -math.inf), -1)
            out[a:b, h * group:(h + 1) * group] = torch.einsum("ngl,le->nge", w, held[1][h])
    return out


def _exact_logprobs(s):
    parts = [[], [], [], []]
    top = s["case"]["top"]
    for x, t in zip(s["logits"].split(64), s["tokens"].split(64)):
        lp = torch.log_softmax(x.double(), -1)
        parts[0].append(lp.gather(1, t.long()))
        parts[1].append(-(lp.exp() * lp).sum(-1))
        if top:
            ids = torch.sort(-x.double(), dim=-1, stable=True).indices[:, :top]
            parts[2].append(ids.int())
            parts[3].append(lp.gather(1, ids))
    return tuple(torch.cat(p) for p in parts if p)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "cache": _exact_cache, "attn": _exact_attn, "logprobs": _exact_logprobs}[case["op"]](s)
