"""64-bit (or exact) restatements of the serving operators, on CPU tensors, for the tests."""
import math
import random

import numpy as np
import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


# ---------------------------------------------------------------- rope
def frequencies(rot, theta=10000.0, scaling="none", factor=1.0, orig_ctx=0, low_freq=1.0, high_freq=4.0,
                beta_fast=32.0, beta_slow=1.0):
    if scaling == "ntk":
        theta = theta * factor ** (rot / (rot - 2))
    f = np.array([theta ** (-2.0 * i / rot) for i in range(rot // 2)])
    mag = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn":
        idx = lambda turns: rot * math.log(orig_ctx / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(idx(beta_fast)), 0), min(math.ceil(idx(beta_slow)), rot - 1)
        ramp = np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 0.001), 0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mag = 0.1 * math.log(factor) + 1
    if scaling == "llama3":
        out = []
        for w in f:
            wave = 2 * math.pi / w
            if wave < orig_ctx / high_freq:
                out.append(w)
            elif wave > orig_ctx / low_freq:
                out.append(w / factor)
            else:
                s = (orig_ctx / wave - low_freq) / (high_freq - low_freq)
                out.append((1 - s) * w / factor + s * w)
        f = np.array(out)
    return f, mag


def rope(x, positions, rot, interleaved, f, mag, inverse=False):
    """x (T, H, D) -> float64; angles reduced with integers and fractions of a turn kept in longdouble."""
    x = x.double().cpu().numpy()
    ang = positions.cpu().numpy().astype(np.longdouble)[:, None] * np.asarray(f, np.longdouble)[None]
    c, s = (np.cos(ang) * mag).astype(np.float64)[:, None], (np.sin(ang) * mag).astype(np.float64)[:, None]
    if inverse:
        s = -s
    y = x.copy()
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y, np.abs(x[..., a]) + np.abs(x[..., b]), a, b


# ---------------------------------------------------------------- cache
def quantised(x, q8):
    """Values that rows (..., head_dim) leave in the cache: f32 arithmetic of the block rules, exact products."""
    b = x.float().cpu().numpy().reshape(-1, 32)
    out = np.empty_like(b)
    with np.errstate(all="ignore"):
        big = np.max(np.abs(b), axis=1)
        d = (big / np.float32(127 if q8 else 7)).astype(np.float32).astype(np.float16)
        for i in range(b.shape[0]):
            if not np.all(np.isfinite(b[i])) or not np.isfinite(d[i]):
                out[i] = np.nan
                continue
            ds = np.float32(d[i])
            if ds == 0:
                out[i] = 0
                continue
            q = (b[i] / ds).astype(np.float32).astype(np.float64)
            q = np.sign(q) * np.floor(np.abs(q) + 0.5)
            q = np.clip(q, -127, 127) if q8 else np.clip(q, -8, 7)
            out[i] = (q * float(ds)).astype(np.float32)
    return torch.from_numpy(out.reshape(x.shape))


# ---------------------------------------------------------------- batches
def make_batch(ctx, new, page, extra_pages=2, seed=0, device="cuda"):
    """Page table of shuffled pages and the rest of a batch's arrays."""
    from m3_avm_b200.attention import KvBatch

    r = random.Random(seed)
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    pages = sum(need) + extra_pages
    order = list(range(pages))
    r.shuffle(order)
    table = torch.full((len(ctx), max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, k in enumerate(need):
        table[i, :k] = torch.tensor(order[at:at + k], dtype=torch.int32)
        at += k
    start = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    t = lambda x: x.to(device)  # noqa: E731
    b = KvBatch(t(start), t(torch.tensor(ctx, dtype=torch.int32)), t(table), int(sum(new)), max(max(new), 0),
                max(c + n for c, n in zip(ctx, new)))
    return b, pages, table, start


def whole(batch, ctx, new, device="cuda"):
    """A batch whose new tokens are all positions of the sequences."""
    from m3_avm_b200.attention import KvBatch

    length = [c + n for c, n in zip(ctx, new)]
    start = torch.tensor([0] + list(np.cumsum(length)), dtype=torch.int32, device=device)
    return KvBatch(start, torch.zeros(len(ctx), dtype=torch.int32, device=device), batch.page_table, sum(length),
                   max(length), batch.max_len)


def tree_bits(new, seed=0, empty=()):
    """Boolean visibility (n, n) per sequence of random trees; rows in `empty` (token numbers) see nothing."""
    r = random.Random(seed)
    out, t = [], 0
    for n in new:
        m = np.zeros((n, n), bool)
        for j in range(n):
            if j:
                m[j] = m[r.randrange(j)]
            m[j, j] = True
        for j in range(n):
            if t + j in empty:
                m[j] = False
        t += n
        out.append(m)
    return out


def pack_bits(bits, words, device="cuda"):
    rows = []
    for m in bits:
        w = np.zeros((m.shape[0], words * 32), np.uint8)
        w[:, :m.shape[1]] = m
        rows.append(np.packbits(w.reshape(m.shape[0], words, 32), axis=-1, bitorder="little").view(np.uint32)[..., 0])
    return torch.from_numpy(np.concatenate(rows).view(np.int32).copy()).to(device)


# ---------------------------------------------------------------- attention
def attention(q, k, v, ctx, new, bits, scale):
    """q (T, H, D); k, v lists of (len, KVH, D) float64 per sequence; bits per sequence.  Returns the result and, per
    (token, head), the largest |v| seen and the largest scale * sum |q_i k_i| over the seen positions."""
    q = q.double().cpu()
    T, H, D = q.shape
    out = torch.zeros(T, H, D, dtype=torch.float64)
    vmax = torch.zeros(T, H, dtype=torch.float64)
    smag = torch.zeros(T, H, dtype=torch.float64)
    t = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        g = H // k[s].shape[1]
        for j in range(n):
            see = np.concatenate([np.ones(c, bool), bits[s][j]])
            if see.any():
                kk = k[s][see].repeat_interleave(g, 1)
                vv = v[s][see].repeat_interleave(g, 1)
                qq = q[t + j]
                w = torch.softmax(torch.einsum("hd,lhd->hl", qq, kk) * scale, -1)
                out[t + j] = torch.einsum("hl,lhd->hd", w, vv)
                vmax[t + j] = vv.abs().amax(dim=(0, 2)) if vv.shape[1] == 1 else vv.abs().amax(0).amax(-1)
                smag[t + j] = (torch.einsum("hd,lhd->hl", qq.abs(), kk.abs()) * scale).amax(-1)
        t += n
    return out, vmax, smag


def attention_bound(out, vmax, smag, dtype):
    """|error| allowed.  A score is off by at most es, so each weight by a factor e^(2 es) ~ 1 + 2 es, and the result
    by (2 es + ew) max|v|, ew the error of weights and values themselves.
      f32: q and p in two f16 parts of 11 bits each (2^-22), codes exact, sums of at most 128 products in f32 of
           32-term blocks (2^-23 each step, 12 steps at most): es = 2^-19 smag; weights: exp2 2^-22, p's parts 2^-21,
           f32 sums over the warps and splits 2^-18: ew = 2^-17.
      16 bits: cached values as f16 products at worst (2^-11 each in es and ew) and p as f16 (2^-11), and what f32 has.
    The result is rounded once."""
    if dtype == torch.float32:
        es, ew = 2.0 ** -19 * smag, 2.0 ** -17
    else:
        es, ew = (2.0 ** -11 + 2.0 ** -19) * smag, 2 * 2.0 ** -11 + 2.0 ** -17
    return ((2 * es + ew) * vmax)[..., None] + EPS[dtype] * out.abs() + 1e-30
