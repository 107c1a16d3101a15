"""Plain implementations, in 64 bits on the CPU, of the 4-bit paged cache and of page bookkeeping."""
from __future__ import annotations

import math

import numpy as np
import torch

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
VALUE = np.concatenate([E2M1, -E2M1])
E4M3 = np.array([i for i in range(127)], dtype=np.uint8)                  # the positive finite codes, in order
E4M3_VALUE = torch.from_numpy(E4M3).view(torch.float8_e4m3fn).double().numpy()
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _nearest(values, x):
    """Index of the nearest of ``values`` (ascending), ties to the even index (whose last mantissa bit is zero), beyond the last: the last."""
    hi = np.clip(np.searchsorted(values, x, side="left"), 1, len(values) - 1)
    lo = hi - 1
    below, above = x - values[lo], values[hi] - x
    return np.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, lo)


def quantise(x: torch.Tensor, unit: float):
    """Codes uint8 [..., E/2] and scale codes uint8 [..., E/16] of rows [..., E]."""
    g = x.double().numpy().reshape(*x.shape[:-1], -1, 16)
    top = np.abs(g).max(-1)
    ok = np.isfinite(g).all(-1)
    scale = np.where(ok, E4M3[_nearest(E4M3_VALUE, np.where(ok, top, 0) / 6 / unit)], 127).astype(np.uint8)
    step = np.where(ok, E4M3_VALUE[np.minimum(scale, 126)], 0)[..., None] * unit
    y = np.where(step > 0, np.abs(np.where(ok[..., None], g, 0)) / np.where(step > 0, step, 1), 0)
    code = np.where(step > 0, _nearest(E2M1, y) + 8 * (g < 0), 0).astype(np.uint8).reshape(x.shape)      # (zeros are positive)
    return torch.from_numpy(code[..., 0::2] | code[..., 1::2] << 4), torch.from_numpy(scale)


def values(codes: torch.Tensor, scales: torch.Tensor, unit: float) -> np.ndarray:
    """What codes and scale codes (uint8) stand for."""
    c = codes.numpy()
    code = np.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)
    s = scales.view(torch.float8_e4m3fn).double().numpy() * unit
    with np.errstate(invalid="ignore"):
        return VALUE[code] * np.repeat(s, 16, -1)


def random_cache(gen, blocks, Hkv, bs, E, unit=1.0):
    codes, scales = quantise(torch.randn(blocks, Hkv, bs, E, generator=gen) * 1.5 * unit, unit)
    return codes, scales


def sequence(codes, scales, unit, table_row, n):
    """Rows 0 .. n-1 of one paged sequence, [Hkv,n,E], and which of them have a page."""
    blocks, Hkv, bs = codes.shape[:3]
    full = values(codes, scales, unit)
    out, there = np.zeros((Hkv, n, full.shape[-1])), np.zeros(n, bool)
    for l in range(n):
        page = int(table_row[l // bs]) if l // bs < len(table_row) else -1
        if 0 <= page < blocks:
            out[:, l], there[l] = full[page, :, l % bs], True
    return out, there


def attention(q, loc, lens, kc, vc, ks, vs, table, scale, ku=1.0, vu=1.0, cu=None):
    """Output [rows, Hq, Ev] in 64 bits and what bounds the error of a kernel's: sum p|v| / sum p, the largest sum |q||k| scale, the most
    keys of a row, the largest |v|.

    ``q [F,rows,Hq,E]``, ``loc [F,rows]``, ``lens [F,W]``; row ``i`` belongs to sequence ``seq[i]`` (``cu``)."""
    F, rows, Hq, E = q.shape
    W, Hkv = table.shape[0], kc.shape[1]
    G, Ev = Hq // Hkv, vc.shape[-1] * 2
    qd = q.double().numpy()
    out, weight, top = np.zeros((rows, Hq, Ev)), np.zeros((rows, Hq, Ev)), 0.0
    most, vmax = 0, 0.0
    for w in range(W):
        mine = range(int(cu[w]), int(cu[w + 1]))
        longest = max([0] + [max(0, min(int(loc[f, i]) + 1, int(lens[f, w]))) for f in range(F) for i in mine])
        K, there = sequence(kc, ks, ku, table[w], longest)
        V, _ = sequence(vc, vs, vu, table[w], longest)
        most, vmax = max(most, F * longest), max(vmax, float(np.nanmax(np.abs(V), initial=0.0)))
        for i in mine:
            for h in range(Hq):
                z, v = [], []
                for f in range(F):
                    n = max(0, min(int(loc[f, i]) + 1, int(lens[f, w])))
                    seen = np.nonzero(there[:n])[0]
                    z.append(K[h // G, seen] @ qd[f, i, h] * scale)
                    v.append(V[h // G, seen])
                    if len(seen):
                        mags = np.abs(K[h // G, seen]) @ np.abs(qd[f, i, h]) * abs(scale)
                        top = max(top, float(np.nanmax(mags, initial=0.0, where=np.isfinite(mags))))
                z, v = np.concatenate(z), np.concatenate(v)
                if len(z):
                    with np.errstate(invalid="ignore"):
                        p = np.exp(z - z.max())
                        out[i, h] = (p[:, None] * v).sum(0) / p.sum()
                        weight[i, h] = (p[:, None] * np.abs(v)).sum(0) / p.sum()
    return out, weight, top, most, vmax


def tolerance(dtype, ref, weight, top, keys, vmax):
    """How far an output may be from the exact one.

    * its rounding: half a step of the type;
    * probabilities: a score is a sum of at most 256 products in fp32 (each addition off by at most a step, 2^-23, of what has been added
      up, which `top` bounds), times the scale and log2 e (3 roundings), so p is off by a factor of at most exp(259 * 2^-23 * top); the
      exponential itself is good to 2 steps; in the numerator and in the denominator: twice;
    * probabilities in fp16 for the tensor cores (16-bit types only): half a step, 2^-11, and below 2^-14 of the row's largest one at
      most 2^-25 absolute, for every key;
    * the sums over `keys` keys in fp32: a step each, in numerator and denominator."""
    p, small = 2 * (259 * 2.0 ** -23 * top + 4 * 2.0 ** -23) + 2 * keys * 2.0 ** -23, 1e-30
    if dtype != torch.float32:
        p += 2.0 ** -11
        small += keys * 2.0 ** -25 * vmax
    return HALF_STEP[dtype] * np.abs(ref) + p * weight + small


def check(out, exact):
    ref = exact[0]
    got = out.detach().cpu().double().numpy().reshape(ref.shape)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), "NaN in other places"
    fine = ~np.isnan(ref)
    worst = (np.abs(got - ref)[fine] / tolerance(out.dtype, ref, np.nan_to_num(exact[1]), *exact[2:])[fine]).max(initial=0.0)
    assert worst <= 1.0, f"{worst:.2f} times the tolerance"


def step_blocks(refs, table, lengths, source, new, bs, caches):
    """The sequential definition.  Plain lists and numpy arrays; caches are changed in place."""
    refs, blocks, width = list(refs), len(refs), len(table[0])
    flags = 0
    rows = [list(r) for r in table]
    for r in rows:
        for p in r:
            if 0 <= p < blocks:
                refs[p] -= 1
    out, lens, room = [], [], []
    for w in range(len(lengths) if source is None else len(source)):
        u = w if source is None else source[w]
        n = max(0, lengths[u]) if 0 <= u < len(rows) else 0
        over = u >= len(rows) or math.ceil(n / bs) > width
        kept = rows[u][:math.ceil(n / bs)] if 0 <= u < len(rows) else []
        if any(not 0 <= p < blocks for p in kept):
            flags |= 1024
        out.append([p if 0 <= p < blocks else -1 for p in kept])
        for p in out[-1]:
            if p >= 0:
                refs[p] += 1
        lens.append(n)
        room.append(-1 if over else 0)
    free = [p for p in range(blocks) if refs[p] == 0]
    left, stopped, pairs = len(free), False, []
    holders = list(refs)                                     # who still holds a page if everybody in front is served
    for w, n in enumerate(lens):
        add = max(0, new[w]) if new is not None else 0
        kept = len(out[w])
        over = room[w] < 0 or math.ceil((n + add) / bs) > width
        room[w] = 0
        if over:
            flags |= 2048
            need, copy = 0, False
        else:
            last = out[w][-1] if add and n % bs else -1
            copy = last >= 0 and holders[last] > 1
            need = math.ceil((n + add) / bs) - kept + copy
            if copy:
                holders[last] -= 1
        stopped = stopped or need > left
        left -= need
        if stopped or over:
            flags |= 512 if add and not over else 0
            continue
        room[w] = add
        got = [free.pop(0) for _ in range(need)]
        for p in got:
            refs[p] = 1
        if copy:
            refs[out[w][-1]] -= 1
            pairs.append((out[w][-1], got[0]))
            out[w][-1] = got.pop(0)
        out[w] += got
    for a, b in pairs:
        for c in caches:
            c[b] = c[a]
    return refs, [r + [-1] * (width - len(r)) for r in out], lens, room, flags


def compact_blocks(refs, table, caches):
    n = sum(r != 0 for r in refs)
    holes = [p for p in range(n) if refs[p] == 0]
    movers = [p for p in range(n, len(refs)) if refs[p] != 0]
    moved = [p if refs[p] != 0 else -1 for p in range(len(refs))]
    refs, flags = list(refs), 0
    for a, b in zip(movers, holes):
        moved[a], refs[b], refs[a] = b, refs[a], 0
        for c in caches:
            c[b] = c[a]
    out = []
    for row in table:
        out.append([moved[p] if 0 <= p < len(refs) else -1 for p in row])
        flags |= 1024 * any(p >= 0 and q < 0 for p, q in zip(row, out[-1]))
    return refs, out, moved, flags
