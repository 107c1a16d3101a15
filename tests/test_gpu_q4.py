"""The 4-bit paged cache on the GPU against the plain implementation in 64 bits."""
import numpy as np
import pytest
import torch

from tests import q4_util

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def A():
    import inference_lib_b200.attention as mod
    return mod


def dev(*tensors):
    return [t.to(DEV) for t in tensors]


def table_of(rng, W, width, blocks):
    """Every page once, in no order; -1 where there are too few."""
    perm = rng.permutation(blocks)[:W * width]
    return torch.from_numpy(np.concatenate([perm, np.full(W * width - len(perm), -1)]).astype(np.int32)).reshape(W, width)


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


# ---- write path -------------------------------------------------------------------------------------------------------
def states(gen, dtype, *shape):
    """Rows with everything a group can hold: ordinary numbers, few-bit ones (ties), zeros, tiny and huge ones, infinities and NaN."""
    x = torch.randn(*shape, generator=gen)
    kind = torch.randint(0, 12, shape[:-1] + (shape[-1] // 16,), generator=gen)[..., None].expand(*shape[:-1], shape[-1] // 16, 16).reshape(shape)
    x = torch.where(kind == 1, (x * 8).round() / 4, x)
    x = torch.where(kind == 2, 0.0, x)
    x = torch.where(kind == 3, x * 2.0 ** -9, x)
    x = torch.where(kind == 4, x * 2000, x)
    x = torch.where(kind == 5, torch.randint(-12, 13, shape, generator=gen) / 2.0, x)
    x = torch.where((kind == 6) & (torch.rand(*shape, generator=gen) < 0.03), float("inf"), x)
    x = torch.where((kind == 7) & (torch.rand(*shape, generator=gen) < 0.03), float("nan"), x)
    return x.to(dtype)


def stored(k, v, kc, vc, ks, vs, table, lengths, unit, counts=None):
    """The four cache tensors (uint8) after the append of k, v [B,Hkv,S,E]."""
    out = [t.clone() for t in (kc, vc, ks, vs)]
    blocks, bs = kc.shape[0], kc.shape[2]
    for x, codes, scales, u in ((k, out[0], out[2], unit[0]), (v, out[1], out[3], unit[1])):
        c, s = q4_util.quantise(x, u)
        for b in range(x.shape[0]):
            for t in range(x.shape[2] if counts is None else min(x.shape[2], max(0, int(counts[b])))):
                pos = int(lengths[b]) + t
                page = int(table[b, pos // bs]) if 0 <= pos // bs < table.shape[1] else -1
                if 0 <= page < blocks:
                    codes[page, :, pos % bs], scales[page, :, pos % bs] = c[b, :, t], s[b, :, t]
    return out


def empty_cache(gen, blocks, Hkv, bs, E, Ev):
    return [torch.randint(0, 256, (blocks, Hkv, bs, n), dtype=torch.uint8, generator=gen) for n in (E // 2, Ev // 2, E // 16, Ev // 16)]


APPENDS = [
    # dtype, B, Hkv, S, E, Ev, bs, units
    (torch.bfloat16, 3, 2, 5, 128, 128, 16, (1.0, 1.0)),
    (torch.float16, 2, 3, 40, 64, 64, 24, (0.25, 2.0)),
    (torch.float32, 2, 1, 9, 16, 256, 8, (1.0, 2.0 ** -20)),
    (torch.bfloat16, 1, 4, 1, 240, 32, 1, (2.0 ** 5, 1.0)),
]


@pytest.mark.parametrize("case", APPENDS, ids=[str(i) for i in range(len(APPENDS))])
@pytest.mark.parametrize("layout", ["contiguous", "transposed", "shifted", "packed"])
def test_append_stores_the_very_bits(A, case, layout):
    dtype, B, Hkv, S, E, Ev, bs, units = case
    gen, rng = torch.Generator().manual_seed(S * E + bs), np.random.default_rng(S)
    width = (S + 30) // bs + 1
    blocks = B * width + 2
    table = table_of(rng, B, width, blocks)
    lengths = torch.tensor([0, 29, 13][:B], dtype=torch.int32)
    k, v = states(gen, dtype, B, Hkv, S, E), states(gen, dtype, B, Hkv, S, Ev)
    cache = empty_cache(gen, blocks, Hkv, bs, E, Ev)
    want = stored(k, v, *cache, table, lengths, units)
    dk, dv, dt, dl = dev(k, v, table, lengths)
    more = {}
    if layout == "transposed":                               # what a projection leaves
        dk, dv = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (dk, dv))
    elif layout == "shifted":                                # rows off the 16-byte boundary
        dk, dv = (torch.cat([x[..., :1], x, x[..., :2]], -1)[..., 1:-2] for x in (dk, dv))
    elif layout == "packed":
        dk, dv = (x.transpose(1, 2).reshape(B * S, Hkv, x.shape[-1]) for x in (dk, dv))
        more = dict(cu_seqlens=torch.arange(B + 1, dtype=torch.int32, device=DEV) * S)
    dc = dev(*cache)
    st = status()
    A.copy_to_blocks_q4(dk, dv, dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), dt, dl, key_unit=units[0], value_unit=units[1], status=st, **more)
    for got, ref in zip(dc, want):
        assert torch.equal(got.cpu(), ref)
    assert int(st) == 0


def test_append_drops_rows_without_a_page(A):
    gen = torch.Generator().manual_seed(0)
    B, Hkv, S, E, bs, blocks = 4, 2, 6, 64, 4, 9
    table = torch.tensor([[0, -1, 2], [3, 9, 4], [5, 6, 7], [1, 8, -1]], dtype=torch.int32)
    lengths = torch.tensor([1, 2, 9, -2], dtype=torch.int32)              # a hole, a page outside, behind the table, in front of it
    k, v = (torch.randn(B, Hkv, S, E, generator=gen).half() for _ in range(2))
    cache = empty_cache(gen, blocks, Hkv, bs, E, E)
    want = stored(k, v, *cache, table, lengths, (1.0, 1.0))
    dc, st = dev(*cache), status()
    A.copy_to_blocks_q4(*dev(k, v), dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), *dev(table, lengths), status=st)
    assert all(torch.equal(g.cpu(), r) for g, r in zip(dc, want)) and int(st) == 1024
    # counts: rows from there on stay out, their pages need not be there
    counts = torch.tensor([3, 2, 3, 0], dtype=torch.int32)
    lengths = torch.tensor([1, 2, 9, -2], dtype=torch.int32)
    want = stored(k, v, *cache, table, lengths, (1.0, 1.0), counts)
    dc, st = dev(*cache), status()
    A.copy_to_blocks_q4(*dev(k, v), dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), *dev(table, lengths), new_rows=counts.to(DEV), status=st)
    assert all(torch.equal(g.cpu(), r) for g, r in zip(dc, want)) and int(st) == 0


def test_packed_append_with_empty_sequences_and_a_tail(A):
    gen = torch.Generator().manual_seed(1)
    Hkv, E, bs, counts = 2, 128, 8, [3, 0, 0, 5, 1, 0]
    B, T = len(counts), sum(counts)
    table = torch.arange(B * 3, dtype=torch.int32).reshape(B, 3)
    lengths = torch.tensor([7, 0, 3, 10, 23, 1], dtype=torch.int32)
    k, v = (torch.randn(T + 4, Hkv, E, generator=gen).bfloat16() for _ in range(2))         # four tokens behind the last sequence
    cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    cache = empty_cache(gen, B * 3, Hkv, bs, E, E)
    padded = [torch.zeros(B, Hkv, max(counts), E) for _ in range(2)]
    for b, n in enumerate(counts):
        for x, p in zip((k, v), padded):
            p[b, :, :n] = x[int(cu[b]):int(cu[b]) + n].transpose(0, 1)
    want = stored(*padded, *cache, table, lengths, (1.0, 1.0), counts)
    dc = dev(*cache)
    A.copy_to_blocks_q4(*dev(k, v), dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), *dev(table, lengths), cu_seqlens=cu.to(DEV))
    assert all(torch.equal(g.cpu(), r) for g, r in zip(dc, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("E,Ev,unit", [(128, 128, 1.0), (64, 32, 0.25), (16, 256, 4.0)])
def test_reading_back(A, dtype, E, Ev, unit):
    gen, rng = torch.Generator().manual_seed(E), np.random.default_rng(E)
    B, Hkv, S, bs, blocks = 3, 2, 11, 8, 14
    table = table_of(rng, B, 4, blocks - 1)
    table[1, 2], table[2, 1] = -1, blocks
    first = torch.tensor([2, 5, 25], dtype=torch.int32)
    cache = empty_cache(gen, blocks, Hkv, bs, E, Ev)                       # any bits: NaN scales and negative ones among them
    dc, st = dev(*cache), status()
    keys, vals = A.copy_from_blocks_q4(dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), *dev(table, first), S, dtype=dtype, key_unit=unit,
                                       value_unit=2 * unit, status=st)
    for got, codes, scales, u in ((keys, cache[0], cache[2], unit), (vals, cache[1], cache[3], 2 * unit)):
        full = q4_util.values(codes, scales, u)
        want = np.full(got.shape, np.nan)
        for b in range(B):
            for t in range(S):
                pos = int(first[b]) + t
                page = int(table[b, pos // bs]) if pos // bs < 4 else -1
                if 0 <= page < blocks:
                    want[b, :, t] = full[page, :, pos % bs]
        assert np.array_equal(got.cpu().double().numpy(), torch.from_numpy(want).to(dtype).double().numpy(), equal_nan=True)
    assert int(st) == 1024


# ---- attention ----------------------------------------------------------------------------------------------------------
def paged(A, q, loc, lens, cache, table, scale, units=(1.0, 1.0), cu=None, out=None, st=None, kernel=None):
    """One call, and the same in 64 bits.  Fixed layout: q [F,W,Hq,S,E]."""
    kc, vc, ks, vs = cache
    dc = dev(*cache)
    more = dict(key_unit=units[0], value_unit=units[1], status=st)
    args = (*dev(q, loc), dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), table.to(DEV), scale, lens.to(DEV))
    if cu is None:
        F, W, Hq, S, E = q.shape
        exact = q4_util.attention(q.transpose(2, 3).reshape(F, W * S, Hq, E), loc.reshape(F, W * S), lens[:, None].expand(F, W), kc, vc, ks, vs,
                                  table, scale, *units, [w * S for w in range(W + 1)])
        got = A.hogwild_paged_sdpa_q4(*args, out, **more).transpose(1, 2).reshape(W * S, Hq, -1)
    else:
        exact = q4_util.attention(q, loc, lens, kc, vc, ks, vs, table, scale, *units, cu)
        got = A.hogwild_varlen_paged_sdpa_q4(*args, cu.to(DEV), out, **more)
    torch.cuda.synchronize()
    if kernel is not None:                                   # the same by a kernel of the caller's choice, workspace full of NaN and canaries behind it
        from inference_lib_b200 import _cabi
        again = torch.full_like(got, float("nan")) if cu is not None else torch.full((q.shape[1], q.shape[2], q.shape[3], vc.shape[3] * 2), float("nan"),
                                                                                       dtype=q.dtype, device=DEV)
        x, keep = _cabi.bind_paged_q4(out=again, queries=args[0], locations=args[1], key_cache=args[2], value_cache=args[3], key_scales=args[4],
                                      value_scales=args[5], block_table=args[6], scale=scale, fragment_lengths=args[8], key_unit=units[0],
                                      value_unit=units[1], cu_seqlens_q=None if cu is None else cu.to(DEV), kernel=kernel)
        keep[0].fill_(0xFF)
        end = x.paged.workspace - keep[0].data_ptr() + x.paged.workspace_bytes
        assert _cabi.launch_paged_q4(x, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        assert bool((keep[0][end:] == 0xFF).all())
        got = again if cu is not None else again.transpose(1, 2).reshape(got.shape)
    return got, exact


KERNELS = [None, 1, 2, 4]                                    # the operator; by name on the CUDA cores; mma.sync; tcgen05


def skip_unless_eligible(kernel, dtype, E, Ev, packed=False, bs=8):
    if kernel == 2 and (dtype == torch.float32 or E != Ev or E not in (64, 128)):
        pytest.skip("not for this type and head size")
    if kernel == 4 and (dtype == torch.float32 or E != 128 or Ev != 128 or not packed or bs % 8):
        pytest.skip("not for this type, head size or layout")


SHAPES = [
    # dtype, W, S, Hkv, G, E, Ev, bs, F, keys, units
    (torch.bfloat16, 2, 1, 2, 4, 128, 128, 16, 1, 1, (1.0, 1.0)),
    (torch.bfloat16, 2, 1, 2, 4, 128, 128, 16, 1, 300, (1.0, 1.0)),
    (torch.float16, 3, 1, 1, 16, 128, 128, 16, 1, 1027, (0.25, 4.0)),
    (torch.bfloat16, 2, 3, 2, 5, 128, 128, 24, 2, 145, (1.0, 0.5)),
    (torch.float16, 2, 2, 2, 7, 64, 64, 8, 2, 130, (1.0, 1.0)),
    (torch.bfloat16, 1, 1, 1, 40, 64, 64, 32, 1, 333, (1.0, 1.0)),
    (torch.float16, 2, 4, 1, 1, 128, 128, 7, 3, 77, (2.0 ** -30, 2.0 ** 10)),
    (torch.bfloat16, 2, 1, 2, 8, 128, 128, 256, 1, 700, (1.0, 1.0)),
    (torch.bfloat16, 1, 9, 1, 3, 64, 64, 1, 1, 60, (1.0, 1.0)),
    (torch.float32, 2, 2, 2, 2, 64, 64, 16, 1, 100, (1.0, 2.0)),
    (torch.float32, 1, 1, 1, 5, 128, 128, 16, 2, 65, (1.0, 1.0)),
    (torch.bfloat16, 2, 2, 1, 2, 112, 32, 16, 1, 90, (1.0, 1.0)),
    (torch.float16, 1, 1, 2, 2, 16, 256, 8, 1, 90, (0.5, 1.0)),
]


@pytest.mark.parametrize("case", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
@pytest.mark.parametrize("kernel", KERNELS)
def test_paged_attention(A, case, kernel):
    dtype, W, S, Hkv, G, E, Ev, bs, F, keys, units = case
    skip_unless_eligible(kernel, dtype, E, Ev)
    gen, rng = torch.Generator().manual_seed(keys), np.random.default_rng(keys)
    width = -(-keys // bs) + 1
    blocks = W * width + 2
    (kc, ks), (vc, vs) = q4_util.random_cache(gen, blocks, Hkv, bs, E, units[0]), q4_util.random_cache(gen, blocks, Hkv, bs, Ev, units[1])
    table = table_of(rng, W, width, blocks)
    q = torch.randn(F, W, Hkv * G, S, E, generator=gen).to(dtype)
    lens = torch.tensor([keys] + [int(x) for x in rng.integers(0, keys + 1, F - 1)], dtype=torch.int32)
    loc = torch.from_numpy(rng.integers(-1, keys + 9, (F, W, S)).astype(np.int32))
    loc[0, 0] = keys - 1
    got, exact = paged(A, q, loc, lens, (kc, vc, ks, vs), table, E ** -0.5 / units[0], units, kernel=kernel)
    q4_util.check(got, exact)


PACKED = [
    # dtype, query tokens, Hkv, G, E, bs, F, keys, units
    (torch.bfloat16, [3, 0, 7, 1], 2, 4, 128, 16, 1, 120, (1.0, 1.0)),
    (torch.float16, [1, 1, 0, 1], 2, 5, 64, 24, 2, 90, (0.5, 1.0)),
    (torch.bfloat16, [40, 1, 0, 2], 1, 7, 128, 8, 1, 301, (1.0, 2.0)),
    (torch.float16, [0, 150, 1, 33], 1, 8, 128, 32, 2, 200, (1.0, 1.0)),
    (torch.bfloat16, [129], 2, 1, 128, 128, 1, 129, (1.0, 1.0)),
    (torch.bfloat16, [200, 1, 70], 2, 4, 128, 24, 1, 700, (0.25, 4.0)),
    (torch.float16, [65, 3, 0, 64], 2, 2, 128, 16, 3, 260, (1.0, 2.0 ** -12)),
    (torch.float32, [2, 3], 1, 20, 128, 16, 1, 50, (1.0, 1.0)),
]


@pytest.mark.parametrize("case", PACKED, ids=[str(i) for i in range(len(PACKED))])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("kernel", KERNELS)
def test_packed_attention(A, case, causal, kernel):
    dtype, counts, Hkv, G, E, bs, F, keys, units = case
    skip_unless_eligible(kernel, dtype, E, E, True, bs)
    gen, rng = torch.Generator().manual_seed(keys), np.random.default_rng(keys)
    W, T, width = len(counts), sum(counts), -(-keys // bs) + 1
    blocks = W * width + 1
    (kc, ks), (vc, vs) = q4_util.random_cache(gen, blocks, Hkv, bs, E, units[0]), q4_util.random_cache(gen, blocks, Hkv, bs, E, units[1])
    table = table_of(rng, W, width, blocks)
    q = torch.randn(F, T, Hkv * G, E, generator=gen).to(dtype)
    lens = torch.from_numpy(np.stack([[max(n, keys - 13 * w) for w, n in enumerate(counts)]] * F).astype(np.int32))
    if causal:
        loc = torch.cat([torch.arange(int(lens[0, w]) - n, int(lens[0, w])) for w, n in enumerate(counts)]).to(torch.int32)[None].repeat(F, 1)
    else:
        loc = torch.from_numpy(rng.integers(-1, keys + 20, (F, T)).astype(np.int32))
    cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    # two rows behind the last sequence: left as they are
    q = torch.cat([q, torch.randn(F, 2, Hkv * G, E, generator=gen).to(dtype)], 1)
    loc = torch.cat([loc, torch.full((F, 2), 5, dtype=torch.int32)], 1)
    out = torch.full((T + 2, Hkv * G, E), 7.0, dtype=dtype, device=DEV)
    st = status()
    got, exact = paged(A, q, loc, lens, (kc, vc, ks, vs), table, E ** -0.5 / units[0], units, cu, out, st, kernel)
    assert bool((out[T:] == 7.0).all()) and int(st) == 0
    q4_util.check(got[:T], (exact[0][:T], exact[1][:T], *exact[2:]))


def odd_scales(rng, cache, table, bs, spots):
    """NaN scales at (sequence, position, key or value, head, group)."""
    for w, pos, which, h, g in spots:
        cache[2 + which][int(table[w, pos // bs]), h, pos % bs, g] = 0x7f if g % 2 else 0xff


@pytest.mark.parametrize("dtype,E,counts,bs", [(torch.bfloat16, 128, [1, 1, 3], 16), (torch.float16, 64, [2, 1, 1], 24), (torch.float32, 64, [1, 2, 1], 16),
                                               (torch.bfloat16, 128, [130, 1, 20], 16)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_numbers_that_are_not(A, dtype, E, counts, bs, kernel):
    """A NaN key is the whole row's, a NaN value its channels', and only of rows that see it; behind the lengths there may be anything."""
    skip_unless_eligible(kernel, dtype, E, E, True, bs)
    gen, rng = torch.Generator().manual_seed(5), np.random.default_rng(5)
    Hkv, G, keys, W, T = 2, 4, 150, len(counts), sum(counts)
    width = -(-keys // bs)
    blocks = W * width
    (kc, ks), (vc, vs) = q4_util.random_cache(gen, blocks, Hkv, bs, E), q4_util.random_cache(gen, blocks, Hkv, bs, E)
    table = table_of(rng, W, width, blocks)
    cache = [kc, vc, ks, vs]
    odd_scales(rng, cache, table, bs, [(0, 40, 1, 0, 3), (0, 147, 1, 1, 0), (1, 60, 0, 1, 2), (2, 149, 1, 0, 1), (2, 149, 0, 1, 1), (2, 100, 0, 0, 0)])
    lens = torch.tensor([[147, 150, 150]], dtype=torch.int32)              # (sequence 0 ends in front of its second one)
    loc = torch.cat([torch.arange(int(lens[0, w]) - n, int(lens[0, w])) for w, n in enumerate(counts)]).to(torch.int32)[None]
    q = torch.randn(1, T, Hkv * G, E, generator=gen).to(dtype)
    q[0, T - 1, 2, 5] = float("nan")
    q[0, 0, 6, 5] = float("inf")                                           # inf * 0 or inf - inf: NaN as well
    cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    got, exact = paged(A, q, loc, lens, cache, table, E ** -0.5, cu=cu, kernel=kernel)
    exact[0][T - 1, 2] = np.nan
    exact[0][0, 6] = np.nan
    q4_util.check(got, exact)


@pytest.mark.parametrize("dtype,E,G", [(torch.bfloat16, 128, 4), (torch.float16, 64, 12), (torch.float32, 128, 2)])
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("bs", [16, 8])
def test_keys_without_a_page_are_not_seen(A, dtype, E, G, kernel, bs):
    skip_unless_eligible(kernel, dtype, E, E)
    gen, rng = torch.Generator().manual_seed(6), np.random.default_rng(6)
    W, Hkv, keys, width = 3, 2, 100, 96 // bs
    (kc, ks), (vc, vs) = (q4_util.random_cache(gen, 4 * width, Hkv, bs, E) for _ in range(2))
    table = table_of(rng, W, width, 4 * width)
    table[0, 2], table[1, 0], table[2] = -1, 4 * width, -7                        # a hole, a page outside, no page at all
    q = torch.randn(1, W, Hkv * G, 2, E, generator=gen).to(dtype)
    loc = torch.tensor([[[98, 99], [20, 95], [50, 99]]], dtype=torch.int32)      # (keys 96 ... lie behind the table)
    st = status()
    got, exact = paged(A, q, loc, torch.tensor([keys], dtype=torch.int32), (kc, vc, ks, vs), table, E ** -0.5, st=st, kernel=kernel)
    q4_util.check(got, exact)
    assert int(st) == 1024 and bool((got.reshape(W, 2, -1)[2] == 0).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kernel", KERNELS)
def test_packed_chunks_over_tables_with_holes(A, dtype, kernel):
    """Keys without a page and values that are not numbers in the middle of chunks, over several fragments; rows that see nothing."""
    gen, rng = torch.Generator().manual_seed(12), np.random.default_rng(12)
    Hkv, G, E, bs, counts, keys, F = 2, 4, 128, 8, [150, 1, 33, 40], 320, 2
    W, T, width, cu = len(counts), sum(counts), keys // bs, torch.tensor([0, 150, 151, 184, 224], dtype=torch.int32)
    (kc, ks), (vc, vs) = (q4_util.random_cache(gen, W * width, Hkv, bs, E) for _ in range(2))
    table = table_of(rng, W, width, W * width)
    cache = [kc, vc, ks, vs]
    odd_scales(rng, cache, table, bs, [(0, 200, 1, 0, 7), (0, 210, 1, 1, 2), (0, 3, 1, 0, 0), (2, 310, 1, 1, 5), (2, 300, 0, 0, 1)])
    table[0, 25], table[0, 12], table[1, :], table[2, 39], table[3, 3] = -1, W * width, -1, 1 << 30, -2        # (25: the page of the first odd value)
    lens = torch.tensor([[320, 320, 320, 0], [100, 7, 320, 33]], dtype=torch.int32)
    loc = torch.from_numpy(rng.integers(-1, keys + 5, (F, T)).astype(np.int32))
    loc[0, :150] = torch.arange(170, 320)
    q = torch.randn(F, T, Hkv * G, E, generator=gen).to(dtype)
    st = status()
    got, exact = paged(A, q, loc, lens, cache, table, E ** -0.5, cu=cu, st=st, kernel=kernel)
    q4_util.check(got, exact)
    assert int(st) == 1024


def test_rows_that_see_nothing_are_zero(A):
    gen = torch.Generator().manual_seed(7)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, 8, 2, 16, 128) for _ in range(2))) for x in pair]
    table = torch.arange(8, dtype=torch.int32).reshape(2, 4)
    q = torch.randn(1, 2, 8, 2, 128, generator=gen).bfloat16()
    loc = torch.tensor([[[-1, -5], [30, -2147483648]]], dtype=torch.int32)
    got, exact = paged(A, q, loc, torch.tensor([50], dtype=torch.int32), cache, table, 0.1)
    q4_util.check(got, exact)
    got, _ = paged(A, q, loc + 60, torch.tensor([0], dtype=torch.int32), cache, table, 0.1)
    assert bool((got == 0).all())


@pytest.mark.parametrize("dtype,E", [(torch.bfloat16, 128), (torch.float16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("kernel", KERNELS)
def test_queries_that_are_no_numbers_and_see_nothing(A, dtype, E, kernel):
    """Zeros, also beside rows of the same tile that see something and over a fragment more that one of them sees."""
    skip_unless_eligible(kernel, dtype, E, E, True, 16)
    gen = torch.Generator().manual_seed(23)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, 8, 2, 16, E) for _ in range(2))) for x in pair]
    table = torch.arange(8, dtype=torch.int32).reshape(2, 4)
    q = torch.randn(2, 8, 8, E, generator=gen).to(dtype)
    loc = torch.tensor([[30, -1, 40, -1, 20, 50, -1, -1], [10, -1, -1, -1, 63, 50, -1, -1]], dtype=torch.int32)
    for row, bad in ((1, float("nan")), (3, float("inf")), (6, float("nan")), (7, -float("inf"))):
        q[:, row, :, 3] = bad
    q[1, 2] = float("nan")                                                    # (sees keys of the other fragment only)
    cu, lens = torch.tensor([0, 4, 8], dtype=torch.int32), torch.tensor([[64, 64], [64, 64]], dtype=torch.int32)
    got, exact = paged(A, q, loc, lens, cache, table, E ** -0.5, cu=cu, kernel=kernel)
    q4_util.check(got, exact)
    assert bool((got[[1, 3, 6, 7]] == 0).all()) and not bool(got.isnan().any())
    if kernel != 4:                                                          # an infinite query of a row that sees one key, whichever sign
        q[0, 0, :, 3], q[0, 5, :, 3], loc[:, 0], loc[:, 5] = float("inf"), -float("inf"), torch.tensor([0, -1]), torch.tensor([0, -1])
        got, exact = paged(A, q, loc, lens, cache, table, E ** -0.5, cu=cu, kernel=kernel)
        q4_util.check(got, exact)
        assert bool(got[[0, 5]].isnan().all())


def test_large_and_small_queries(A):
    """bf16 queries beyond fp16's range, and below it."""
    gen = torch.Generator().manual_seed(8)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, 8, 1, 16, 128) for _ in range(2))) for x in pair]
    table = torch.arange(8, dtype=torch.int32).reshape(2, 4)
    q = torch.randn(1, 2, 8, 1, 128, generator=gen)
    size = 2.0 ** torch.tensor([-40.0, -14, -3, 0, 10, 20, 30, 60])[:, None, None]
    for scale_with in (True, False):                         # (as large as they are; or all rows peaked)
        x = (q * size).bfloat16()
        for h in range(8):
            one = torch.cat([x[:, :, h:h + 1]] * 2, 2)
            got, exact = paged(A, one, torch.full((1, 2, 1), 49, dtype=torch.int32), torch.tensor([50], dtype=torch.int32), cache, table,
                               0.1 / float(size[h]) if scale_with else min(0.1, 0.5 / float(size[h])))
            q4_util.check(got, exact)


@pytest.mark.parametrize("dtype,G,E,bs,W", [(torch.bfloat16, 4, 128, 16, 150), (torch.float16, 2, 64, 8, 330), (torch.bfloat16, 12, 128, 12, 150),
                                            (torch.float16, 3, 64, 24, 80)])
@pytest.mark.parametrize("packed", [False, True])
def test_many_short_sequences(A, dtype, G, E, bs, W, packed):
    """More units than resident CTAs: each has one to itself."""
    gen, rng = torch.Generator().manual_seed(W), np.random.default_rng(W)
    Hkv, keys = 4, 70
    width = -(-keys // bs)
    (kc, ks), (vc, vs) = (q4_util.random_cache(gen, 2 * width + 9, Hkv, bs, E) for _ in range(2))
    table = torch.from_numpy(rng.integers(0, 2 * width + 9, (W, width)).astype(np.int32))              # (pages of many rows)
    q = torch.randn(1, W, Hkv * G, 1, E, generator=gen).to(dtype)
    loc = torch.from_numpy(rng.integers(-1, keys, (1, W, 1)).astype(np.int32))
    if packed:
        got, exact = paged(A, q[:, :, :, 0].contiguous(), loc[:, :, 0], torch.full((1, W), keys, dtype=torch.int32), (kc, vc, ks, vs), table, E ** -0.5,
                           cu=torch.arange(W + 1, dtype=torch.int32))
    else:
        got, exact = paged(A, q, loc, torch.tensor([keys], dtype=torch.int32), (kc, vc, ks, vs), table, E ** -0.5)
    q4_util.check(got, exact)


@pytest.mark.parametrize("dtype,G,E,bs,W,F,longest", [(torch.bfloat16, 4, 128, 16, 50, 1, 500), (torch.float16, 2, 64, 8, 40, 2, 130), (torch.bfloat16, 12, 128, 32, 60, 1, 300),
                                                      (torch.float16, 5, 128, 16, 45, 1, 1), (torch.bfloat16, 4, 128, 16, 39, 3, 900)])
def test_shares_of_many_ragged_units(A, dtype, G, E, bs, W, F, longest):
    """A list whose units' ends count: units of a few tiles and of none, shares that end in front of a unit's first tile."""
    gen, rng = torch.Generator().manual_seed(W), np.random.default_rng(W)
    Hkv, width, pages = 4, -(-longest // bs), 37
    (kc, ks), (vc, vs) = (q4_util.random_cache(gen, pages, Hkv, bs, E) for _ in range(2))
    table = torch.from_numpy(rng.integers(0, pages, (W, width)).astype(np.int32))
    lens = torch.from_numpy(np.where(rng.random((F, W)) < 0.2, 0, rng.integers(1, longest + 1, (F, W))).astype(np.int32))
    counts = rng.integers(0, 3, W)
    counts[0] += W - min(W, int(counts.sum()))                              # (a token per sequence on average, at least)
    cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    T = int(cu[-1])
    loc = torch.from_numpy(rng.integers(longest - 1 - longest // 4, longest, (F, T)).astype(np.int32))
    got, exact = paged(A, torch.randn(F, T, Hkv * G, E, generator=gen).to(dtype), loc, lens, (kc, vc, ks, vs), table, E ** -0.5, cu=cu, kernel=2)
    q4_util.check(got, exact)


@pytest.mark.parametrize("scale", [0.0, -0.1, 1e-30, 3.0])
@pytest.mark.parametrize("kernel", KERNELS)
def test_scales_of_the_scores(A, scale, kernel):
    skip_unless_eligible(kernel, torch.bfloat16, 128, 128)
    gen = torch.Generator().manual_seed(10)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, 8, 2, 16, 128) for _ in range(2))) for x in pair]
    q = torch.randn(1, 2, 6, 1, 128, generator=gen).bfloat16()
    q[0, 0, 1] = 0
    got, exact = paged(A, q, torch.tensor([[[37], [63]]], dtype=torch.int32), torch.tensor([60], dtype=torch.int32), cache,
                       torch.arange(8, dtype=torch.int32).reshape(2, 4), scale, kernel=kernel)
    q4_util.check(got, exact)


CALLS = [
    # packed?, query tokens, W, G, E, bs, keys: shares of a list, units of their own, tcgen05, CUDA cores
    (False, 1, 2, 4, 128, 16, 700), (False, 1, 90, 8, 64, 8, 60), (True, 140, 2, 4, 128, 16, 300), (False, 2, 1, 2, 32, 16, 90),
]


@pytest.mark.parametrize("case", CALLS, ids=[str(i) for i in range(len(CALLS))])
def test_graphs_and_streams(A, case):
    """Append and attention in a graph that is replayed on other contents; the same twice at once on two streams."""
    packed, tokens, W, G, E, bs, keys = case
    gen = torch.Generator().manual_seed(keys)
    Hkv, width = 4, -(-keys // bs) + 1
    blocks, T = W * width, tokens * W
    cu = torch.arange(W + 1, dtype=torch.int32, device=DEV) * tokens
    table = torch.randperm(blocks, generator=gen).to(torch.int32).reshape(W, width).to(DEV)

    def state(seed):
        g = torch.Generator().manual_seed(seed)
        (kc, ks), (vc, vs) = (q4_util.random_cache(g, blocks, Hkv, bs, E) for _ in range(2))
        new = [torch.randn(T, Hkv, E, generator=g).bfloat16() if packed else torch.randn(W, Hkv, tokens, E, generator=g).bfloat16() for _ in range(2)]
        q = torch.randn((1, T, Hkv * G, E) if packed else (1, W, Hkv * G, tokens, E), generator=g).bfloat16()
        have = torch.randint(keys // 2, keys - tokens, (W,), generator=g).to(torch.int32)
        loc = (have[:, None] + torch.arange(tokens)).to(torch.int32)
        return dev(kc, vc, ks, vs, *new, q, have, (loc.reshape(1, T) if packed else loc[None]).contiguous())

    def call(s):
        kc, vc, ks, vs, k, v, q, have, loc = s
        cache = (kc, vc, ks.view(E4M3), vs.view(E4M3), table)
        A.copy_to_blocks_q4(k, v, *cache, have, cu_seqlens=cu if packed else None)
        if packed:
            return A.hogwild_varlen_paged_sdpa_q4(q, loc, *cache, E ** -0.5, (have + tokens)[None], cu)
        return A.hogwild_paged_sdpa_q4(q, loc, *cache, E ** -0.5, torch.full((1,), keys, dtype=torch.int32, device=DEV))

    wants = [call(state(s)).clone() for s in range(3)]
    buffers = state(0)
    call(buffers)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(buffers)
    for s in (1, 2, 0):
        for b, x in zip(buffers, state(s)):
            b.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, wants[s])
    streams, states, got = [torch.cuda.Stream() for _ in range(2)], [state(1), state(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(call(states[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, wants[i + 1]) for i in range(2) for x in got[i])


@pytest.mark.parametrize("kernel,packed", [(None, False), (1, False), (2, False), (None, True), (4, True)])
def test_lengths_that_are_wrong_end(A, kernel, packed):
    """A length of two billion: the keys of the table are seen, the others have no page."""
    gen = torch.Generator().manual_seed(13)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, 8, 2, 16, 128) for _ in range(2))) for x in pair]
    table, huge, st = torch.arange(8, dtype=torch.int32).reshape(2, 4), 2 ** 31 - 1, status()
    q = torch.randn((1, 140, 8, 128) if packed else (1, 2, 8, 1, 128), generator=gen).bfloat16()
    loc = torch.full((1, 140) if packed else (1, 2, 1), huge, dtype=torch.int32)
    cu = torch.tensor([0, 139, 140], dtype=torch.int32) if packed else None
    lens = torch.tensor([[huge, huge]] if packed else [huge], dtype=torch.int32)
    seen = paged(A, q, torch.clamp(loc, max=63), torch.clamp(lens, max=64), cache, table, 0.1, cu=cu)[0]
    dc = dev(*cache)
    args = (*dev(q, loc), dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), table.to(DEV), 0.1, lens.to(DEV))
    if kernel is None:
        got = A.hogwild_varlen_paged_sdpa_q4(*args, cu.to(DEV), status=st) if packed else A.hogwild_paged_sdpa_q4(*args, status=st)
    else:
        from inference_lib_b200 import _cabi
        got = torch.empty((140, 8, 128) if packed else (2, 8, 1, 128), dtype=q.dtype, device=DEV)
        x, keep = _cabi.bind_paged_q4(out=got, queries=args[0], locations=args[1], key_cache=args[2], value_cache=args[3], key_scales=args[4],
                                      value_scales=args[5], block_table=args[6], scale=0.1, fragment_lengths=args[8],
                                      cu_seqlens_q=cu.to(DEV) if packed else None, kernel=kernel, status=st)
        assert _cabi.launch_paged_q4(x, torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
    assert int(st) == 1024
    torch.testing.assert_close(got.reshape(seen.shape).float(), seen.float(), rtol=2 * 2.0 ** -8, atol=2.0 ** -9)      # (other kernels: a rounding apart)


@pytest.mark.parametrize("kernel", KERNELS)
def test_lengths_below_zero_are_none(A, kernel):
    gen = torch.Generator().manual_seed(17)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, 8, 2, 16, 128) for _ in range(2))) for x in pair]
    table, st = torch.arange(8, dtype=torch.int32).reshape(4, 2), status()
    q = torch.randn(1, 6, 8, 128, generator=gen).bfloat16()
    loc = torch.tensor([[30, 31, 31, 2 ** 31 - 1, -2 ** 31, 31]], dtype=torch.int32)
    cu, lens = torch.tensor([0, 2, 3, 5, 6], dtype=torch.int32), torch.tensor([[-2 ** 31, -2 ** 31 + 1, -7, 32]], dtype=torch.int32)
    got, exact = paged(A, q, loc, lens, cache, table, 0.1, cu=cu, st=st, kernel=kernel)
    q4_util.check(got, exact)
    assert bool((got[:5] == 0).all()) and bool((got[5] != 0).any()) and int(st) == 0


def test_refusals_of_the_operators(A):
    gen = torch.Generator().manual_seed(9)
    kc, vc, ks, vs = dev(*empty_cache(gen, 4, 2, 16, 64, 64))
    ks, vs = ks.view(E4M3), vs.view(E4M3)
    table = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    x = torch.randn(2, 2, 3, 64, device=DEV).half()
    q, loc, flen = torch.randn(1, 2, 4, 1, 64, device=DEV).half(), torch.zeros(1, 2, 1, dtype=torch.int32, device=DEV), lens[:1]
    for bad in [dict(key_cache=kc.to(torch.int8)), dict(key_scales=ks.view(torch.uint8)), dict(key_scales=ks[:, :1]), dict(value_cache=vc[..., :16]),
                dict(block_table=table.long()), dict(key_unit=0.3), dict(value_unit=0.0), dict(block_table=table.cpu()),
                dict(value_scales=vs.transpose(0, 1)), dict(status=torch.zeros(1, device=DEV))]:
        cache = dict(key_cache=kc, value_cache=vc, key_scales=ks, value_scales=vs, block_table=table)
        cache.update(bad)
        with pytest.raises(RuntimeError):
            A.copy_to_blocks_q4(x, x, seq_lengths=lens, **cache)
        with pytest.raises(RuntimeError):
            A.copy_from_blocks_q4(first_rows=lens, rows=2, **cache)
        with pytest.raises(RuntimeError):
            A.hogwild_paged_sdpa_q4(q, loc, scale=0.1, fragment_lengths=flen, **cache)
    cache = (kc, vc, ks, vs, table)
    for k, v, more in [(x, x[..., :32], {}), (x, x.float(), {}), (x[:1], x[:1], {}), (x, x, dict(new_rows=lens[:1])), (x, x, dict(cu_seqlens=lens)),
                       (x.double(), x.double(), {}), (x[:, :1], x[:, :1], {})]:
        with pytest.raises(RuntimeError):
            A.copy_to_blocks_q4(k, v, *cache, lens, **more)
    for qq, ll in [(q[..., :32], loc), (q, loc[:, :1]), (q[:, :1], loc), (q[:, :, :3], loc), (q, loc.long())]:
        with pytest.raises(RuntimeError):
            A.hogwild_paged_sdpa_q4(qq, ll, *cache, 0.1, flen)
    with pytest.raises(RuntimeError):
        A.hogwild_varlen_paged_sdpa_q4(q[0].transpose(0, 1).contiguous(), loc[0], *cache, 0.1, flen[None], lens[:1])
