"""The 4-bit paged operators at the ends of their range: scales, queries and scores that are no ordinary numbers, long sequences."""
import numpy as np
import pytest
import torch

from tests import q4_util
from tests.test_gpu_q4 import DEV, E4M3, KERNELS, A, dev, paged, skip_unless_eligible, status  # noqa: F401

pytestmark = pytest.mark.gpu


def small_cache(seed, blocks, Hkv, bs, E, units=(1.0, 1.0)):
    gen = torch.Generator().manual_seed(seed)
    (kc, ks), (vc, vs) = q4_util.random_cache(gen, blocks, Hkv, bs, E, units[0]), q4_util.random_cache(gen, blocks, Hkv, bs, E, units[1])
    return [kc, vc, ks, vs], gen


@pytest.mark.parametrize("dtype,E,G", [(torch.bfloat16, 128, 4), (torch.float16, 64, 12), (torch.float32, 128, 2)])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("kernel", KERNELS[:3])
def test_a_scale_that_is_no_number(A, dtype, E, G, scale, kernel):
    """NaN for every row that sees a key (inf - inf, 0 * inf), zeros for the others."""
    skip_unless_eligible(kernel, dtype, E, E)
    cache, gen = small_cache(41, 8, 2, 16, E)
    table = torch.arange(8, dtype=torch.int32).reshape(2, 4)
    q = torch.randn(1, 2, 2 * G, 2, E, generator=gen).to(dtype)
    loc = torch.tensor([[[40, -1], [0, 63]]], dtype=torch.int32)
    got, exact = paged(A, q, loc, torch.tensor([50], dtype=torch.int32), cache, table, scale, kernel=kernel)
    q4_util.check(got, exact)
    assert bool(got[[0, 2, 3]].isnan().all()) and bool((got[1] == 0).all())
    # packed, and enough of it for the kernel that chunks take
    counts = [150, 1]
    q = torch.randn(1, 151, 2 * G, E, generator=gen).to(dtype)
    loc = torch.full((1, 151), 40, dtype=torch.int32)
    loc[0, 7:20] = -1
    wide = torch.full((2, 300), -1, dtype=torch.int32)
    wide[:, :4] = table
    got, exact = paged(A, q, loc, torch.tensor([[50, 50]], dtype=torch.int32), cache, wide, scale, cu=torch.tensor([0, 150, 151], dtype=torch.int32), kernel=kernel)
    q4_util.check(got, exact)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kernel", KERNELS)
def test_fragments_whose_queries_differ_in_size(A, dtype, kernel):
    """What a row holds for a fragment that it does not see does not reach what it sees, however large; and where it sees both, each counts as it is."""
    cache, gen = small_cache(43, 24, 2, 16, 128)
    table = torch.arange(24, dtype=torch.int32).reshape(2, 12)
    T, cu = 200, torch.tensor([0, 199, 200], dtype=torch.int32)
    large = 1e30 if dtype == torch.bfloat16 else 6e4
    q = torch.randn(3, T, 8, 128, generator=gen)
    loc = torch.from_numpy(np.random.default_rng(43).integers(-1, 190, (3, T)).astype(np.int32))
    lens = torch.tensor([[192, 192], [192, 0], [150, 192]], dtype=torch.int32)
    blind = torch.arange(T) % 3 == 0
    loc[0, blind], q[0, blind] = -1, large                       # in front of what it sees
    loc[2, 50:60], q[2, 50:60] = -5, -large                      # behind it
    q[1, 199] = large                                            # a length of zero
    q[1, 100:110], q[2, 100:110] = q[1, 100:110] * 2.0 ** -9, q[2, 100:110] * 2.0 ** 2       # seen, of different sizes
    got, exact = paged(A, q.to(dtype), loc, lens, cache, table, 128 ** -0.5, cu=cu, kernel=kernel)
    # (`large` stands behind no visible key: the bound on the scores is that of the others)
    q4_util.check(got, exact)


@pytest.mark.parametrize("dtype,E", [(torch.bfloat16, 128), (torch.float16, 128), (torch.float16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("F", [1, 2])
def test_infinite_queries_are_nan_by_every_kernel(A, dtype, E, kernel, F):
    """A row whose query holds an infinity is NaN where it sees a key, whichever sign its scores have; alone, in a chunk, over two fragments."""
    skip_unless_eligible(kernel, dtype, E, E, True, 16)
    cache, gen = small_cache(42, 24, 2, 16, E)
    table = torch.arange(24, dtype=torch.int32).reshape(2, 12)
    T, cu = 150, torch.tensor([0, 149, 150], dtype=torch.int32)
    q = torch.randn(F, T, 8, E, generator=gen).to(dtype)
    loc = torch.from_numpy(np.random.default_rng(42).integers(-1, 190, (F, T)).astype(np.int32))
    for row, value, seen in ((3, float("inf"), 0), (4, -float("inf"), 0), (60, float("inf"), 150), (61, -float("inf"), 150), (100, float("nan"), 5),
                             (149, -float("inf"), 0), (90, float("inf"), -1), (91, float("nan"), -1)):
        q[F - 1, row, :, 3] = value
        loc[F - 1, row] = seen
        if F == 2:
            loc[0, row] = 20 if row != 149 else -1               # (the other fragment's rows are ordinary ones)
    lens = torch.tensor([[192, 192]] * F, dtype=torch.int32)
    got, exact = paged(A, q, loc, lens, cache, table, E ** -0.5, cu=cu, kernel=kernel)
    bad = [3, 4, 60, 61, 100, 149]
    exact[0][bad] = np.nan
    q4_util.check(got, exact)
    assert bool(got[bad].isnan().all()) and not bool(got[[90, 91]].isnan().any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale,unit,size", [(1e-30, 2.0 ** -64, 1.0), (1e-30, 2.0 ** -28, 1.0), (1e-12, 2.0 ** -40, 1.0), (2e3, 2.0 ** -12, 0.5), (0.088, 2.0 ** -20, 10000.0),
                                             (1e20, 2.0 ** -63, 0.3), (1e-30, 2.0 ** 64, 0.1), (3e-4, 2.0 ** 20, 2.0 ** -10)])
def test_scales_and_units_of_a_chunk(A, dtype, scale, unit, size):
    """A chunk large enough for the kernel that chunks take by themselves, scale times unit from one end of its range to the other."""
    cache, gen = small_cache(44, 40, 2, 8, 128)                  # (codes and scales; what they stand for goes by the unit)
    W, width = 2, 480
    table = torch.full((W, width), -1, dtype=torch.int32)
    table[:, :20] = torch.randperm(40, generator=gen).to(torch.int32).reshape(W, 20)
    T, cu = 161, torch.tensor([0, 160, 161], dtype=torch.int32)
    assert (T - W) * 8 * width * 8 >= 4.5e6
    q = (torch.randn(1, T, 8, 128, generator=gen) * size).to(dtype)
    loc = torch.cat([torch.arange(160), torch.tensor([159])]).to(torch.int32)[None]
    loc[0, 5] = -1
    got, exact = paged(A, q, loc, torch.tensor([[160, 155]], dtype=torch.int32), cache, table, scale, (unit, 1.0), cu=cu)
    q4_util.check(got, exact)


def fine_tolerance(dtype, ref, weight, top, keys, vmax):
    """q4_util.tolerance with what the tensor-core kernels hold of small probabilities: the row's largest one stands at 2^7 or more of fp16's
    range, so a probability below 2^-14 is off by at most 2^-25 / 2^7 of the largest one (instead of 2^-25).  `keys`: per key that is as large."""
    p = 2 * (259 * 2.0 ** -23 * top + 4 * 2.0 ** -23) + 2 * keys * 2.0 ** -23 + (0 if dtype == torch.float32 else 2.0 ** -11)
    return q4_util.HALF_STEP[dtype] * np.abs(ref) + p * weight + keys * 2.0 ** -32 * vmax + (2.0 ** -25 if dtype == torch.float16 else 1e-30)


@pytest.mark.parametrize("dtype,E", [(torch.bfloat16, 128), (torch.float16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("G", [2, 12])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_small_probabilities_beside_large_ones(A, dtype, E, G, many, kernel):
    """One key, or one of every sixteen, has nearly all of a row's weight and values of zero: the output is what the others add up to, 2^-25 of it each."""
    skip_unless_eligible(kernel, dtype, E, E, True, 16)
    gen = torch.Generator().manual_seed(45)
    bs, blocks, keys, T, unit = 16, 20, 3000, 40, 1024.0
    k, v = torch.zeros(blocks, 1, bs, E), unit * (1 + torch.randint(0, 4, (blocks, 1, bs, E), generator=gen) * 0.5)
    heavy = slice(0, blocks if many else 1)
    k[heavy, 0, 3, 0], v[heavy, 0, 3] = 6.0, 0.0
    k[..., 16:] = torch.where(torch.rand(blocks, 1, bs, E - 16, generator=gen) < 0.5, 0.25, -0.25)
    (kc, ks), (vc, vs) = q4_util.quantise(k, 1.0), q4_util.quantise(v, unit)
    table = torch.from_numpy(np.random.default_rng(45).integers(1, blocks, (1, 188)).astype(np.int32))
    table[0, 5] = 0                                          # (key 83 is the heavy one, where there is one)
    q = torch.zeros(1, T, G, E)
    q[..., 0] = 25.5 * np.log(2) / 6.0 * 8
    q[..., 16:] = torch.randn(1, T, G, E - 16, generator=gen) * 0.5
    loc = torch.from_numpy(np.random.default_rng(46).integers(100, keys, (1, T)).astype(np.int32))
    loc[0, 0] = keys - 1
    got, exact = paged(A, q.to(dtype), loc, torch.tensor([[keys]], dtype=torch.int32), [kc, vc, ks, vs], table, 0.125, (1.0, unit),
                       cu=torch.tensor([0, T], dtype=torch.int32), kernel=kernel)
    ref, weight, top, _, vmax = exact
    assert 1e-4 < np.abs(ref).max() < 1.0
    # (at least six large ones among the first 101 keys: no more than 32 keys for each)
    far = np.abs(got.cpu().double().numpy() - ref) / fine_tolerance(dtype, ref, weight, top, 32 if many else keys, vmax)
    assert far.max() <= 1.0, f"{far.max():.2f} times the tolerance"


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 2.0 ** 16), (torch.bfloat16, 2.0 ** 27), (torch.bfloat16, 2.0 ** 70), (torch.float16, 2.0 ** 15)])
@pytest.mark.parametrize("E", [128, 64])
@pytest.mark.parametrize("G", [2, 12])
@pytest.mark.parametrize("kernel", KERNELS)
def test_scores_beyond_what_an_exponent_resolves(A, dtype, size, E, G, kernel):
    """Scores of 2^27 and far beyond, some below zero: the key with the largest one has all of the weight."""
    skip_unless_eligible(kernel, dtype, E, E, True, 16)
    gen, rng = torch.Generator().manual_seed(47), np.random.default_rng(47)
    bs, blocks, T = 16, 12, 140
    k = torch.zeros(blocks, 1, bs, E)
    k[..., 0] = torch.tensor([6.0, 4, 3, 2, 1.5, 1, 0.5, 0, -6])[torch.randint(0, 9, (blocks, 1, bs), generator=gen)]
    scales = 2.0 ** torch.randint(-3, 9, (blocks, 1, bs, 1), generator=gen)          # (powers of two times 1.5 at most: rows differ by a quarter or are equal)
    (kc, ks), (vc, vs) = q4_util.quantise(k * scales, 1.0), q4_util.random_cache(gen, blocks, 1, bs, E)
    table = torch.randperm(blocks, generator=gen).to(torch.int32)[None]
    q = torch.zeros(1, T, G, E)
    q[..., 0] = size
    q[0, ::3, :, 0] = -size
    loc = torch.from_numpy(rng.integers(0, 192, (1, T)).astype(np.int32))
    got, _ = paged(A, q.to(dtype), loc, torch.tensor([[192]], dtype=torch.int32), [kc, vc, ks, vs], table, 1.0, cu=torch.tensor([0, T], dtype=torch.int32), kernel=kernel)
    key = q4_util.sequence(kc, ks, 1.0, table[0], 192)[0][0, :, 0]
    val = q4_util.sequence(vc, vs, 1.0, table[0], 192)[0][0]
    for i in range(T):
        z = key[:int(loc[0, i]) + 1] * (-1 if i % 3 == 0 else 1)
        want = val[:len(z)][z == z.max()].mean(0)                # (equal keys share; the next one is 2^15 / 16 or more behind)
        assert np.abs(got[i].cpu().double().numpy() - want).max() <= (q4_util.HALF_STEP[dtype] + 2.0 ** -11 + 200 * 2.0 ** -23) * np.abs(val).max(), i


@pytest.mark.parametrize("size", [2.0 ** 10, 2.0 ** 60, 2.0 ** 100])
@pytest.mark.parametrize("first", [0, 1])
@pytest.mark.parametrize("G", [2, 12])
@pytest.mark.parametrize("kernel", KERNELS)
def test_fragments_whose_scores_lie_far_apart(A, size, first, G, kernel):
    """One fragment's scores are ordinary, the other's so large that they take all of the weight or none of it; equal ones share."""
    gen, rng = torch.Generator().manual_seed(48), np.random.default_rng(48)
    bs, blocks, T, E = 16, 24, 140, 128
    k = torch.zeros(blocks, 1, bs, E)
    k[..., 0] = torch.tensor([6.0, 3, 1, 0.5, 0, -1, -6])[torch.randint(0, 7, (blocks, 1, bs), generator=gen)]
    k[:14, ..., 0] = -k[:14, ..., 0].abs()                       # (rows that see few keys: none above zero)
    (kc, ks), (vc, vs) = q4_util.quantise(k, 1.0), q4_util.random_cache(gen, blocks, 1, bs, E)
    table = torch.arange(blocks, dtype=torch.int32)[None]
    q = torch.zeros(2, T, G, E)
    q[first, ..., 0], q[1 - first, ..., 0] = size, 0.25
    loc = torch.from_numpy(rng.integers(-1, blocks * bs, (2, T)).astype(np.int32))
    lens = torch.full((2, 1), blocks * bs, dtype=torch.int32)
    got, _ = paged(A, q.bfloat16(), loc, lens, [kc, vc, ks, vs], table, 1.0, cu=torch.tensor([0, T], dtype=torch.int32), kernel=kernel)
    key, val = (q4_util.sequence(*x, 1.0, table[0], blocks * bs)[0][0] for x in ((kc, ks), (vc, vs)))
    for i in range(T):
        n = [int(x) + 1 for x in loc[:, i]]
        z = np.concatenate([key[:n[f], 0] * (size if f == first else 0.25) for f in range(2)])
        if not len(z):
            assert bool((got[i] == 0).all())
            continue
        p = np.exp(z - z.max())
        want = (p[:, None] * np.concatenate([val[:x] for x in n])).sum(0) / p.sum()
        # the output's rounding, the probabilities' in fp16 and what 768 keys' sums and scores below 2^4 add in fp32
        assert np.abs(got[i].cpu().double().numpy() - want).max() <= (2.0 ** -8 + 2.0 ** -11 + 2 * 800 * 2.0 ** -23) * np.abs(val).max(), i


LONG = [
    # sequences of keys (one token each), Hkv, G, E, bs, kernel: what runs
    ([9000], 1, 4, 128, 16, 2),                    # shares of one unit: many partials, the merge step's second round
    ([40000], 1, 8, 64, 32, 2),
    ([70000, 33], 1, 12, 128, 16, 2),              # sixteen rows
    ([150001], 2, 2, 64, 64, 2),
    ([30000, 9000, 129], 2, 4, 128, 8, 2),         # rows looked up one by one
    ([1300003], 1, 2, 64, 64, 2),                  # more than 32 tiles of a share: the second window of page numbers
    ([4300] * 75, 4, 4, 128, 16, 2),               # units with a CTA each, 34 tiles
    ([2300] * 3 + [100] * 220, 4, 2, 64, 16, 2),   # four warps a CTA, 36 tiles
    ([5000, 4096, 4097], 1, 2, 128, 16, 1),        # CUDA cores
]


def long_exact(q, lens, cache, table, scale, bs):
    """Output and what bounds its error, like q4_util.attention, for single tokens that see all keys, with whole arrays."""
    kc, vc, ks, vs = cache
    K, V = q4_util.values(kc, ks, 1.0), q4_util.values(vc, vs, 1.0)
    W, Hq, E = q.shape
    Hkv = kc.shape[1]
    out, weight, top = np.zeros((W, Hq, V.shape[-1])), np.zeros((W, Hq, V.shape[-1])), 0.0
    qd = q.double().numpy().reshape(W, Hkv, Hq // Hkv, E)
    for w, n in enumerate(lens):
        pages = table[w, :-(-n // bs)].numpy()
        k, v = (x[pages].transpose(1, 0, 2, 3).reshape(Hkv, -1, E)[:, :n] for x in (K, V))
        z = np.einsum("hge,hle->hgl", qd[w], k) * scale
        top = max(top, float(np.einsum("hge,hle->hgl", np.abs(qd[w]), np.abs(k)).max() * scale))
        p = np.exp(z - z.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        out[w], weight[w] = (np.einsum("hgl,hle->hge", p, x).reshape(Hq, E) for x in (v, np.abs(v)))
    return out, weight, top, max(lens), float(np.abs(V).max())


@pytest.mark.parametrize("case", LONG, ids=[str(i) for i in range(len(LONG))])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_sequences(A, case, dtype):
    """Few pages under many table entries; a loud key now and then, so that the rows' references move."""
    lens, Hkv, G, E, bs, kernel = case
    gen, rng = torch.Generator().manual_seed(sum(lens)), np.random.default_rng(sum(lens))
    W, blocks, width = len(lens), 53, -(-max(lens) // bs)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, blocks, Hkv, bs, E) for _ in range(2))) for x in pair]
    table = torch.from_numpy(rng.integers(0, blocks - 1, (W, width)).astype(np.int32))
    cache[2][blocks - 1] += 12                               # (a page of keys that are larger by half an exponent: far back, once)
    table[:, width * 3 // 4] = blocks - 1
    q = torch.randn(1, W, Hkv * G, 1, E, generator=gen).to(dtype)
    exact = long_exact(q[0, :, :, 0], lens, cache, table, E ** -0.5, bs)
    dc = dev(*cache)
    from inference_lib_b200 import _cabi
    out = torch.full((W, Hkv * G, E), float("nan"), dtype=dtype, device=DEV)
    ints = dev(torch.tensor([[n - 1 for n in lens]], dtype=torch.int32), table, torch.tensor([lens], dtype=torch.int32), torch.arange(W + 1, dtype=torch.int32))
    x, keep = _cabi.bind_paged_q4(out=out, queries=q[:, :, :, 0].contiguous().to(DEV), locations=ints[0], key_cache=dc[0], value_cache=dc[1], key_scales=dc[2].view(E4M3),
                                  value_scales=dc[3].view(E4M3), block_table=ints[1], scale=E ** -0.5, fragment_lengths=ints[2], cu_seqlens_q=ints[3], kernel=kernel)
    keep[0].fill_(0xFF)
    assert _cabi.launch_paged_q4(x, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    q4_util.check(out, exact)
    # the fixed layout, where every sequence has as many
    if len(set(lens)) == 1:
        got = A.hogwild_paged_sdpa_q4(q.to(DEV), ints[0][..., None], dc[0], dc[1], dc[2].view(E4M3), dc[3].view(E4M3), ints[1], E ** -0.5, ints[2][0, :1])
        q4_util.check(got[:, :, 0], exact)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,keys", [([130], 9000), ([33, 257, 1], 5000)])
def test_chunks_behind_long_sequences(A, dtype, counts, keys):
    """A chunk's rows at the end of thousands of keys, on the kernel that chunks take."""
    gen, rng = torch.Generator().manual_seed(keys), np.random.default_rng(keys)
    Hkv, G, E, bs, blocks, W = 1, 4, 128, 16, 53, len(counts)
    cache = [x for pair in zip(*(q4_util.random_cache(gen, blocks, Hkv, bs, E) for _ in range(2))) for x in pair]
    table = torch.from_numpy(rng.integers(0, blocks, (W, -(-keys // bs))).astype(np.int32))
    rows = [(w, keys - n + i) for w, n in enumerate(counts) for i in range(n)]
    q = torch.randn(1, len(rows), Hkv * G, E, generator=gen).to(dtype)
    cu = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
    loc = torch.tensor([[p for _, p in rows]], dtype=torch.int32)
    st = status()
    got = torch.empty(len(rows), Hkv * G, E, dtype=dtype, device=DEV)
    from inference_lib_b200 import _cabi
    dc = dev(*cache)
    x, keep = _cabi.bind_paged_q4(out=got, queries=q.to(DEV), locations=loc.to(DEV), key_cache=dc[0], value_cache=dc[1], key_scales=dc[2].view(E4M3),
                                  value_scales=dc[3].view(E4M3), block_table=table.to(DEV), scale=E ** -0.5, fragment_lengths=torch.tensor([[keys] * W], dtype=torch.int32, device=DEV),
                                  cu_seqlens_q=cu.to(DEV), kernel=4, status=st)
    assert _cabi.launch_paged_q4(x, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    some = sorted({0, 1, len(rows) - 1, *(int(i) for i in rng.integers(0, len(rows), 12))})
    exact = long_exact(q[0, some], [rows[i][1] + 1 for i in some], cache, table[[rows[i][0] for i in some]], E ** -0.5, bs)
    q4_util.check(got[some], exact)
    assert int(st) == 0 and bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("G", [4, 16])
@pytest.mark.parametrize("kernel", [1, 2, 4])
@pytest.mark.parametrize("power", [20, 24, 25, 26, 27, 28, 30])
def test_scores_a_few_steps_apart(A, dtype, G, kernel, power):
    """Scores of 2^power, where fp32 has steps of 2 to 128: 128 keys of them, then 128 that are j steps larger, j by row."""
    gen = torch.Generator().manual_seed(49)
    Hkv, E, bs, T, unit = 8, 128, 16, 300, 2.0 ** (power - 25)
    k = torch.zeros(16, Hkv, bs, E)
    k[..., 0], k[..., 1], k[8:, ..., 16], k[8:, ..., 17] = 1024 * unit, 1536 * unit, unit, 1.5 * unit       # (6 times the scale beside 4 times it: exact)
    (kc, ks), (vc, vs) = q4_util.quantise(k, unit), q4_util.random_cache(gen, 16, Hkv, bs, E)
    assert np.array_equal(q4_util.values(kc, ks, unit), k.double().numpy())
    step = 2.0 ** (power - 23)
    j = torch.arange(T) % 50
    q = torch.zeros(1, T, Hkv * G, E)
    q[..., 0], q[..., 16] = 2.0 ** 15, (j * step / unit)[None, :, None]
    table, loc = torch.arange(16, dtype=torch.int32)[None], torch.full((1, T), 255, dtype=torch.int32)
    dc = dev(kc, vc, ks, vs)
    out = torch.full((T, Hkv * G, E), 7.0, dtype=dtype, device=DEV)
    from inference_lib_b200 import _cabi
    x, keep = _cabi.bind_paged_q4(out=out, queries=q.to(dtype).to(DEV), locations=loc.to(DEV), key_cache=dc[0], value_cache=dc[1], key_scales=dc[2].view(E4M3),
                                  value_scales=dc[3].view(E4M3), block_table=table.to(DEV), scale=float(np.log(2)), key_unit=unit,
                                  fragment_lengths=torch.tensor([[256]], dtype=torch.int32, device=DEV), cu_seqlens_q=torch.tensor([0, T], dtype=torch.int32, device=DEV),
                                  kernel=kernel)
    assert _cabi.launch_paged_q4(x, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    # (log2 e * ln 2 is 1 in fp32, and every score is a number of it)
    v = q4_util.sequence(vc, vs, 1.0, table[0], 256)[0].repeat(G, 0)                # [Hq,256,E]
    less = 2.0 ** -(j.double().numpy() * step)[:, None, None]
    want = (v[None, :, :128].sum(2) * less + v[None, :, 128:].sum(2)) / (128 * (1 + less))
    assert np.abs(out.cpu().double().numpy() - want).max() <= (q4_util.HALF_STEP[dtype] + 2.0 ** -11 + 260 * 2.0 ** -23) * np.abs(v).max()
