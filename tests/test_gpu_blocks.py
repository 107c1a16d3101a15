"""Pages of a paged cache on the GPU: every number and every byte as the sequential definition has it; and all paged operators together."""
import numpy as np
import pytest
import torch

from tests import q4_util
from tests.test_gpu_q4 import DEV, E4M3, A, dev, status  # noqa: F401

pytestmark = pytest.mark.gpu


def pool(rng, blocks, bs, width, lengths, share=0):
    """A consistent state: tables whose pages are counted; `share` rows at the end hold the pages of the first ones."""
    table, refs, order, at = [], [0] * blocks, list(rng.permutation(blocks)), 0
    for w, n in enumerate(lengths):
        pages = -(-n // bs)
        if w >= len(lengths) - share:
            row = table[w - (len(lengths) - share)][:pages]
        else:
            row = [int(p) for p in order[at:at + pages]]
            at += pages
        table.append(row + [-1] * (width - len(row)))
        for p in row:
            refs[p] += 1
    return refs, table


def some_caches(rng, blocks):
    """16-bit rows, codes and scales, a page that is no multiple of 16 bytes, and one of more than a piece."""
    return [torch.from_numpy(rng.integers(0, 256, (blocks, *shape)).astype(np.uint8)) for shape in ((2, 8, 64), (2, 8, 8), (7,), (3, 1500), (16,))]


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def run_step(A, refs, table, lengths, source, new, bs, caches, out=None):
    dc, st = dev(*caches), status()
    want_caches = [c.clone() for c in caches]
    want = q4_util.step_blocks(refs, table, lengths, source, new, bs, want_caches)
    args = [ints(refs), ints(table), ints(lengths)]
    got = A.step_blocks(*args, dc, bs, source=None if source is None else ints(source), new_tokens=None if new is None else ints(new),
                        out=None if out is None else out(args), status=st)
    for g, w, name in zip(got, want, ("refs", "table", "lengths", "room")):
        assert g.tolist() == w, name
    assert int(st) == want[4]
    for g, w in zip(dc, want_caches):
        assert torch.equal(g.cpu(), w)
    return want


@pytest.mark.parametrize("blocks", [61, 1500, 9000])
@pytest.mark.parametrize("seed", range(4))
def test_steps_of_a_batch(A, blocks, seed):
    """Forks, moves, frees and growth in turn, as long as there are pages and beyond."""
    rng = np.random.default_rng(100 * blocks + seed)
    bs, width = (4, 9) if blocks == 61 else (8, 40)
    W = 6 if blocks == 61 else 30
    lengths = [int(n) for n in rng.integers(0, min(width * bs, 30), W)]
    refs, table = pool(rng, blocks, bs, width, lengths, share=0)
    refs[[p for p in range(blocks) if refs[p] == 0][0]] = 1                 # somebody keeps a page without a row
    caches = some_caches(rng, blocks)
    for _ in range(4):
        W = max(1, len(lengths) + int(rng.integers(-2, 3)))
        source = [int(x) for x in rng.integers(-1, len(lengths), W)] if rng.random() < 0.7 else None
        W = len(lengths) if source is None else W
        new = [int(x) for x in rng.integers(0, 2 * bs, W)] if rng.random() < 0.8 else None
        refs, table, lengths, room, _ = run_step(A, refs, table, lengths, source, new, bs, caches)
        lengths = [n + r for n, r in zip(lengths, room)]


def test_shared_last_pages(A):
    """Every writer of a shared page but the last holder takes a copy; somebody who does not write, or a count without a row, keeps it."""
    rng = np.random.default_rng(1)
    caches = some_caches(rng, 40)
    refs, table = pool(rng, 40, 8, 6, [13, 8, 21])
    run_step(A, refs, table, [13, 8, 21], [0, 0, 0, 1, 1, 2, 2, 2], [1, 1, 1, 1, 1, 0, 9, 4], 8, caches)
    refs[table[0][1]] += 1
    run_step(A, refs, table, [13, 8, 21], [0, 0, 2, 0, -1], [1, 1, 1, 30, 3], 8, caches)
    run_step(A, refs, table, [13, 8, 21], [2, 2, 2, 2], None, 8, caches)                              # a fork alone copies nothing


def test_a_pool_that_runs_dry(A):
    rng = np.random.default_rng(2)
    caches = some_caches(rng, 12)
    refs, table = pool(rng, 12, 4, 8, [9, 6, 7])
    for new in ([1, 30, 0], [3, 3, 40], [20, 1, 1], [0, 0, 0]):
        run_step(A, refs, table, [9, 6, 7], None, new, 4, caches)
        run_step(A, refs, table, [9, 6, 7], [1, 1, 0, 2], new + [5], 4, caches)
    run_step(A, [0] * 12, [[-1] * 8], [0], None, [48], 4, caches)                                     # more than the table is wide
    run_step(A, [0] * 12, [[-1] * 12], [0], None, [48], 4, caches)                                    # the whole pool
    run_step(A, [0] * 12, [[-1] * 13], [0], None, [49], 4, caches)


def test_tables_that_are_wrong(A):
    rng = np.random.default_rng(3)
    caches = some_caches(rng, 16)
    table = [[3, 99, -1, 7], [-1, -1, -1, -1], [5, 6, -8, -1], [1, 2, 4, 8]]
    refs = [0] * 16
    for row in table:
        for p in row:
            if 0 <= p < 16:
                refs[p] += 1
    run_step(A, refs, table, [9, 5, -3, 99], None, [1, 1, 1, 1], 4, caches)
    run_step(A, refs, table, [9, 5, -3, 99], [3, 0, 9, -4, 2], [1, -5, 1, 1, 6], 4, caches)


def test_a_step_in_place(A):
    rng = np.random.default_rng(4)
    caches = some_caches(rng, 64)
    refs, table = pool(rng, 64, 8, 10, [17, 30, 17], share=1)
    run_step(A, refs, table, [17, 30, 17], None, [9, 1, 2], 8, caches, out=lambda a: (a[0], a[1], a[2], ints([7] * 3)))
    # a row that held more than its length fills gives it back
    refs, table = pool(rng, 64, 8, 10, [60, 30])
    run_step(A, refs, table, [20, 30], None, [1, 0], 8, caches, out=lambda a: (a[0], a[1], a[2], ints([7] * 2)))
    run_step(A, refs, table, [20, 30], [1, 0, 0], [1, 0, 3], 8, caches, out=lambda a: (a[0], torch.empty(3, 10, dtype=torch.int32, device=DEV), ints([0] * 3), ints([0] * 3)))


def test_one_row_and_many(A):
    rng = np.random.default_rng(5)
    run_step(A, [1, 0], [[0]], [1], None, [1], 4, [])
    run_step(A, [1, 0], [[0]], [1], [0, 0], [1, 1], 4, [torch.zeros(2, 3, dtype=torch.uint8)])
    W = 2500                                                                                          # more rows than a CTA has threads
    lengths = [int(n) for n in rng.integers(0, 40, W)]
    refs, table = pool(rng, 30000, 8, 6, lengths, share=400)
    lengths[W - 400:] = lengths[:400]
    refs, table = pool(rng, 30000, 8, 6, lengths, share=400)
    run_step(A, refs, table, lengths, None, [int(x) for x in rng.integers(0, 9, W)], 8, [torch.arange(30000 * 16, dtype=torch.int32).reshape(30000, 16)])


@pytest.mark.parametrize("W", [1, 300, 1025, 2049])
def test_everybody_forks_from_one(A, W):
    """One last page that many rows write: all but the last holder take a copy."""
    rng = np.random.default_rng(W)
    refs, table = pool(rng, 2 * W + 20, 8, 4, [13, 5])
    run_step(A, refs, table, [13, 5], [0] * W, [int(x) for x in rng.integers(0, 3, W)], 8, some_caches(rng, 2 * W + 20))


def test_more_caches_than_a_launch_takes(A):
    rng = np.random.default_rng(6)
    caches = [torch.from_numpy(rng.integers(0, 99, (24, 5)).astype(np.int32)) for _ in range(150)]
    refs, table = pool(rng, 24, 4, 4, [6, 7])
    run_step(A, refs, table, [6, 7], [0, 0, 1, 1], [1, 1, 1, 1], 4, caches)
    run_compact(A, refs, table, caches)


def run_compact(A, refs, table, caches, in_place=False):
    dc, st = dev(*caches), status()
    want_caches = [c.clone() for c in caches]
    want = q4_util.compact_blocks(refs, table, want_caches)
    args = [ints(refs), ints(table)]
    got = A.compact_blocks(*args, dc, out=(args[0], args[1], torch.empty_like(args[0])) if in_place else None, status=st)
    for g, w, name in zip(got, want, ("refs", "table", "moved")):
        assert g.tolist() == w, name
    assert int(st) == want[3]
    n = sum(r != 0 for r in refs)
    for g, w in zip(dc, want_caches):
        assert torch.equal(g.cpu(), w)
    assert all(r != 0 for r in want[0][:n]) and not any(want[0][n:])


@pytest.mark.parametrize("blocks,lengths", [(1, [3]), (2, [0]), (61, [9, 0, 17, 4]), (3000, [100, 80, 3, 77]), (20011, [2000, 1000, 1, 5000]),
                                            (64, [64 * 8])])
@pytest.mark.parametrize("in_place", [False, True])
def test_compaction(A, blocks, lengths, in_place):
    rng = np.random.default_rng(blocks)
    bs = 8
    refs, table = pool(rng, blocks, bs, max(-(-n // bs) for n in lengths) + 1, lengths + lengths[:1], share=1)
    if blocks > 60:
        refs[next((p for p in range(blocks - 1, 0, -1) if refs[p] == 0), 0)] += 1
    run_compact(A, refs, table, some_caches(rng, blocks) if blocks < 4000 else [torch.arange(blocks * 4).reshape(blocks, 4)], in_place)


def test_compaction_of_a_table_that_is_wrong(A):
    rng = np.random.default_rng(8)
    run_compact(A, [0, 2, 0, 0, 1, 0, 0, 1], [[4, 1, -1, 99], [7, 1, 3, -5]], some_caches(rng, 8))


def test_steps_in_a_graph(A):
    """Captured once, replayed on what the buffers then hold."""
    rng = np.random.default_rng(9)
    caches = some_caches(rng, 200)
    lengths = [13, 40, 7]
    refs, table = pool(rng, 200, 8, 20, lengths)
    state = [ints(refs), ints(table), ints(lengths)]
    source, new, room = ints([0, 1, 2]), ints([0, 0, 0]), ints([0] * 3)
    out = [torch.empty_like(x) for x in state] + [room]
    dc = dev(*caches)
    A.step_blocks(*state, dc, 8, source=source, new_tokens=new, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        A.step_blocks(*state, dc, 8, source=source, new_tokens=new, out=out)
    for s, n in (([0, 0, 1], [3, 3, 30]), ([2, 1, 1], [1, 9, 1]), ([1, -1, 0], [0, 8, 1])):
        source.copy_(ints(s))
        new.copy_(ints(n))
        want_caches = [c.cpu() for c in dc]
        want = q4_util.step_blocks(refs, table, lengths, s, n, 8, want_caches)
        graph.replay()
        torch.cuda.synchronize()
        assert [x.tolist() for x in out] == list(want[:4])
        assert all(torch.equal(g.cpu(), w) for g, w in zip(dc, want_caches))
        refs, table, room_now = want[0], want[1], want[3]
        lengths = [a + b for a, b in zip(want[2], room_now)]
        for x, y in zip(state, (refs, table, lengths)):
            x.copy_(ints(y))


def test_refusals(A):
    refs, table, lengths = ints([1, 0, 0]), ints([[0, -1]]), ints([3])
    cache = torch.zeros(3, 4, device=DEV)
    for bad in [dict(caches=[cache[:2]]), dict(caches=[cache.t().contiguous().t()]), dict(caches=[cache.cpu()]), dict(block_size=0),
                dict(source=ints([[0]])), dict(source=torch.zeros(1, device=DEV)), dict(new_tokens=ints([1, 1])), dict(new_tokens=ints([1]).long()),
                dict(seq_lengths=ints([3, 3])), dict(block_refs=refs.long()), dict(block_table=table[0]), dict(source=ints([]))]:
        call = dict(block_refs=refs, block_table=table, seq_lengths=lengths, caches=[cache], block_size=4)
        call.update(bad)
        with pytest.raises(RuntimeError):
            A.step_blocks(**call)
    with pytest.raises(RuntimeError):                        # rows that change places cannot do so in place
        A.step_blocks(refs, table, lengths, [cache], 4, source=ints([0]), out=(refs, table, ints([0]), ints([0])))
    with pytest.raises(RuntimeError):
        A.compact_blocks(refs, table, [cache], out=(refs, table, refs))
    with pytest.raises(RuntimeError):
        A.compact_blocks(refs.cpu(), table, [cache])
    assert refs.tolist() == [1, 0, 0] and table.tolist() == [[0, -1]]


# ---- all of it together -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,E,bs", [(torch.bfloat16, 128, 16), (torch.float16, 64, 8)])
def test_a_batch_from_prompt_to_the_end(A, dtype, E, bs):
    """Two layers' 4-bit caches of one pool: prompts come in packed, are answered several ways, sequences end, the pool is compacted; after
    every step each row attends to exactly the tokens of its own history, quantised."""
    gen, rng = torch.Generator().manual_seed(11), np.random.default_rng(11)
    Hkv, G, blocks, width, layers = 2, 4, 70, 12, 2
    caches = [[torch.zeros(blocks, Hkv, bs, n, dtype=torch.uint8, device=DEV) for n in (E // 2, E // 2, E // 16, E // 16)] for _ in range(layers)]
    parts = [[c[0], c[1], c[2].view(E4M3), c[3].view(E4M3)] for c in caches]
    flat = [t for c in parts for t in c]
    refs, table, lengths = ints([0] * blocks), ints([[-1] * width]), ints([0])
    history = [[[] for _ in range(layers)]]                   # per row and layer: (key codes, scales, value codes, scales) of every token
    plan = [([0, -1, 0], [21, 2 * bs, 3]), ([0, 0, 1, 2, 0], [1, 1, 1, 1, 1]), (None, [1] * 5), ([3, 1, 4, 4], [2, 1, 1, 5]), ("compact", None),
            ([0, 1, 2, 3, 3], [1, 1, 1, 1, 1]), (None, [1, 0, 3, 1, bs])]
    st = status()
    for source, new in plan:
        if source == "compact":
            refs, table, moved = A.compact_blocks(refs, table, flat, status=st)
            live = int((refs > 0).sum())
            assert bool((refs[:live] > 0).all())
            continue
        W = len(new)
        refs, table, lengths, room = A.step_blocks(refs, table, lengths, flat, bs, source=None if source is None else ints(source),
                                                   new_tokens=ints(new), status=st)
        assert room.tolist() == new
        rows = list(range(W)) if source is None else source
        history = [[list(history[u][x]) if u >= 0 else [] for x in range(layers)] for u in rows]
        cu = ints([0] + list(np.cumsum(new)))
        now = ints([len(h[0]) + n for h, n in zip(history, new)])
        loc = torch.cat([torch.arange(len(h[0]), len(h[0]) + n) for h, n in zip(history, new)]).to(torch.int32)[None].to(DEV)
        for x in range(layers):
            k, v = (torch.randn(sum(new), Hkv, E, generator=gen).to(dtype) for _ in range(2))
            q = torch.randn(1, sum(new), Hkv * G, E, generator=gen).to(dtype)
            A.copy_to_blocks_q4(*dev(k, v), *parts[x], table, lengths, cu_seqlens=cu, new_rows=room, status=st)
            got = A.hogwild_varlen_paged_sdpa_q4(q.to(DEV), loc, *parts[x], table, E ** -0.5, now[None], cu, status=st)
            (kc, ks), (vc, vs) = q4_util.quantise(k, 1.0), q4_util.quantise(v, 1.0)
            for w in range(W):
                history[w][x] += [(kc[i], ks[i], vc[i], vs[i]) for i in range(int(cu[w]), int(cu[w + 1]))]
            # the same histories as one page per token
            own = [[t[n] for h in history for t in h[x]] for n in range(4)]
            one = [torch.stack(o)[:, :, None].contiguous() for o in (own[0], own[2], own[1], own[3])]
            starts = np.cumsum([0] + [len(h[x]) for h in history])
            most = max(len(h[x]) for h in history)
            plain_table = torch.tensor([[int(starts[w]) + i if i < len(history[w][x]) else -1 for i in range(most)] for w in range(W)])
            exact = q4_util.attention(q, loc.cpu(), now.cpu()[None], one[0], one[1], one[2], one[3], plain_table, E ** -0.5, cu=cu.cpu())
            q4_util.check(got, exact)
        lengths = lengths + room
        held = [p for row in table.tolist() for p in row if p >= 0]
        assert [held.count(p) for p in range(blocks)] == refs.tolist()
    keys, vals = A.copy_from_blocks_q4(*parts[0], table, ints([0] * len(lengths)), int(lengths.max()), dtype=dtype)
    for w, h in enumerate(history):
        want = q4_util.values(torch.stack([t[0] for t in h[0]]), torch.stack([t[1] for t in h[0]]), 1.0)
        assert np.array_equal(keys[w, :, :len(h[0])].cpu().double().numpy(), want.transpose(1, 0, 2))
    refs, table, lengths, _ = A.step_blocks(refs, table, lengths, flat, bs, source=ints([-1]))          # everything goes back
    assert not bool(refs.any()) and lengths.tolist() == [0] and bool((table == -1).all()) and int(st) & ~1024 == 0


def test_caches_of_more_than_four_gigabytes(A):
    """Pages whose bytes begin behind 2^32: written, read, attended to by every kernel, copied and moved like pages in front."""
    gen = torch.Generator().manual_seed(31)
    Hkv, G, bs, E, W, width = 8, 4, 16, 128, 2, 10
    blocks = 2 ** 19 + 64                                                        # 8 KiB of codes a page
    small = [torch.zeros(W * width + 2, Hkv, bs, n, dtype=t, device=DEV) for n, t in ((E // 2, torch.uint8), (E // 2, torch.uint8), (E // 16, E4M3), (E // 16, E4M3))]
    large = [torch.empty(blocks, *c.shape[1:], dtype=c.dtype, device=DEV) for c in small]
    assert large[0].numel() > 2 ** 32
    near = torch.arange(W * width, dtype=torch.int32, device=DEV).reshape(W, width)
    far = blocks - 1 - near
    k, v = (torch.randn(W, Hkv, width * bs, E, generator=gen).bfloat16().to(DEV) for _ in range(2))
    start = ints([0] * W)
    for caches, table in ((small, near), (large, far)):
        A.copy_to_blocks_q4(k, v, *caches, table, start)
    for a, b in zip(small, large):
        assert torch.equal(a.view(torch.uint8)[near.flatten().long()], b.view(torch.uint8)[far.flatten().long()])
    for a, b in zip(*(A.copy_from_blocks_q4(*c, t, start, width * bs) for c, t in ((small, near), (large, far)))):
        assert torch.equal(a, b)
    from inference_lib_b200 import _cabi
    counts, lens = [130, 1], [150, 157]
    q = torch.randn(1, sum(counts), Hkv * G, E, generator=gen).bfloat16().to(DEV)
    loc = ints([[n - c + i for n, c in zip(lens, counts) for i in range(c)]])
    for kernel in (1, 2, 4):
        out = []
        for c, t in ((small, near), (large, far)):
            out.append(torch.empty_like(q[0]))
            x, keep = _cabi.bind_paged_q4(out=out[-1], queries=q, locations=loc, key_cache=c[0], value_cache=c[1], key_scales=c[2], value_scales=c[3],
                                          block_table=t, scale=0.1, fragment_lengths=ints([lens]), cu_seqlens_q=ints([0, 130, 131]), kernel=kernel)
            assert _cabi.launch_paged_q4(x, torch.cuda.current_stream().cuda_stream) == 0
            torch.cuda.synchronize()
        assert torch.equal(*out) and bool(out[0].isfinite().all())
    # blocks of eight rows (rows looked up one by one), the same bytes
    small8, large8 = ([t.view(t.shape[0] * 2, Hkv, 8, t.shape[3]) for t in c] for c in (small, large))
    near8, far8 = (torch.stack([2 * t, 2 * t + 1], -1).reshape(W, 2 * width) for t in (near, far))
    q1, loc1 = q[:, :W].reshape(1, W, Hkv * G, 1, E).contiguous(), ints([[[150], [157]]])
    assert torch.equal(*(A.hogwild_paged_sdpa_q4(q1, loc1, *c, t.int(), 0.1, ints([158])) for c, t in ((small8, near8), (large8, far8))))
    # a fork of a row whose last page lies far behind, onto a free page in front of it; then everything to the front
    refs = torch.zeros(blocks, dtype=torch.int32, device=DEV)
    refs[:blocks - 64] = 1                                                       # somebody else's
    refs[far.flatten().long()] = 1
    n = ints([width * bs - 3, 8])
    refs, table, n, room = A.step_blocks(refs, far.contiguous(), n, large, bs, source=ints([0, 0]), new_tokens=ints([1, 1]))
    copied = int(table[0, width - 1])
    assert room.tolist() == [1, 1] and copied == blocks - 64 and int(table[1, width - 1]) == int(far[0, width - 1])
    for c in large:
        assert torch.equal(c.view(torch.uint8)[copied], c.view(torch.uint8)[int(far[0, width - 1])])
    refs[:blocks - 64] = 0
    refs, table, moved = A.compact_blocks(refs, table, large)
    assert sorted(set(table[table >= 0].tolist())) == list(range(width + 1)) and int((refs != 0).sum()) == width + 1
    for a, b in zip(A.copy_from_blocks_q4(*small, near[:1], start[:1], width * bs - 3), A.copy_from_blocks_q4(*large, table[:1], start[:1], width * bs - 3)):
        assert torch.equal(a, b)
