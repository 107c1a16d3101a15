"""Page bookkeeping at the ends of its range, and together with the 16-bit paged operators."""
import numpy as np
import pytest
import torch

from tests.test_gpu_blocks import ints, pool, run_step, some_caches
from tests.test_gpu_q4 import DEV, A, dev, status  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_sixteen_bit_append_drops_rows_without_a_page(A, dtype):
    gen = torch.Generator().manual_seed(51)
    B, Hkv, S, E, Ev, bs, blocks = 5, 2, 6, 64, 32, 4, 12
    table = torch.tensor([[0, -1, 2], [3, 12, 4], [5, 6, 7], [1, 8, -1], [-7, 1 << 30, 9]], dtype=torch.int32)
    lengths = torch.tensor([1, 2, 9, -2, 3], dtype=torch.int32)              # a hole, a page outside, behind the table, in front of it
    k, v = torch.randn(B, Hkv, S, E, generator=gen).to(dtype), torch.randn(B, Hkv, S, Ev, generator=gen).to(dtype)
    for counts in (None, torch.tensor([3, 2, 0, -1, 6], dtype=torch.int32)):
        kc, vc = torch.randn(blocks, Hkv, bs, E, generator=gen).to(dtype), torch.randn(blocks, Hkv, bs, Ev, generator=gen).to(dtype)
        # 64 pages of canaries on either side of each cache
        around = [torch.full((blocks + 128, *c.shape[1:]), 3.0, dtype=dtype, device=DEV) for c in (kc, vc)]
        mine = [a[64:64 + blocks] for a in around]
        for m, c in zip(mine, (kc, vc)):
            m.copy_(c)
        for b in range(B):
            for t in range(S if counts is None else max(0, int(counts[b]))):
                pos = int(lengths[b]) + t
                page = int(table[b, pos // bs]) if 0 <= pos // bs < 3 else -1
                if 0 <= page < blocks:
                    kc[page, :, pos % bs], vc[page, :, pos % bs] = k[b, :, t], v[b, :, t]
        A.copy_to_blocks(*dev(k, v), *mine, *dev(table, lengths), new_rows=None if counts is None else counts.to(DEV))
        for a, m, want in zip(around, mine, (kc, vc)):
            assert torch.equal(m.cpu(), want) and bool((a[:64] == 3).all()) and bool((a[64 + blocks:] == 3).all())


def test_new_rows_of_the_sixteen_bit_append_are_checked(A):
    x, c = torch.zeros(2, 1, 1, 8, device=DEV).half(), torch.zeros(3, 1, 4, 8, device=DEV).half()
    table, n = ints([[0], [1]]), ints([0, 0])
    for bad in (ints([1]), ints([1, 1]).long(), ints([[1, 1]]), torch.zeros(2, dtype=torch.int32), ints([1, 0, 1, 0])[::2]):
        with pytest.raises(RuntimeError):
            A.copy_to_blocks(x, x, c, c, table, n, new_rows=bad)


@pytest.mark.parametrize("dtype,G,E,bs", [(torch.bfloat16, 4, 128, 16), (torch.float16, 2, 64, 8), (torch.float32, 2, 64, 4), (torch.bfloat16, 3, 128, 12)])
def test_a_batch_over_sixteen_bit_pages(A, dtype, G, E, bs):
    """Rows forked, emptied and grown in a pool that runs dry, appended to and attended to: every row has its own history, nothing else changes."""
    gen = torch.Generator().manual_seed(52)
    Hkv, blocks, width = 2, 11, 6
    caches = [torch.full((blocks, Hkv, bs, E), 9.0, dtype=dtype, device=DEV) for _ in range(2)]
    refs, table, lengths = ints([0] * blocks), ints([[-1] * width]), ints([0])
    history = [[]]
    ran_dry = 0
    # (fork of a partly filled page, an emptied row, room for some only: the last rows of the third and fourth step find no pages)
    for source, new in (([0, -1], [bs + 3, 2 * bs]), ([0, 0, 1, -1, 0], [1] * 5), (None, [1, 2 * bs, bs, 3 * bs, 1]), ([0, 0, 0, 1, 0], [1, 1, 1, 2 * bs, 1]),
                        ([1, -1, 4], [0, 1, 2]), (None, [bs, 1, 1])):
        refs, table, lengths, room = A.step_blocks(refs, table, lengths, caches, bs, source=None if source is None else ints(source), new_tokens=ints(new))
        rows = range(len(new)) if source is None else source
        history = [list(history[u]) if u >= 0 else [] for u in rows]
        got_room, W, S = room.tolist(), len(new), max(new)
        ran_dry += sum(r < n for r, n in zip(got_room, new))
        k, v = (torch.randn(W, Hkv, S, E, generator=gen).to(dtype) for _ in range(2))
        A.copy_to_blocks(*dev(k, v), *caches, table, lengths, new_rows=room)
        for w in range(W):
            history[w] += [(k[w, :, t], v[w, :, t]) for t in range(got_room[w])]
        lengths = lengths + room
        assert lengths.tolist() == [len(h) for h in history]
        stored = [c.cpu() for c in caches]
        for w, h in enumerate(history):
            for n, (a, b) in enumerate(h):
                page = int(table[w, n // bs])
                assert torch.equal(stored[0][page, :, n % bs], a) and torch.equal(stored[1][page, :, n % bs], b)
        q = torch.randn(1, W, Hkv * G, 1, E, generator=gen).to(dtype)
        got = A.hogwild_paged_sdpa(q.to(DEV), (lengths - 1)[None, :, None].contiguous(), *caches, table, E ** -0.5, ints([width * bs])).cpu().double()
        for w, h in enumerate(history):
            if not h:
                assert bool((got[w] == 0).all())
                continue
            kk, vv = (torch.stack([x[n] for x in h], 1).double().repeat_interleave(G, 0) for n in (0, 1))
            p = torch.softmax((kk @ q[0, w].double().transpose(1, 2))[..., 0] * E ** -0.5, -1)
            want = (p[:, None] @ vv)[:, 0]
            # the output's rounding, the probabilities' (to the caches' type), fp32 scores and sums: 2^-24 each times the 64 terms they have at most
            half = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
            limit = half * want.abs() + (half + 300 * 2.0 ** -23) * (p[:, None] @ vv.abs())[:, 0] * 2
            assert bool(((got[w, :, 0] - want).abs() <= limit).all())
    assert ran_dry >= 2


def test_needs_that_32_bits_do_not_hold(A):
    """65,536 rows that together ask for 2^31 pages and more: those in front get theirs, from the first that finds too few on nobody does."""
    rows, width, blocks, bs = 65536, 32769, 70000, 4
    table = torch.full((rows, width), -1, dtype=torch.int32, device=DEV)
    refs, lengths = ints([0] * blocks), ints([0] * rows)
    new = torch.full((rows,), width * bs, dtype=torch.int32, device=DEV)
    st, room = status(), torch.empty(rows, dtype=torch.int32, device=DEV)
    A.step_blocks(refs, table, lengths, [], bs, new_tokens=new, out=(refs, table, lengths, room), status=st)
    assert int(st) == 512 and room[:2].tolist() == [width * bs] * 2 and not bool(room[2:].any())
    assert torch.equal(table[:2].flatten(), torch.arange(2 * width, dtype=torch.int32, device=DEV)) and bool((table[2:] == -1).all())
    assert bool((refs[:2 * width] == 1).all()) and not bool(refs[2 * width:].any())


def test_a_length_below_zero_in_place(A):
    """Is none, also where the lengths are written where they are read."""
    rng = np.random.default_rng(12)
    refs, table = pool(rng, 20, 4, 5, [7, 0, 9])
    run_step(A, refs, table, [7, -3, 9], None, [1, 2, 0], 4, some_caches(rng, 20), out=lambda a: (a[0], a[1], a[2], ints([7] * 3)))


@pytest.mark.parametrize("dtype,G,E,bs,packed", [(torch.bfloat16, 4, 128, 16, False), (torch.float16, 2, 64, 12, False), (torch.float32, 2, 64, 8, False),
                                                 (torch.bfloat16, 4, 128, 16, True), (torch.float16, 16, 128, 8, False)])
def test_sixteen_bit_reads_stay_inside_the_cache(A, dtype, G, E, bs, packed):
    """Rows that see keys of pages that are not there are the caller's error: what they hold is not defined, but it comes from the cache, and other rows are
    as they would be beside any table."""
    gen = torch.Generator().manual_seed(53)
    Hkv, blocks, width, W = 2, 40, 20, 3
    around = [torch.full((blocks + 200, Hkv, bs, E), float("nan"), dtype=dtype, device=DEV) for _ in range(2)]
    caches = [a[200:] for a in around]
    for c in caches:
        c.copy_(torch.randn(c.shape, generator=gen).to(dtype))
    table = torch.randperm(blocks, generator=gen).to(torch.int32)[:width].repeat(W, 1)
    bad = table.clone()
    bad[1, 2], bad[1, 7:] = -1, -1
    keys = width * bs
    if packed:
        counts = [1, 300, 1]
        cu = ints([0, 1, 301, 302])
        q = torch.randn(1, 302, Hkv * G, E, generator=gen).to(dtype).to(DEV)
        loc, lens = torch.full((1, 302), keys - 1, dtype=torch.int32, device=DEV), ints([[keys] * W])
        outs = [A.hogwild_varlen_paged_sdpa(q, loc, *caches, t.to(DEV), 0.1, lens, cu) for t in (table, bad)]
        good = [0, 301]
    else:
        q = torch.randn(1, W, Hkv * G, 1, E, generator=gen).to(dtype).to(DEV)
        loc = torch.full((1, W, 1), keys - 1, dtype=torch.int32, device=DEV)
        outs = [A.hogwild_paged_sdpa(q, loc, *caches, t.to(DEV), 0.1, ints([keys])) for t in (table, bad)]
        good = [0, 2]
    assert torch.equal(outs[0][good], outs[1][good]) and bool(torch.cat(outs).isfinite().all())
