"""The 4-bit cache and page bookkeeping without a GPU: the plain implementations themselves, and what the C ABI refuses."""
import ctypes as C

import numpy as np
import pytest
import torch

from inference_lib_b200 import _build, _cabi
from tests import q4_util

OK, NULL, SHAPE, HEAD, DTYPE, ALIGN, WS, CHOICE, LARGE, UNIT = 0, -1, -2, -3, -4, -6, -7, -9, -10, -12


@pytest.fixture(scope="module")
def lib():
    _build.build_cabi()
    return _cabi.load()


def test_the_plain_scale_is_the_nearest_e4m3():
    x = torch.cat([torch.linspace(0, 500, 4001), torch.logspace(-12, 2.6, 3001, base=10.0)]).float()
    got = q4_util.E4M3[q4_util._nearest(q4_util.E4M3_VALUE, x.double().numpy())]
    assert np.array_equal(got, x.clamp(max=448).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_the_plain_codes():
    x = torch.zeros(16)
    x[:14] = torch.tensor([6, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, -0.25, -2.4, -6, 0.74])
    codes, scales = q4_util.quantise(x, 1.0)                  # scale 1
    assert scales.view(torch.float8_e4m3fn).float().tolist() == [1.0]
    assert q4_util.values(codes, scales, 1.0)[:14].tolist() == [6, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 0, -2, -6, 0.5]
    for bad in (float("nan"), float("inf")):
        x[3] = bad
        assert np.isnan(q4_util.values(*q4_util.quantise(x, 1.0), 1.0)).all()


def _paged(**kw):
    x = _cabi.PagedQ4Problem()
    p = x.paged
    p.F, p.W, p.Hq, p.Hkv, p.E, p.Ev, p.S, p.block_size, p.max_blocks_per_seq, p.num_blocks = 1, 2, 8, 2, 128, 128, 1, 16, 4, 9
    p.dtype, p.scale = _cabi.BF16, 0.1
    for n in ("out", "queries", "locations", "fragment_lengths", "key_cache", "value_cache", "block_table", "workspace"):
        setattr(p, n, 4096)
    x.key_scales = x.value_scales = 4096
    x.key_unit = x.value_unit = 1.0
    for k, v in kw.items():
        setattr(x if hasattr(x, k) else p, k, v)
    return x


@pytest.mark.parametrize("change,rc", [
    (dict(Hq=7), SHAPE), (dict(num_blocks=0), SHAPE), (dict(S=0), SHAPE), (dict(block_size=0), SHAPE), (dict(dtype=7), DTYPE),
    (dict(E=120), HEAD), (dict(E=272), HEAD), (dict(Ev=48), HEAD), (dict(Ev=8), HEAD), (dict(kernel=3), CHOICE), (dict(F=5000), -5),
    (dict(key_unit=0.3), UNIT), (dict(value_unit=-1.0), UNIT), (dict(key_unit=0.0), UNIT), (dict(value_unit=float("nan")), UNIT),
    (dict(value_unit=float("inf")), UNIT), (dict(key_unit=2.0 ** 70), UNIT), (dict(key_scales=None), NULL), (dict(workspace=None), NULL),
    (dict(value_scales=4104), ALIGN), (dict(key_cache=4097), ALIGN), (dict(workspace=4112), ALIGN), (dict(W=1 << 30, S=4), LARGE),
    (dict(scale=1e25, key_unit=2.0 ** 64), UNIT),                          # the scores' factor is no fp32 number
    (dict(F=4096, max_blocks_per_seq=1 << 20, block_size=1 << 10), LARGE), # more tiles than 32 bits count
    (dict(F=4096, max_blocks_per_seq=1 << 20, block_size=1 << 10, dtype=_cabi.F32), LARGE),
    # sequences and tokens whose units do not fit 32 bits: asked of the kernel for chunks
    (dict(W=2147483392, total_q_tokens=2147483647, Hq=1, Hkv=1, cu_seqlens_q=4096, kernel=4), LARGE),
])
def test_attention_refuses(lib, change, rc):
    assert lib.hogatt_paged_q4_sdpa_launch(C.byref(_paged(**change)), None) == rc


def _append(struct, **kw):
    p = struct()
    p.B, p.Hkv, p.S, p.E, p.Ev, p.block_size, p.max_blocks, p.num_blocks, p.dtype = 2, 2, 3, 64, 64, 16, 4, 9, _cabi.F16
    p.key_unit = p.value_unit = 0.5
    for n, t in struct._fields_:
        if t is C.c_void_p and n not in ("cu_seqlens", "new_rows", "device_status"):
            setattr(p, n, 4096)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,rc", [
    (dict(B=0), SHAPE), (dict(S=-1), SHAPE), (dict(max_blocks=0), SHAPE), (dict(E=72), HEAD), (dict(Ev=512), HEAD), (dict(dtype=-1), DTYPE),
    (dict(key_unit=3.0), UNIT), (dict(block_table=None), NULL), (dict(key_scales=4100), ALIGN), (dict(S=0), OK),
])
def test_append_and_read_refuse(lib, change, rc):
    assert lib.hogatt_copy_to_blocks_q4_launch(C.byref(_append(_cabi.Q4Append, **change)), None) == rc
    assert lib.hogatt_copy_from_blocks_q4_launch(C.byref(_append(_cabi.Q4Read, **change)), None) == rc


def _blocks(struct, **kw):
    p = struct()
    for n, t in struct._fields_:
        if t is C.c_void_p and n not in ("source", "new_tokens", "device_status"):
            setattr(p, n, 4096 * (1 + [f[0] for f in struct._fields_].index(n)))
    p.num_blocks, p.workspace_bytes = 9, 1 << 20
    if struct is _cabi.StepBlocks:
        p.block_size, p.max_blocks, p.rows_in, p.rows_out = 16, 4, 2, 2
    else:
        p.table_entries = 8
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("change,rc", [
    (dict(num_blocks=0), SHAPE), (dict(block_size=0), SHAPE), (dict(rows_out=3), SHAPE), (dict(rows_in=70000, rows_out=70000), LARGE),
    (dict(refs_out=None), NULL), (dict(room=None), NULL), (dict(workspace=4097), ALIGN), (dict(workspace_bytes=8), WS),
    (dict(source=4096, table_out=64, table_in=64), SHAPE), (dict(source=4096, lengths_out=64, lengths_in=64), SHAPE),
])
def test_step_blocks_refuses(lib, change, rc):
    assert lib.hogatt_step_blocks_launch(C.byref(_blocks(_cabi.StepBlocks, **change)), None) == rc


@pytest.mark.parametrize("change,rc", [
    (dict(num_blocks=0), SHAPE), (dict(table_entries=-1), SHAPE), (dict(moved=None), NULL), (dict(table_in=None), NULL),
    (dict(workspace=4097), ALIGN), (dict(workspace_bytes=8), WS),
])
def test_compact_blocks_refuses(lib, change, rc):
    assert lib.hogatt_compact_blocks_launch(C.byref(_blocks(_cabi.CompactBlocks, **change)), None) == rc


@pytest.mark.parametrize("struct", [_cabi.StepBlocks, _cabi.CompactBlocks])
def test_page_tensors_are_checked(lib, struct):
    fn = lib.hogatt_step_blocks_launch if struct is _cabi.StepBlocks else lib.hogatt_compact_blocks_launch
    p = _blocks(struct)
    p.caches.count = 1
    assert fn(C.byref(p), None) == NULL
    data, size = (C.c_void_p * 1)(4096), (C.c_int64 * 1)(0)
    p.caches.data, p.caches.block_bytes = data, size
    assert fn(C.byref(p), None) == SHAPE
    size[0], data[0] = 64, None
    assert fn(C.byref(p), None) == NULL


def test_workspace_sizes(lib):
    assert lib.hogatt_step_blocks_workspace_bytes(0) == 0 and lib.hogatt_step_blocks_workspace_bytes(65537) == 0
    assert lib.hogatt_step_blocks_workspace_bytes(64) >= 4 * (16 + 5 * 64)
    assert lib.hogatt_compact_blocks_workspace_bytes(0) == 0 and lib.hogatt_compact_blocks_workspace_bytes(1000) >= 4 * (32 + 1002)


def test_the_plain_step_keeps_count():
    """The sequential definition that the GPU tests compare with: counts stay the number of table entries."""
    rng = np.random.default_rng(3)
    table, lengths, refs, at = [], [], [0] * 40, 0
    for n in (33, 16, 5):
        pages = [at + i for i in range(-(-n // 8))]
        at += len(pages)
        table.append(pages + [-1] * (8 - len(pages)))
        lengths.append(n)
        for p in pages:
            refs[p] += 1
    for _ in range(30):
        source = [int(x) for x in rng.integers(-1, len(lengths), 5)]
        new = [int(x) for x in rng.integers(0, 9, 5)]
        refs, table, lengths, room, flags = q4_util.step_blocks(refs, table, lengths, source, new, 8, [])
        lengths = [n + r for n, r in zip(lengths, room)]
        held = [p for row in table for p in row if p >= 0]
        assert [held.count(p) for p in range(40)] == refs
        for w, (row, n) in enumerate(zip(table, lengths)):
            assert all(p >= 0 for p in row[:-(-n // 8)])
            if room[w] > 0:                                   # what is written next is nobody else's
                assert all(refs[p] == 1 for p in row[(n - room[w]) // 8:-(-n // 8)])
        if max(lengths) > 40:
            lengths = [n % 30 for n in lengths]
