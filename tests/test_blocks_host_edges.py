"""What the C ABI refuses of the calls that go with page bookkeeping, without a GPU."""
import pytest

from inference_lib_b200 import _build, _cabi

OK, NULL, SHAPE, HEAD, DTYPE, ALIGN = 0, -1, -2, -3, -4, -6


@pytest.fixture(scope="module")
def lib():
    _build.build_cabi()
    return _cabi.load()


@pytest.mark.parametrize("change,rc", [
    ({}, OK), ({0: None}, NULL), ({4: None}, NULL), ({5: None}, NULL), ({6: None}, OK), ({7: 0}, SHAPE), ({9: -1}, SHAPE), ({14: 0}, OK), ({14: -3}, SHAPE),
    ({15: 7}, DTYPE), ({10: 60}, HEAD), ({1: 4104}, ALIGN),
])
def test_append_of_rows_refuses(lib, change, rc):
    #         states, caches, table, lengths, new_rows, B, Hkv, S, E, Ev, block size, table width, blocks, dtype
    args = [4096] * 7 + [2, 2, 0, 64, 64, 16, 4, 9, _cabi.BF16, None]
    for i, x in change.items():
        args[i] = x
    if rc not in (OK, SHAPE):
        args[9] = 3
    assert lib.hogatt_copy_to_blocks_rows_launch(*args) == rc


def test_a_pool_beyond_the_count_of_pages_is_refused(lib):
    import ctypes as C
    from tests.test_q4_host import _blocks
    assert lib.hogatt_step_blocks_launch(C.byref(_blocks(_cabi.StepBlocks, num_blocks=2 ** 31 - 1)), None) == -10


@pytest.mark.parametrize("width,rc", [(2 ** 30 - 1, -7), (2 ** 30, -10), (2 ** 31 - 1, -10)])
def test_tables_wider_than_a_row_counts_are_refused(lib, width, rc):
    """(The one below is refused for the workspace it is given.)"""
    import ctypes as C
    from tests.test_q4_host import _blocks
    assert lib.hogatt_step_blocks_launch(C.byref(_blocks(_cabi.StepBlocks, max_blocks=width, workspace_bytes=8)), None) == rc


@pytest.mark.parametrize("scale,unit,rc", [(0.1, 1.0, NULL), (1e-30, 1.0, NULL), (1e-20, 2.0 ** -64, -9), (1e-30, 2.0 ** -28, -9), (1e-30, 2.0 ** 64, NULL), (5e3, 1.0, NULL),
                                           (6e3, 1.0, -9), (0.1, 2.0 ** 20, -9), (1e25, 2.0 ** -63, -9), (float("nan"), 1.0, -9), (float("inf"), 1.0, -9),
                                           (0.0, 1.0, -9), (-0.1, 1.0, -9)])
def test_the_chunks_kernel_goes_by_scale_times_unit(lib, scale, unit, rc):
    """Asked for by name where it is refused; where it is not, the missing output is what is refused."""
    import ctypes as C
    from tests.test_q4_host import _paged
    x = _paged(kernel=4, cu_seqlens_q=4096, total_q_tokens=4, scale=scale, key_unit=unit, out=None)
    assert lib.hogatt_paged_q4_sdpa_launch(C.byref(x), None) == rc


def test_the_unit_error_names_both_of_its_causes(lib):
    text = lib.hogatt_status_string(-12).decode()
    assert "power of two" in text and "scale" in text
