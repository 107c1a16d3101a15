"""The 4-bit paged operators at the ends of their range: scales, queries and scores that are no ordinary numbers, long sequences."""
import numpy as np
import pytest
import torch

from tests import q4_util
from tests.test_gpu_q4 import DEV, E4M3, KERNELS, A, dev, odd_scales, paged, skip_unless_eligible, status, table_of  # noqa: F401

pytestmark = pytest.mark.gpu


def small_cache(seed, blocks, Hkv, bs, E, units=(1.0, 1.0)):
    gen = torch.Generator().manual_seed(seed)
    (kc, ks), (vc, vs) = q4_util.random_cache(gen, blocks, Hkv, bs, E, units[0]), q4_util.random_cache(gen, blocks, Hkv, bs, E, units[1])
    return [kc, vc, ks, vs], gen


def sign_rows(gen, blocks, Hkv, bs, E):
    """Codes and scales of rows of +-1."""
    return q4_util.quantise(torch.where(torch.rand(blocks, Hkv, bs, E, generator=gen) < 0.5, 6.0, -6.0), 6.0)


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
