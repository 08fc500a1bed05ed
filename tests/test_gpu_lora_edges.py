"""Where the per-request operators could lose a value that the definition has: magnitudes near the ends of the type,
infinities, cancelling results, long rows. Against the definition in 64 bits; tolerances stand with each test."""
import numpy as np
import pytest
import torch

from aipu_b200 import formats as F
from aipu_b200 import ops

pytestmark = pytest.mark.gpu
BF, FP, HF = torch.bfloat16, torch.float32, torch.float16
TYPES = [F.Q4_K, F.Q6_K, F.Q8_0, F.F16]


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _plain(d, K, N):
    """Adapters that no row names."""
    return ops.LoraAdapters(torch.zeros((1, 1, K), dtype=BF, device=d), torch.zeros((1, N, 1), dtype=BF, device=d))


def _weights(wt, N, K, seed, d):
    w = torch.from_numpy(F.random_rows_np(wt, N, K, seed=seed)).to(d)
    return w, ops.dequant(wt, w, N, K).double()


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("M", [9, 70, 140, 300])
def test_rows_of_extreme_magnitudes_above_8_rows(wt, M):
    """Token rows near the largest and the smallest numbers, beside ordinary ones: the scale of a row is exact.
    A result is off by its rounding to bf16 (2^-8), by the 32-bit sums of K products (K * 2^-23 of their magnitudes) and
    the weights' rounding (2^-11 of each)."""
    d, K, N = _dev(), 512, 130
    w, wd = _weights(wt, N, K, 5, d)
    x = torch.randn((M, K), device=d, generator=torch.Generator(d).manual_seed(M)).clamp_(-3.9, 3.9)
    e = [0, 100, 112, 116, 117, 124, 125, -90, -100, -110, -117, -120]
    shift = torch.tensor([e[m % len(e)] for m in range(M)], device=d)
    x = torch.ldexp(x.double(), shift.view(M, 1)).to(BF)
    want = x.double() @ wd.t()
    tol = x.double().abs() @ wd.abs().t() * (K * 2.0 ** -23 + 2.0 ** -11)
    # (the projection of a large row may pass the range of the type)
    fits = want.abs() + tol < 3e38
    ids = torch.full((M,), -1, dtype=torch.int32, device=d)
    got = ops.gemm_lora(wt, w, N, K, x, _plain(d, K, N), ids).double()
    bad = fits & ~((got - want).abs() <= tol + (want.abs() + tol) * 2.0 ** -8 + 2.0 ** -126)
    assert not bad.any(), (shift[bad.any(1)].tolist(), got[bad][:4], want[bad][:4])
    assert fits[shift.view(M, 1).expand(M, N) <= 117].float().mean() > 0.95
