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


def _residual(wt, w, N, K, x, y64):
    """gemm_lora's sums less bf16(y64), through an adapter for each row (x[:, 0] is 1): what the result's rounding hides."""
    M, d = x.shape[0], x.device
    a = torch.zeros((M, 1, K), dtype=BF, device=d)
    a[:, 0, 0] = 1
    near = y64.to(BF).contiguous()
    A = ops.LoraAdapters(a, -near.view(M, N, 1))
    return ops.gemm_lora(wt, w, N, K, x, A, torch.arange(M, dtype=torch.int32, device=d)).double(), y64 - near.double()


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("M", [1, 3, 8, 9, 65, 129, 300])
def test_weights_keep_their_bits_at_every_row_count(wt, M):
    """One weight a result, as x picks it, less its bf16 value: off by the rounding of the rest (2^-8 of it) and by 2^-19
    of the row's largest weight (fp16 halves: 2^-22 of the weight; Q4_K's two terms in fp32; one row: x to 2^-21)."""
    d, K, N = _dev(), 512, 200
    w, wd = _weights(wt, N, K, M, d)
    x = torch.zeros((M, K), dtype=BF, device=d)
    x[:, 0] = 1
    k = torch.randint(1, K, (M,), generator=torch.Generator().manual_seed(M)).to(d)
    x[torch.arange(M, device=d), k] = 1
    y64 = wd[:, 0].view(1, N) + wd[:, k].t()
    got, want = _residual(wt, w, N, K, x, y64)
    tol = want.abs() * 2.0 ** -8 + 2.0 ** -19 * 2 * wd.abs().amax(1)
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("M,K", [(16, 4096), (40, 2048), (300, 6144)])
def test_the_projections_sums_have_32_bits(wt, M, K):
    """Root mean square of the sums' error: K / 16 steps of the MMA, each cut off by at most 2^-23 of a running sum that is at
    most about the result, and the rounding of the rest to bf16 (2^-9 of up to 2^-9, rms). Weights of 11 bits would give 2^-12
    / sqrt(3), 1.4e-4."""
    d, N = _dev(), 264
    w, wd = _weights(wt, N, K, M, d)
    x = torch.randn((M, K), device=d, generator=torch.Generator(d).manual_seed(K)).to(BF)
    x[:, 0] = 1
    y64 = x.double() @ wd.t()
    got, want = _residual(wt, w, N, K, x, y64)
    err = (got - want).square().mean().sqrt() / y64.square().mean().sqrt()
    assert err <= K / 16 * 2.0 ** -23 + 2.0 ** -18, float(err)


@pytest.mark.parametrize("wt", [F.Q8_0, F.F16])
@pytest.mark.parametrize("M", [9, 150, 300])
def test_an_infinite_token_keeps_its_signs(wt, M):
    """An infinite value times weights that are not 0 is infinite with the weight's sign, whatever the weight's bits."""
    d, K, N = _dev(), 256, 140
    w, wd = _weights(wt, N, K, 9, d)
    x = torch.randn((M, K), device=d, generator=torch.Generator(d).manual_seed(M)).to(BF)
    ids = torch.full((M,), -1, dtype=torch.int32, device=d)
    clean = ops.gemm_lora(wt, w, N, K, x, _plain(d, K, N), ids)
    x[1, 7], x[4, 30], x[5, 2] = float("inf"), float("-inf"), float("nan")
    got = ops.gemm_lora(wt, w, N, K, x, _plain(d, K, N), ids)
    keep = [m for m in range(M) if m not in (1, 4, 5)]
    assert torch.equal(got[keep], clean[keep]) and got[5].isnan().all()
    for m, k, s in ((1, 7, 1), (4, 30, -1)):
        live = wd[:, k] != 0
        assert torch.equal(got[m, live].double(), (s * wd[live, k].sign()) * float("inf"))
        assert got[m, ~live].isnan().all()


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("K", [11008, 14336, 28672])
@pytest.mark.parametrize("N", [80, 2400])
def test_few_rows_of_long_weights(wt, K, N):
    """Tokens that do not all fit the shared memory of one GEMV launch. Sums of K products by steps of 16, each off by at
    most 2^-23 of the magnitudes (Q4_K: of d sc q and dmin m apart); one row: x to 2^-21 of its largest."""
    d = _dev()
    w, wd = _weights(wt, N, K, 3, d)
    x = torch.randn((8, K), device=d, generator=torch.Generator(d).manual_seed(K)).to(BF)
    g = torch.Generator(d).manual_seed(N)
    A = ops.LoraAdapters((torch.randn((2, 8, K), device=d, generator=g) * K ** -0.5).to(BF),
                         (torch.randn((2, N, 8), device=d, generator=g) * float(wd.square().mean().sqrt()) * K ** 0.5).to(BF))
    ids = torch.tensor([0, 1, -1, 1, 0, 0, -1, 1], dtype=torch.int32, device=d)
    h = torch.einsum("mk,lrk->mlr", x.double(), A.a.double())
    size = torch.einsum("mk,lrk->mlr", x.double().abs(), A.a.double().abs())
    want, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    if wt == F.Q4_K:
        dm = w.view(-1, 144)[:, 2:4].contiguous().view(HF).double().view(N, K // 256)
        mag = mag + 2 * 63 * (x.double().abs().view(8, -1, 256).sum(2) @ dm.abs().t())
    for m in range(8):
        if ids[m] >= 0:
            n = int(ids[m])
            want[m] += A.b[n].double() @ h[m, n]
            mag[m] += A.b[n].double().abs() @ size[m, n] + (A.b[n].double().abs() @ h[m, n].abs()) * 2.0 ** -15 / (K / 16 * 2.0 ** -23)
    tol = mag * (K / 16 * 2.0 ** -23)
    for M in (1, 2, 3, 5, 6, 7, 8):
        got = ops.gemm_lora(wt, w, N, K, x[:M], A, ids[:M]).double()
        t = tol[:M] + (2.0 ** -21 * x[:1].double().abs().amax() * wd.abs().sum(1) if M == 1 else 0)
        t = t + (want[:M].abs() + t) * 2.0 ** -8
        assert ((got - want[:M]).abs() <= t).all(), (M, ((got - want[:M]).abs() / t).max())
    assert torch.equal(ops.gemm_lora(wt, w, N, K, x[2:3], A, ids[2:3]), ops.gemm(wt, w, N, K, x[2:3]))


@pytest.mark.parametrize("wt", [F.Q4_K, F.F16])
@pytest.mark.parametrize("M", [1, 5])
def test_few_rows_of_weights_longer_than_the_gemv_takes(wt, M):
    """K above 65536: the fp16 GEMM takes any number of rows."""
    d, K, N = _dev(), 65536 + 512, 40
    w, wd = _weights(wt, N, K, 3, d)
    x = torch.randn((M, K), device=d, generator=torch.Generator(d).manual_seed(K)).to(BF)
    ids = torch.full((M,), -1, dtype=torch.int32, device=d)
    got = ops.gemm_lora(wt, w, N, K, x, _plain(d, K, N), ids).double()
    want, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    assert ((got - want).abs() <= mag * (K / 16 * 2.0 ** -23) + want.abs() * 2.0 ** -7).all()


@pytest.mark.parametrize("M", [1, 8])
def test_few_rows_of_more_weight_rows_than_the_gemv_counts(M):
    """N above 2^20, an LM head's rows of many vocabularies in one: results on both sides of the border and at the end."""
    d, K, N = _dev(), 256, (1 << 20) + 1000
    w = torch.randint(0, 256, (N, 8, 34), dtype=torch.uint8, device=d, generator=torch.Generator(d).manual_seed(1))
    w[:, :, 0] = 0
    w[:, :, 1] = 0x1C  # fp16 2^-8
    x = torch.randn((M, K), device=d, generator=torch.Generator(d).manual_seed(M)).to(BF)
    A = _plain(d, K, N)
    A.a[0, 0, 0] = 1
    A.b[0, :, 0] = torch.arange(N, device=d) % 128
    ids = torch.tensor([0, -1] * 4, dtype=torch.int32, device=d)[:M]
    got = ops.gemm_lora(F.Q8_0, w, N, K, x, A, ids).double()
    wd = w[:, :, 2:].view(torch.int8).reshape(N, K)
    for a, b in ((0, 3000), ((1 << 20) - 3000, (1 << 20) + 500), (N - 600, N)):
        v = wd[a:b].double() * 2.0 ** -8
        want, mag = x.double() @ v.t(), x.double().abs() @ v.abs().t()
        add = x[:, :1].double() * A.b[0, a:b, 0].double() * (ids >= 0).view(M, 1)
        tol = mag * (16 * 2.0 ** -23) + add.abs() * 2.0 ** -15
        tol = tol + ((want + add).abs() + tol) * 2.0 ** -8
        assert ((got[:, a:b] - want - add).abs() <= tol).all()


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("e", [0, 100, 105, 111, 116, 121, 124, -90, -100])
def test_rows_of_extreme_magnitudes_up_to_8_rows(wt, M, e):
    """As above 8 rows; Q4_K's sums of d sc q and of dmin m apart, and one row's x is rounded to 2^-21 of its largest."""
    d, K, N = _dev(), 512, 130
    w, wd = _weights(wt, N, K, 5, d)
    x = torch.randn((M, K), device=d, generator=torch.Generator(d).manual_seed(M)).clamp_(-3.9, 3.9)
    x = (x.double() * 2.0 ** e).to(BF)
    want, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    if wt == F.Q4_K:
        dm = w.view(-1, 144)[:, 2:4].contiguous().view(HF).double().view(N, K // 256)
        mag = mag + 2 * 63 * (x.double().abs().view(M, -1, 256).sum(2) @ dm.abs().t())
    tol = mag * (K * 2.0 ** -23) + (2.0 ** -21 * x.double().abs().amax() * wd.abs().sum(1) if M == 1 else 0)
    ids = torch.full((M,), -1, dtype=torch.int32, device=d)
    got = ops.gemm_lora(wt, w, N, K, x, _plain(d, K, N), ids)
    fits = want.abs() + tol < 3e38
    bad = fits & ~((got.double() - want).abs() <= tol + (want.abs() + tol) * 2.0 ** -8)
    assert not bad.any(), (got[bad][:4], want[bad][:4])
    assert torch.equal(ops.gemm(wt, w, N, K, x), got)


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("M", [1, 2, 3, 4, 8])
@pytest.mark.parametrize("v", ["inf", "-inf", "nan"])
def test_tokens_that_are_not_finite_up_to_8_rows(wt, M, v):
    """No finite result of such a row, and none of the others' changes."""
    d, K, N = _dev(), 512, 130
    w, _ = _weights(wt, N, K, 5, d)
    x = torch.randn((M, K), device=d, generator=torch.Generator(d).manual_seed(M)).to(BF)
    A, ids = _plain(d, K, N), torch.full((M,), -1, dtype=torch.int32, device=d)
    clean = ops.gemm_lora(wt, w, N, K, x, A, ids)
    x[M - 1, 300] = float(v)
    got = ops.gemm_lora(wt, w, N, K, x, A, ids)
    assert torch.equal(got[:M - 1], clean[:M - 1]) and not torch.isfinite(got[M - 1]).any()
    assert not torch.isfinite(ops.gemm(wt, w, N, K, x)[M - 1]).any()


@pytest.mark.parametrize("ad", [BF, HF])
@pytest.mark.parametrize("M", [6, 70, 270])
@pytest.mark.parametrize("t", [BF, FP])
def test_infinite_values_keep_their_signs_in_adapters(ad, M, t):
    """x, A, B or h infinite, beside values of few significant bits (1, powers of two, zero pieces): the infinity or NaN that
    the definition gives, in the rows, ranks and columns that it has them in."""
    d, K, N, R = _dev(), 72, 48, 5
    g = torch.Generator(d).manual_seed(M)
    pick = torch.tensor([1.0, 2.0, -1.0, 0.5, 1.5, -0.375, 3.0, 1.0 + 2.0 ** -7], device=d)

    def values(*s):
        return pick[torch.randint(0, len(pick), s, device=d, generator=g)]

    x, a, b = values(M, K).to(BF), values(2, R, K).to(ad), values(2, N, R).to(ad)
    x[1, 3], x[2, 5], x[3, 9] = float("inf"), float("-inf"), float("nan")
    a[1, 2, 7] = float("inf")
    b[1, 4, 1], b[1, 5, 3], b[1, 6, 0] = float("inf"), float("-inf"), float("nan")
    x[4, 7] = 0  # times the infinite value of A: NaN
    ids = torch.zeros(M, dtype=torch.int32, device=d)
    ids[4:] = 1
    # one rank: an infinite x times one row of A; then several
    for r in (1, R):
        A = ops.LoraAdapters(a[:, :r].contiguous(), b[:, :, :r].contiguous())
        y = torch.zeros((M, N), dtype=t, device=d)
        out = ops.lora_add(A, ids, x, y).double()
        h = torch.einsum("mk,mrk->mr", x.double(), A.a.double()[ids.long()])
        want = torch.einsum("mr,mnr->mn", h, A.b.double()[ids.long()])
        live = torch.isfinite(want)
        assert torch.equal(torch.isfinite(out), live)
        assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isposinf(), want.isposinf())
        # finite: few significant bits; h of 16 bits for a bf16 result
        size = 3 * torch.einsum("mk,mnr->mn", x.double().abs(), A.b.double()[ids.long()].abs())  # |a| is at most 3
        assert ((out - want).abs()[live] <= (want.abs() * 2.0 ** -8 + size * 2.0 ** -15)[live]).all()
    # the sum over K is infinite: a finite x and A
    x = torch.full((M, K), 2.0 ** 120, device=d).to(BF)
    A = ops.LoraAdapters(torch.full((1, 1, K), 2.0 ** 15, device=d).to(ad), values(1, N, 1).to(ad))
    out = ops.lora_add(A, torch.zeros(M, dtype=torch.int32, device=d), x, torch.zeros((M, N), dtype=t, device=d))
    assert torch.equal(out, (A.b[0, :, 0].double().sign() * float("inf")).to(t).expand(M, N))


@pytest.mark.parametrize("ad", [BF, HF])
@pytest.mark.parametrize("M", [5, 256, 300])
def test_single_products_have_all_bits(ad, M):
    """x = 1, a = 1, y = 0: scale * b. h holds the factor's 24 bits, b is exact, so what is off is the last product's sum:
    one unit of fp32, 2^-23, for the MMA that adds the largest pieces and cuts off, and 2^-23 of the pieces before it,
    2^-7 of the value, for each of the five MMAs of two steps that may have gone before."""
    d, K, N, L = _dev(), 64, 72, 5
    g = torch.Generator(d).manual_seed(M)
    x = torch.zeros((M, K), device=d).to(BF)
    x[:, 11] = 1
    a = torch.zeros((L, 1, K), device=d).to(ad)
    a[:, 0, 11] = 1
    b = (1 + torch.rand((L, N, 1), device=d, generator=g)).to(ad) * torch.where(torch.rand((L, N, 1), device=d, generator=g) < 0.5, 1, -1).to(ad)
    scale = 1 + torch.rand(L, device=d, generator=g)
    # the largest rests: upper bits 0, lower bits all set
    scale[0] = 1 + 2.0 ** -15 - 2.0 ** -23
    b[0, 0, 0] = 1 + 7 * 2.0 ** -10 if ad == HF else 1
    ids = (torch.arange(M, device=d) % L).to(torch.int32)
    out = ops.lora_add(ops.LoraAdapters(a, b, scale), ids, x, torch.zeros((M, N), device=d))
    want = (scale.double().view(L, 1) * b[:, :, 0].double())[ids.long()]
    rel = ((out.double() - want).abs() / want.abs()).max()
    assert rel <= 2.0 ** -23 * (1 + 10 * 2.0 ** -7), float(rel * 2 ** 23)


@pytest.mark.parametrize("ad", [BF, HF])
@pytest.mark.parametrize("M,K", [(8, 65536), (8, 1 << 20), (300, 65536)])
def test_long_sums_of_one_sign_are_rounded_not_cut_off(ad, M, K):
    """All of x and a positive: sums that are cut off fall short by half a unit a step, K / 16 of them. Root mean square of
    the results' error, in 2^-24 of them: blocks of 64 k by the MMA, four steps (eight with fp16 pieces) of at most 2^-23 of
    the block; rounded adds at random, at most sqrt of their number (K / 64 / 64 in a warp of the few rows' 64, K / 64 / 8 in
    a share of the many rows', and the joins) of 1; the second product 2."""
    d, N, R = _dev(), 40, 4
    g = torch.Generator(d).manual_seed(K)
    x = torch.rand((M, K), device=d, generator=g).to(BF)
    a = torch.rand((1, R, K), device=d, generator=g).to(ad)
    b = (1 + torch.arange(N * R, device=d) % 97).view(1, N, R).to(ad)  # exact
    out = ops.lora_add(ops.LoraAdapters(a, b), torch.zeros(M, dtype=torch.int32, device=d), x, torch.zeros((M, N), device=d)).double()
    want = (x.double() @ a[0].double().t()) @ b[0].double().t()
    rms = float(((out - want) / want).square().mean().sqrt()) * 2 ** 24
    adds = (K / 4096 + 15) if M <= 256 else K / 512 + 8
    assert rms <= (8 if ad == BF else 16) + adds ** 0.5 + 2, rms


@pytest.mark.parametrize("wt", TYPES)
@pytest.mark.parametrize("K,N", [(4096, 4096), (4096, 4104), (11008, 1600)])
def test_9_to_17_rows_of_large_weights(wt, K, N):
    """On both sides of the borders between launches of the GEMV and the fp16 GEMM, in the rows and in the weights. Tolerance
    as for few rows of long weights."""
    d = _dev()
    w, wd = _weights(wt, N, K, 3, d)
    x = torch.randn((17, K), device=d, generator=torch.Generator(d).manual_seed(K)).to(BF)
    want, mag = x.double() @ wd.t(), x.double().abs() @ wd.abs().t()
    if wt == F.Q4_K:
        dm = w.view(-1, 144)[:, 2:4].contiguous().view(HF).double().view(N, K // 256)
        mag = mag + 2 * 63 * (x.double().abs().view(17, -1, 256).sum(2) @ dm.abs().t())
    tol = mag * (K / 16 * 2.0 ** -23)
    tol = tol + (want.abs() + tol) * 2.0 ** -8
    for M in (9, 12, 16, 17):
        ids = torch.full((M,), -1, dtype=torch.int32, device=d)
        got = ops.gemm_lora(wt, w, N, K, x[:M], _plain(d, K, N), ids).double()
        assert ((got - want[:M]).abs() <= tol[:M]).all(), M


@pytest.mark.parametrize("wt", [F.Q4_K, F.Q6_K])
def test_9_to_16_rows_on_several_streams_at_once(wt):
    """Calls of more than 8 rows share nothing of their context."""
    d, K, N, M = _dev(), 4096, 8192, 13
    w, _ = _weights(wt, N, K, 2, d)
    x = torch.randn((3, M, K), device=d, generator=torch.Generator(d).manual_seed(1)).to(BF)
    A, ids = _plain(d, K, N), torch.full((M,), -1, dtype=torch.int32, device=d)
    want = [ops.gemm_lora(wt, w, N, K, x[i], A, ids) for i in range(3)]
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for _ in range(6):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs.append((i, ops.gemm_lora(wt, w, N, K, x[i], A, ids)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i, o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = ops.gemm_lora(wt, w, N, K, x[0], A, ids)
    for i in (1, 2):
        x[0].copy_(x[i])
        g.replay()
        assert torch.equal(o, want[i])


@pytest.mark.parametrize("N", [32000, 128000, 50257])
@pytest.mark.parametrize("M,R", [(1, 16), (5, 64), (8, 13), (9, 128)])
@pytest.mark.parametrize("t", [BF, FP])
def test_few_rows_of_one_adapter_on_a_vocabulary(N, M, R, t):
    """The LM head's adapter in a verify pass, in place. Off by the result's rounding, by h's 16 bits (bf16 results) and by
    the sums of K and R products, at most 2^-23 of the magnitudes for each 16 terms and join."""
    d, K = _dev(), 512
    g = torch.Generator(d).manual_seed(N + M)
    a = (torch.randn((2, R, K), device=d, generator=g) * K ** -0.5).to(BF)
    b = (torch.randn((2, N, R), device=d, generator=g) * R ** -0.5).to(BF)
    x = torch.randn((M, K), device=d, generator=g).to(BF)
    y = torch.randn((M, N), device=d, generator=g).to(t)
    want, size = y.double(), (x.double().abs() @ a[1].double().abs().t()) @ b[1].double().abs().t()
    want = want + (x.double() @ a[1].double().t()) @ b[1].double().t()
    ids = torch.ones(M, dtype=torch.int32, device=d)
    assert ops.lora_add(ops.LoraAdapters(a, b), ids, x, y, out=y) is y
    tol = size * ((K / 16 + 64 + R) * 2.0 ** -23 + (2.0 ** -15 if t == BF else 0))
    tol = tol + (want.abs() + tol) * (2.0 ** -8 if t == BF else 2.0 ** -23)
    assert ((y.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("M", [1, 8, 12, 20, 300])
@pytest.mark.parametrize("wt", [F.Q4_K, F.F16])
def test_projection_with_the_programmatic_flag(M, wt):
    """Behind the kernel that writes x and before the next call that reads the result, on a context with the flag."""
    d, K, N = _dev(), 1024, 512
    w, _ = _weights(wt, N, K, 1, d)
    g = torch.Generator(d).manual_seed(M)
    A = ops.LoraAdapters((torch.randn((3, 16, K), device=d, generator=g) * K ** -0.5).to(BF), torch.randn((3, N, 16), device=d, generator=g).to(BF))
    back = ops.LoraAdapters((torch.randn((3, 16, N), device=d, generator=g) * 1e-3).to(BF), torch.randn((3, K, 16), device=d, generator=g).to(BF))
    x0 = torch.randn((M, K), device=d, generator=g).to(BF)
    ids = (torch.arange(M, device=d) % 4 - 1).to(torch.int32)
    ctx, flagged = ops.Context(d), ops.Context(d).set_flags(pdl=True)

    def chain(c):
        x = x0 + 0
        for _ in range(4):
            y = ops.gemm_lora(wt, w, N, K, x, A, ids, ctx=c)
            x = ops.lora_add(back, ids, y, x0, ctx=c)
        return y, x

    want = chain(ctx)
    for _ in range(10):
        got = chain(flagged)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert ctx.status() == 0 and flagged.status() == 0
    ctx.close()
    flagged.close()
