"""Low-rank adapters of many requests on the GPU against the definition in 64 bits.

Tolerance of an output element. The exact value is e = y + d; u(t) is half a step of type t relative to
the value, eps(t) / 2: bf16 has 8 significant bits, so 2^-8; fp32 2^-24. Error sources:
  * the rounding of the result: u(out) * |result|;
  * fp32 sums of K products (first product) and of at most 128 (second), added in some order by the MMA
    and the joins: at most (number of terms) * 2^-23 relative to the sum of the magnitudes (2^-23, not
    2^-24: the MMA's sums may truncate). Sums run through blocks, so K / 16 + 64 bounds the length;
  * h as bf16 pieces: the first is h truncated to 8 bits, its rest is below 2^-7 |h|; two pieces (bf16
    result) round that rest by 2^-8 of itself, 2^-15 |h|; three (fp32 result) hold all 24 bits;
  * for gemm, the projection's own sum of K products, 4 * K * 2^-24 relative to its magnitudes, and its
    operands' rounding (see there).
With S = sum_r |scale| (sum_k |x a|) |b| every term is at most a fixed multiple of S."""
import numpy as np
import pytest
import torch

from aipu_b200 import formats as F
from aipu_b200 import ops

pytestmark = pytest.mark.gpu
BF, FP, HF = torch.bfloat16, torch.float32, torch.float16
HALF = {BF: 2.0 ** -8, FP: 2.0 ** -24}


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def _case(M, K, N, R, L, ad=BF, ids=None, ranks=False, seed=0):
    d = _dev()
    g = torch.Generator().manual_seed(seed + 1000 * M + K + 7 * N + R)
    x = torch.randn((M, K), generator=g).to(BF).to(d)
    a = (torch.randn((L, R, K), generator=g) * K ** -0.5).to(ad).to(d)
    b = (torch.randn((L, N, R), generator=g) * R ** -0.5).to(ad).to(d)
    scale = (torch.rand((L,), generator=g) + 0.5).to(d)
    rk = torch.randint(0, R + 1, (L,), generator=g).to(torch.int32).to(d) if ranks else None
    if ids is None:
        ids = torch.randint(-1, L, (M,), generator=g)
    return ops.LoraAdapters(a, b, scale, rk), torch.as_tensor(ids, dtype=torch.int32).to(d), x


def _delta(ad, ids, x):
    """(delta, magnitudes S) in 64 bits on the CPU."""
    x64 = x.double().cpu()
    L, R, _ = ad.a.shape
    d = torch.zeros(x.shape[0], ad.b.shape[1], dtype=torch.float64)
    s = torch.zeros_like(d)
    for n in range(L):
        m = (ids.cpu() == n).nonzero().view(-1)
        r = R if ad.ranks is None else min(max(int(ad.ranks[n]), 0), R)
        f = 1.0 if ad.scale is None else float(ad.scale[n])
        a, b = ad.a[n, :r].double().cpu(), ad.b[n, :, :r].double().cpu()
        d[m] = f * ((x64[m] @ a.t()) @ b.t())
        s[m] = abs(f) * ((x64[m].abs() @ a.abs().t()) @ b.abs().t())
    return d, s


def _check(out, y64, d, s, K, extra=0.0):
    e = y64 + d
    got = out.double().cpu()
    pieces = 2.0 ** -15 if out.dtype == BF else 0.0
    tol = s * ((K / 16 + 64 + 128) * 2.0 ** -23 + pieces) + extra
    # the fp32 sum before the last rounding, and the rounding of what may be off by tol already
    tol = tol + (e.abs() + tol) * (HALF[out.dtype] + 2.0 ** -24)
    bad = (got - e).abs() > tol
    assert not bad.any(), ((got - e).abs() / tol).max()


@pytest.mark.parametrize("M,K,N,R,L", [
    (1, 4096, 4096, 16, 4), (1, 8, 8, 1, 1), (3, 256, 64, 8, 2), (8, 512, 520, 32, 1), (9, 1024, 192, 64, 1),
    (64, 640, 256, 16, 64), (64, 2048, 512, 128, 3), (65, 512, 256, 16, 2), (200, 768, 320, 64, 3), (256, 256, 96, 16, 9),
    (257, 256, 96, 16, 9), (257, 4160, 576, 32, 1), (300, 512, 192, 128, 2), (40, 512, 192, 128, 40), (1000, 256, 1024, 32, 5),
    (700, 256, 128, 16, 200), (130, 384, 264, 24, 1), (640, 192, 72, 64, 3)])
@pytest.mark.parametrize("ad", [BF, HF])
def test_add_matches_the_definition(M, K, N, R, L, ad):
    A, ids, x = _case(M, K, N, R, L, ad, ranks=R > 8)
    y = torch.randn((M, N), device=x.device).to(BF)
    d, s = _delta(A, ids, x)
    _check(ops.lora_add(A, ids, x, y), y.double().cpu(), d, s, K)
    y32 = torch.randn((M, N), device=x.device)
    o = ops.lora_add(A, ids, x, y32)
    assert o.dtype == FP
    _check(o, y32.double().cpu(), d, s, K)
    _check(ops.lora_add(A, ids, x, y32, out=torch.empty_like(y)), y32.double().cpu(), d, s, K)


@pytest.mark.parametrize("M,K,N,R", [(1, 1, 1, 1), (5, 13, 7, 3), (77, 1001, 2051, 13), (12, 100, 33, 5), (90, 34, 70, 127),
                                     (66, 999, 9, 128), (300, 34, 70, 127), (301, 999, 9, 128), (277, 1001, 515, 13), (400, 1, 1, 1)])
@pytest.mark.parametrize("ad", [BF, HF])
def test_odd_sizes(M, K, N, R, ad):
    A, ids, x = _case(M, K, N, R, 3, ad, ranks=True)
    y = torch.randn((M, N), device=x.device)
    d, s = _delta(A, ids, x)
    _check(ops.lora_add(A, ids, x, y), y.double().cpu(), d, s, K)
    _check(ops.lora_add(A, ids, x, y.to(BF)), y.to(BF).double().cpu(), d, s, K)


@pytest.mark.parametrize("M", [6, 150, 300])
def test_columns_of_wider_tensors_and_in_place(M):
    """Queries and values of a fused projection: columns of one tensor, added to in place; what lies beside stays."""
    A, ids, x = _case(M, 256, 72, 16, 3)
    wide_x = torch.randn((M, 300), device=x.device).to(BF)
    wide_x[:, 8:264] = x
    wide = torch.randn((M, 200), device=x.device).to(BF)
    before = wide.clone()
    d, s = _delta(A, ids, x)
    for at in (0, 72, 101):  # the last one is not 16-byte aligned
        y = wide[:, at:at + 72]
        y0 = y.clone()
        assert ops.lora_add(A, ids, wide_x[:, 8:264], y, out=y) is y
        _check(y, y0.double().cpu(), d, s, 256)
        assert torch.equal(y[ids < 0], y0[ids < 0])
    assert torch.equal(wide[:, 144 + 29:], before[:, 144 + 29:])


@pytest.mark.parametrize("M", [1, 40, 64, 65, 256, 500])
def test_rows_without_an_adapter(M):
    """Left as they are to the bit, signs of zero and NaN among them; all rows, or all but one."""
    A, _, x = _case(M, 128, 96, 8, 2)
    y = torch.randn((M, 96), device=x.device).to(BF)
    y[0, :4] = torch.tensor([-0.0, 0.0, float("inf"), float("nan")])
    ids = torch.full((M,), -1, dtype=torch.int32, device=x.device)
    o = ops.lora_add(A, ids, x, y)
    assert torch.equal(o[:, 4:].view(torch.int16), y[:, 4:].view(torch.int16))
    assert torch.equal(o[0, :3].view(torch.int16), y[0, :3].view(torch.int16)) and bool(o[0, 3].isnan())
    ids[M - 1] = 1
    o2 = ops.lora_add(A, ids, x, y)
    assert torch.equal(o2[:M - 1, 4:], y[:M - 1, 4:])
    d, s = _delta(A, ids, x)
    _check(o2[M - 1:, 4:], y[M - 1:, 4:].double().cpu(), d[M - 1:, 4:], s[M - 1:, 4:], 128)


def test_an_id_out_of_range_is_no_adapter_and_sets_the_status():
    for M in (5, 80, 300):
        A, _, x = _case(M, 128, 64, 8, 2)
        ctx = ops.Context(x.device)
        y = torch.randn((M, 64), device=x.device).to(BF)
        ids = torch.zeros(M, dtype=torch.int32, device=x.device)
        ops.lora_add(A, ids, x, y, ctx=ctx)
        assert ctx.status() == 0
        ids[1], ids[2] = 2, 2 ** 31 - 1
        o = ops.lora_add(A, ids, x, y, ctx=ctx)
        assert torch.equal(o[1:3], y[1:3]) and ctx.status() == 4
        ids[1], ids[2] = -2 ** 31, -5
        assert torch.equal(ops.lora_add(A, ids, x, y, ctx=ctx)[1:3], y[1:3]) and ctx.status() == 0
        ctx.close()


@pytest.mark.parametrize("M", [4, 100, 300])
def test_nothing_is_read_past_a_rank(M):
    """NaN in the rows of a and columns of b past an adapter's rank, rank 0, and ranks outside 0..R."""
    A, ids, x = _case(M, 96, 80, 24, 5, ids=[m % 5 for m in range(M)])
    A.ranks = torch.tensor([0, 5, 16, 24, 24], dtype=torch.int32, device=x.device)
    for n, r in enumerate([0, 5, 16, 24, 24]):
        A.a[n, r:] = float("nan")
        A.b[n, :, r:] = float("nan")
    y = torch.randn((M, 80), device=x.device).to(BF)
    d, s = _delta(A, ids, x)
    o = ops.lora_add(A, ids, x, y)
    _check(o, y.double().cpu(), d, s, 96)
    A.ranks = torch.tensor([-3, 5, 16, 24, 1000], dtype=torch.int32, device=x.device)
    assert torch.equal(ops.lora_add(A, ids, x, y), o)


def test_infinities_and_nan_stay_in_their_row():
    for M in (6, 70, 270):
        A, ids, x = _case(M, 128, 64, 16, 1, ids=[0] * M)
        y = torch.zeros((M, 64), device=x.device)
        clean = ops.lora_add(A, ids, x, y)
        x[1, 3], x[4, 7] = float("inf"), float("nan")
        o = ops.lora_add(A, ids, x, y)
        keep = [m for m in range(M) if m not in (1, 4)]
        assert torch.equal(o[keep], clean[keep])
        assert not torch.isfinite(o[1]).any() and o[4].isnan().all()
        # an infinite h times a finite b of one sign is that infinity, not NaN
        B = ops.LoraAdapters(A.a[:, :1].abs().contiguous(), A.b[:, :, :1].abs().add(0.5).contiguous())
        o = ops.lora_add(B, ids, x, y)
        assert (o[1] == float("inf")).all()


def test_equal_calls_give_equal_bits_whatever_shares_the_batch():
    A, ids, x = _case(500, 512, 256, 32, 7)
    y = torch.randn((500, 256), device=x.device)
    o = ops.lora_add(A, ids, x, y)
    for _ in range(5):
        assert torch.equal(ops.lora_add(A, ids, x, y), o)


def test_up_to_256_rows_do_not_depend_on_what_shares_the_call():
    for R in (16, 100):
        A, ids, x = _case(256, 512, 300, R, 9)
        y = torch.randn((256, 300), device=x.device)
        o = ops.lora_add(A, ids, x, y)
        for m in range(0, 256, 7):
            assert torch.equal(ops.lora_add(A, ids[m:m + 1], x[m:m + 1], y[m:m + 1]), o[m:m + 1])


@pytest.mark.parametrize("M,L", [(20, 32768), (300, 32768), (5000, 3), (70001, 40)])
def test_many_adapters_and_many_rows(M, L):
    A, ids, x = _case(M, 16, 8, 1, L)
    y = torch.randn((M, 8), device=x.device)
    i = ids.long().clamp_min(0)
    h = (x.double() * A.a.double()[i, 0]).sum(1, keepdim=True)
    size = (x.double() * A.a.double()[i, 0]).abs().sum(1, keepdim=True)
    f = torch.where(ids >= 0, A.scale.double()[i], 0.0).view(M, 1)
    b = A.b.double()[i, :, 0]
    _check(ops.lora_add(A, ids, x, y), y.double().cpu(), (f * h * b).cpu(), (f * size * b.abs()).cpu(), 16)


def test_no_rows():
    A, _, x = _case(2, 64, 32, 4, 1)
    e = torch.empty((0,), dtype=torch.int32, device=x.device)
    assert ops.lora_add(A, e, x[:0], torch.empty((0, 32), dtype=BF, device=x.device)).shape == (0, 32)
    w = torch.from_numpy(F.random_rows_np(F.Q4_K, 32, 256)).to(x.device)
    A, _, x = _case(2, 256, 32, 4, 1)
    assert ops.gemm_lora(F.Q4_K, w, 32, 256, x[:0], A, e).shape == (0, 32)


@pytest.mark.parametrize("M", [6, 150, 300])
@pytest.mark.parametrize("N", [1, 71, 259, 515])
@pytest.mark.parametrize("t", [BF, FP])
def test_odd_widths_in_aligned_rows(M, N, t):
    """Rows that begin on 16 bytes and end inside a 16-byte piece: the columns behind them are neither read nor written."""
    A, ids, x = _case(M, 128, N, 8, 2)
    wide = torch.full((M, 520), float("nan"), dtype=t, device=x.device)
    y = wide[:, :N]
    y.copy_(torch.randn((M, N), device=x.device))
    y64 = y.double().cpu()
    d, s = _delta(A, ids, x)
    ops.lora_add(A, ids, x, y, out=y)
    _check(y, y64, d, s, 128)
    assert wide[:, N:].isnan().all()


@pytest.mark.parametrize("wt", [F.Q4_K, F.Q6_K, F.Q8_0, F.F16])
@pytest.mark.parametrize("M,K,N,R", [(1, 1024, 512, 16), (1, 256, 1, 1), (2, 512, 100, 8), (8, 2048, 260, 32), (11, 768, 130, 5),
                                     (63, 512, 96, 16), (64, 512, 96, 16), (150, 1024, 333, 64)])
def test_gemm_lora_matches_the_definition(wt, M, K, N, R):
    A, ids, x = _case(M, K, N, R, 3)
    w = torch.from_numpy(F.random_rows_np(wt, N, K, seed=N)).to(x.device)
    wd = ops.dequant(wt, w, N, K).double().cpu()
    x64 = x.double().cpu()
    A.b.mul_(float(wd.square().mean().sqrt()) * K ** 0.5)  # a share of the result that 16 bits show
    d, s = _delta(A, ids, x)
    o = ops.gemm_lora(wt, w, N, K, x, A, ids)
    # the projection's fp32 sums: relative to the magnitudes of its products
    mag = x64.abs() @ wd.abs().t()
    if M > 8 and wt != F.F16:
        # fp16 GEMM: a weight is rounded by 2^-11 of itself at most (half a step), and the tokens, scaled to 2^9 .. 2^10,
        # by half the smallest fp16 step, 2^-25, where they are small: 2^-34 of the row's largest
        extra = mag * (4 * K * 2.0 ** -24 + 2.0 ** -11)
    else:
        if wt == F.Q4_K and M <= 8:  # d * sum - dmin * sum: |d sc q| + |dmin m| of a weight is at most |w| + 2 |dmin m|
            dm = np.ascontiguousarray(w.view(-1, 144).cpu().numpy()[:, 2:4]).view(np.float16).astype(np.float64).reshape(N, K // 256)
            mag = mag + 2 * 63 * (x64.abs().view(M, -1, 256).sum(2) @ torch.from_numpy(dm).t())
        extra = mag * (4 * K * 2.0 ** -24)
    if M == 1:  # the integer engine rounds x once to 2^-21 of the row's maximum, relative to sums of |w|
        extra = extra + 2.0 ** -21 * x64.abs().amax(1, keepdim=True) * wd.abs().sum(1)
    if M > 8:
        extra = extra + 2.0 ** -34 * x64.abs().amax(1, keepdim=True) * wd.abs().sum(1)
    _check(o, x64 @ wd.t(), d, s, K, extra)


def test_gemm_lora_without_adapters_is_the_projection():
    """Rows without an adapter: up to 8 rows give the bits of gemm; more rows do not depend on the adapters at all."""
    for M in (1, 5, 8, 100):
        A, _, x = _case(M, 512, 200, 8, 2)
        ids = torch.full((M,), -1, dtype=torch.int32, device=x.device)
        w = torch.from_numpy(F.random_rows_np(F.Q4_K, 200, 512, seed=3)).to(x.device)
        o = ops.gemm_lora(F.Q4_K, w, 200, 512, x, A, ids)
        if M <= 8:
            assert torch.equal(o, ops.gemm(F.Q4_K, w, 200, 512, x))
        A.a.fill_(float("nan"))
        assert torch.equal(ops.gemm_lora(F.Q4_K, w, 200, 512, x, A, ids), o)


@pytest.mark.parametrize("wt", [F.Q4_K, F.Q6_K, F.Q8_0, F.F16])
@pytest.mark.parametrize("M,K,N", [(9, 256, 1), (64, 2048, 128), (65, 256, 129), (128, 512, 127), (129, 768, 300), (256, 512, 256),
                                   (257, 256, 640), (700, 2304, 520), (300, 5120, 5), (257, 8192, 259), (290, 2048, 1003)])
def test_gemm_lora_many_rows_at_tile_borders(wt, M, K, N):
    """Weights of the extremes too: scales of zero, of fp16's smallest and of its largest numbers, in some rows."""
    A, ids, x = _case(M, K, N, 8, 2)
    w_np = F.random_rows_np(wt, N, K, seed=N + 1)
    if wt != F.F16:
        bb, at = F.BLOCK_BYTES[wt], {F.Q4_K: 0, F.Q6_K: 208, F.Q8_0: 0}[wt]
        blocks = w_np.reshape(N, -1, bb)
        for row, scale in ((0, 0.0), (N // 2, 2.0 ** -24), (N - 1, 300.0)):
            blocks[row, :, at:at + 2] = np.frombuffer(np.float16(scale).tobytes(), np.uint8)
            if wt == F.Q4_K:
                blocks[row, :, 2:4] = 0
    w = torch.from_numpy(w_np).to(x.device)
    x[0] = 0
    x[M - 1] *= 2.0 ** 60
    wd = ops.dequant(wt, w, N, K).double().cpu()
    x64 = x.double().cpu()
    ids.fill_(-1)
    o = ops.gemm_lora(wt, w, N, K, x, A, ids)
    mag, big = x64.abs() @ wd.abs().t(), x64.abs().amax(1, keepdim=True) * wd.abs().sum(1)
    extra = mag * (4 * K * 2.0 ** -24 + (0.0 if wt == F.F16 else 2.0 ** -11)) + 2.0 ** -34 * big
    _check(o, x64 @ wd.t(), torch.zeros_like(mag), torch.zeros_like(mag), K, extra)


@pytest.mark.parametrize("wt", [F.Q4_K, F.F16])
@pytest.mark.parametrize("M", [4, 40, 200, 300])
def test_gemm_lora_fp16_adapters_ranks_out_and_another_stream(wt, M):
    K, N, R = 512, 333, 24
    A, ids, x = _case(M, K, N, R, 4, HF, ranks=True)
    w = torch.from_numpy(F.random_rows_np(wt, N, K, seed=M)).to(x.device)
    wd = ops.dequant(wt, w, N, K).double().cpu()
    A.b.mul_(float(wd.square().mean().sqrt()) * K ** 0.5)
    d, s = _delta(A, ids, x)
    ctx = ops.Context(x.device)
    out = torch.full((M + 2, N), 7.0, dtype=BF, device=x.device)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        o = ops.gemm_lora(wt, w, N, K, x, A, ids, ctx=ctx, out=out[1:M + 1])
    st.synchronize()
    assert o.data_ptr() == out[1:].data_ptr() and (out[0] == 7).all() and (out[M + 1] == 7).all()
    mag = x.double().cpu().abs() @ wd.abs().t()
    if wt == F.Q4_K:
        dm = np.ascontiguousarray(w.view(-1, 144).cpu().numpy()[:, 2:4]).view(np.float16).astype(np.float64).reshape(N, K // 256)
        mag = mag + 2 * 63 * (x.double().cpu().abs().view(M, -1, 256).sum(2) @ torch.from_numpy(dm).t())
    extra = mag * (4 * K * 2.0 ** -24 + (2.0 ** -11 if M > 8 and wt != F.F16 else 0.0))
    extra = extra + 2.0 ** -34 * x.double().cpu().abs().amax(1, keepdim=True) * wd.abs().sum(1)
    _check(o, x.double().cpu() @ wd.t(), d, s, K, extra)
    assert ctx.status() == 0
    bad = ids.clone()
    bad[1] = 4
    ids[1] = -1
    assert torch.equal(ops.gemm_lora(wt, w, N, K, x, A, bad, ctx=ctx), ops.gemm_lora(wt, w, N, K, x, A, ids, ctx=ctx))
    assert ctx.status() == 4
    ctx.close()


def test_two_devices():
    """A context and tensors on another device than the current one; tensors on two devices are refused."""
    if _dev() is None or torch.cuda.device_count() < 2:
        pytest.skip("needs two CUDA devices")
    A, ids, x = _case(70, 512, 96, 16, 3)
    y = torch.randn((70, 96), device=x.device)
    w = torch.from_numpy(F.random_rows_np(F.Q4_K, 96, 512, seed=1)).to(x.device)
    far = torch.device("cuda", 1)
    B = ops.LoraAdapters(A.a.to(far), A.b.to(far), A.scale.to(far))
    assert torch.equal(ops.lora_add(B, ids.to(far), x.to(far), y.to(far)).cpu(), ops.lora_add(A, ids, x, y).cpu())
    assert torch.equal(ops.gemm_lora(F.Q4_K, w.to(far), 96, 512, x.to(far), B, ids.to(far)).cpu(),
                       ops.gemm_lora(F.Q4_K, w, 96, 512, x, A, ids).cpu())
    assert torch.equal(ops.greedy_tokens(y.to(far)).cpu(), ops.greedy_tokens(y).cpu())
    with pytest.raises(ValueError):
        ops.lora_add(A, ids, x, y.to(far))


@pytest.mark.parametrize("M", [3, 90, 290])
def test_captured_and_replayed_with_new_inputs(M):
    A, ids, x = _case(M, 512, 96, 16, 3)
    w = torch.from_numpy(F.random_rows_np(F.Q4_K, 96, 512, seed=1)).to(x.device)
    y = torch.randn((M, 96), device=x.device)
    ops.gemm_lora(F.Q4_K, w, 96, 512, x, A, ids)
    ops.lora_add(A, ids, x, y)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o1 = ops.gemm_lora(F.Q4_K, w, 96, 512, x, A, ids)
        o2 = ops.lora_add(A, ids, x, y)
    for n in range(3):
        B, ids2, x2 = _case(M, 512, 96, 16, 3, seed=n + 5)
        x.copy_(x2)
        ids.copy_(ids2)
        g.replay()
        assert torch.equal(o1, ops.gemm_lora(F.Q4_K, w, 96, 512, x, A, ids))
        assert torch.equal(o2, ops.lora_add(A, ids, x, y))


def test_two_streams_at_once():
    A, ids, x = _case(300, 1024, 512, 32, 4)
    y = torch.randn((300, 512), device=x.device)
    want = ops.lora_add(A, ids, x, y)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for _ in range(4):
        for st in streams:
            with torch.cuda.stream(st):
                outs.append(ops.lora_add(A, ids, x, y))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


@pytest.mark.parametrize("M", [20, 300])
def test_programmatic_launch_flag_keeps_the_results(M):
    A, ids, x = _case(M, 512, 256, 16, 4)
    ctx = ops.Context(x.device).set_flags(pdl=True)
    y = torch.randn((M, 256), device=x.device)
    want = ops.lora_add(A, ids, x, y + 0)
    for _ in range(20):
        z = y + 0  # a kernel right before, whose output is read
        assert torch.equal(ops.lora_add(A, ids, x, z, ctx=ctx), want)
    ctx.close()


def test_refusals():
    A, ids, x = _case(4, 64, 32, 8, 2)
    d = x.device
    y = torch.zeros((4, 32), dtype=BF, device=d)
    with pytest.raises(ValueError):
        ops.lora_add(A, ids.long(), x, y)
    with pytest.raises(ValueError):
        ops.lora_add(A, ids[:3], x, y)
    with pytest.raises(ValueError):
        ops.lora_add(A, ids, x.float(), y)
    with pytest.raises(ValueError):
        ops.lora_add(A, ids, x, y[:, :31])
    with pytest.raises(ValueError):
        ops.lora_add(A, ids, x, y, out=torch.zeros((4, 32), device=d))  # bf16 in, fp32 out
    with pytest.raises(ValueError):
        ops.lora_add(A, ids, x, y.to(HF))
    with pytest.raises(ValueError):
        ops.lora_add(A, ids, x, y.t().contiguous().t())
    with pytest.raises(ValueError):
        ops.lora_add(A, ids, x, y[:1].expand(4, 32))
    with pytest.raises(ValueError):
        ops.lora_add(ops.LoraAdapters(A.a, A.b.to(HF)), ids, x, y)
    with pytest.raises(ValueError):
        ops.lora_add(ops.LoraAdapters(A.a, A.b.transpose(1, 2).contiguous()), ids, x, y)
    with pytest.raises(ValueError):
        ops.lora_add(ops.LoraAdapters(A.a, A.b, ranks=torch.zeros(3, dtype=torch.int32, device=d)), ids, x, y)
    with pytest.raises(ops.L.AipuError):
        big = ops.LoraAdapters(torch.zeros((1, 129, 64), dtype=BF, device=d), torch.zeros((1, 32, 129), dtype=BF, device=d))
        ops.lora_add(big, ids, x, y)
    w = torch.from_numpy(F.random_rows_np(F.Q8_0, 32, 64)).to(d)
    with pytest.raises(ops.L.AipuError):
        ops.gemm_lora(F.Q8_0, w, 32, 64, x, A, ids)  # K not a multiple of 256
    with pytest.raises(ValueError):
        ops.gemm_lora(F.Q8_0, w, 31, 64, x, A, ids)
