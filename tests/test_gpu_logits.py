"""Penalties, biases and masks on logits, and the greedy token, on the GPU: bit for bit against the same
steps in numpy fp32, and against the definition in 64 bits.

64-bit tolerance: the steps are at most 1 (repetition) + 2 (frequency: product and difference) + 1
(presence) + n (bias entries) roundings of 2^-24, each relative to a value of at most
|logit| * max(rep, 1/rep) + |freq| count + |pres| + sum |bias|."""
import numpy as np
import pytest
import torch

from aipu_b200 import ops

pytestmark = pytest.mark.gpu
F32 = np.float32


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return torch.device("cuda", 0)


def oracle(logits, tokens=None, spans=None, penalties=None, bias_begin=None, bias_ids=None, bias_vals=None, mask=None,
           mask_rows=None, ftype=F32):
    """The definition, step by step in `ftype`: (values, tokens)."""
    z = logits.astype(ftype).copy()
    M, V = z.shape
    for m in range(M):
        if spans is not None:
            b, g, e = spans[m]
            rep, pres, freq = penalties[m].astype(ftype)
            ctx, gen = tokens[b:e], tokens[g:e]
            ctx, gen = ctx[(ctx >= 0) & (ctx < V)], gen[(gen >= 0) & (gen < V)]
            ids = np.unique(ctx)
            with np.errstate(all="ignore"):
                z[m, ids] = np.where(z[m, ids] > 0, z[m, ids] / rep, z[m, ids] * rep)
            ids, n = np.unique(gen, return_counts=True)
            z[m, ids] = z[m, ids] - freq * n.astype(ftype)
            z[m, ids] = z[m, ids] - pres
        if bias_begin is not None:
            for i in range(bias_begin[m], bias_begin[m + 1]):
                if 0 <= bias_ids[i] < V:
                    z[m, bias_ids[i]] += bias_vals[i].astype(ftype)
        if mask is not None and mask_rows[m] >= 0:
            bits = np.unpackbits(mask[mask_rows[m]].view(np.uint8), bitorder="little")[:V]
            z[m, bits == 0] = -np.inf
    tok = []
    for row in z:
        ok = ~np.isnan(row) & (row > -np.inf)
        tok.append(int(np.argmax(np.where(ok, row, -np.inf))) if ok.any() else -1)
    return z, np.array(tok, np.int32)


def _controls(rng, M, V, history=0, shared=False, bias=0, masks=0, repeat=False):
    c = {}
    if history:
        lens = rng.integers(0, history + 1, M)
        if shared:
            T = history + M
            b, e = np.zeros(M, np.int64), history + np.arange(M)
        else:
            e = lens.cumsum()
            b, T = e - lens, int(lens.sum())
        c["tokens"] = (V * rng.random(T) ** 3).astype(np.int32)
        c["spans"] = np.stack([b, (b + e) // 2, e], 1).astype(np.int64)
        c["penalties"] = np.stack([rng.uniform(0.7, 1.5, M), rng.uniform(-1, 1, M), rng.uniform(-1, 1, M)], 1).astype(F32)
    if bias:
        lens = rng.integers(0, bias + 1, M)
        c["bias_begin"] = np.concatenate([[0], lens.cumsum()]).astype(np.int64)
        n = int(lens.sum())
        hi = max(1, V // 20) if repeat else V
        ids = [rng.integers(0, hi, k) if repeat else rng.choice(V, min(k, V), replace=False) for k in lens]
        c["bias_ids"] = np.concatenate(ids).astype(np.int32) if n else np.zeros(0, np.int32)
        c["bias_vals"] = rng.normal(0, 3, n).astype(F32)
    if masks:
        W = (V + 31) // 32
        p = rng.random((masks, 1))
        bits = rng.random((masks, W * 32)) < p
        c["mask"] = np.packbits(bits, axis=1, bitorder="little").view(np.int32).reshape(masks, W)
        c["mask_rows"] = (np.arange(M) % (masks + 1) - 1).astype(np.int32)
    return c


def _dev_controls(c, d):
    return ops.LogitControls(**{k: torch.from_numpy(v).to(d) for k, v in c.items()})


def _logits(rng, M, V, dtype, d):
    t = torch.from_numpy(rng.normal(0, 4, (M, V)).astype(F32)).to(dtype)
    return t.to(d), t.float().numpy()


def _run(M, V, dtype=torch.bfloat16, seed=0, **kw):
    d = _dev()
    rng = np.random.default_rng(seed + 31 * M + V)
    x, x_np = _logits(rng, M, V, dtype, d)
    c = _controls(rng, M, V, **kw)
    ctl = _dev_controls(c, d)
    ctx = ops.Context(d)
    out, tok = ops.process_logits(x, ctl, ctx=ctx)
    z, t = oracle(x_np, **c)
    np.testing.assert_array_equal(out.cpu().numpy(), z)
    np.testing.assert_array_equal(tok.cpu().numpy(), t)
    assert torch.equal(ops.greedy_tokens(x, ctl, ctx=ctx), tok)
    assert ctx.status() == 0
    ctx.close()
    z64, _ = oracle(x_np, ftype=np.float64, **c)
    size = np.abs(x_np) * 1.5
    steps = 4
    if "penalties" in c:
        size = size + np.abs(c["penalties"][:, 1:2]) + np.abs(c["penalties"][:, 2:3]) * kw["history"]
    if "bias_vals" in c:
        steps += kw["bias"]
        size = size + np.abs(c["bias_vals"]).sum()
    size = np.broadcast_to(size, z.shape)
    f = np.isfinite(z64)
    assert (np.abs(z[f] - z64[f]) <= (steps * 2.0 ** -24 * size)[f]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,V", [(1, 1), (1, 31), (2, 32), (3, 33), (1, 32000), (5, 50001), (40, 1000), (3, 255), (2, 257)])
def test_all_controls(M, V, dtype):
    _run(M, V, dtype, history=min(4 * V, 700), bias=min(V, 40), masks=2)


@pytest.mark.parametrize("kw", [dict(), dict(history=100), dict(history=9), dict(history=50, shared=True), dict(bias=20),
                                dict(bias=60, repeat=True), dict(masks=1), dict(masks=3, bias=5), dict(history=70, masks=4)])
def test_each_group_alone(kw):
    _run(4, 3001, **kw)
    _run(9, 512, torch.float32, **kw)


def test_a_long_context_and_many_rows():
    _run(2, 5000, history=100000)
    _run(200, 777, history=300, bias=7, masks=5)


@pytest.mark.parametrize("n", [32767, 32768, 70000])
def test_counts_that_pass_sixteen_bits(n):
    """One token generated n times beside others, and n times in the prompt of another row."""
    d = _dev()
    V = 45000
    rng = np.random.default_rng(n)
    x, x_np = _logits(rng, 2, V, torch.float32, d)
    gen = np.full(n, 4321, np.int32)
    c = dict(tokens=np.concatenate([gen, [4320, 4322, 44999, 4321]]).astype(np.int32),
             spans=np.array([[0, 0, n + 3], [0, n + 3, n + 4]], np.int64),
             penalties=np.array([[1.1, 0.5, 2.0 ** -9], [1.2, 0.25, 1.0]], F32))
    out, tok = ops.process_logits(x, _dev_controls(c, d))
    z, t = oracle(x_np, **c)
    np.testing.assert_array_equal(out.cpu().numpy(), z)
    np.testing.assert_array_equal(tok.cpu().numpy(), t)


def test_a_vocabulary_of_several_windows():
    """More tokens than a cluster counts at once: the context is scanned for each part."""
    _run(2, 250001, torch.float32, history=900, bias=300, masks=1)
    _run(1, 600000, history=900, bias=300, repeat=True, masks=1)
    _run(1, 400003, history=300000, bias=30, seed=5)


def test_rows_a_mask_leaves_nothing_of_and_values_that_are_not_finite():
    d = _dev()
    V, inf, nan = 100, float("inf"), float("nan")
    x = torch.randn((7, V), device=d)
    low = torch.finfo(torch.float32).min
    x[1] = -inf
    x[2], x[2, 60] = nan, -3.0
    x[3] = nan
    x[4], x[4, 70], x[4, 30] = low, low, nan  # the lowest value is above -inf
    x[5, 10], x[5, 11] = inf, inf
    x[6, 5], x[6, 50] = nan, inf  # both masked
    mask = torch.full((2, 4), -1, dtype=torch.int32, device=d)
    mask[0] = 0
    mask[1, 0], mask[1, 1] = ~(1 << 5), ~(1 << 18)
    rows = torch.tensor([0, -1, -1, -1, -1, -1, 1], dtype=torch.int32, device=d)
    out, tok = ops.process_logits(x, ops.LogitControls(mask=mask, mask_rows=rows))
    assert (out[0] == -inf).all() and out[6, 5] == -inf and out[6, 50] == -inf
    want = x[6].clone()
    want[5] = want[50] = -inf
    assert torch.equal(out[6], want)
    assert tok.tolist() == [-1, -1, 60, -1, 0, 10, int(want.argmax())]
    assert torch.equal(out[5], x[5]) and torch.equal(out[3].isnan(), x[3].isnan())


def test_ties_go_to_the_lowest_token():
    d = _dev()
    x = torch.zeros((3, 40000), device=d, dtype=torch.bfloat16)
    x[1, 39999] = x[1, 20000] = x[1, 777] = 2.0
    x[2, 1:] = -0.0
    assert ops.greedy_tokens(x).tolist() == [0, 777, 0]


def test_bad_spans_tokens_biases_and_mask_rows():
    """Spans and ranges are cut to their arrays, tokens outside the vocabulary count for nothing, a mask row past
    the masks is none; spans, ranges and rows that were wrong show in the status."""
    d = _dev()
    ctx = ops.Context(d)
    V = 64
    x = torch.randn((4, V), device=d)
    tokens = torch.tensor([-1, 3, V, 2 ** 31 - 1, -2 ** 31, 3, 5], dtype=torch.int32, device=d)
    pen = torch.tensor([[2.0, 1.0, 0.5]] * 4, device=d)

    def run(spans, **kw):
        ctl = ops.LogitControls(tokens=tokens, spans=torch.tensor(spans, device=d), penalties=pen, **kw)
        out, _ = ops.process_logits(x, ctl, ctx=ctx)
        return out, ctx.status()

    good, st = run([[0, 0, 7], [0, 7, 7], [3, 3, 3], [5, 6, 7]])
    assert st == 0 and torch.equal(good[2], x[2])
    z, _ = oracle(x.cpu().numpy(), tokens.cpu().numpy(), np.array([[0, 0, 7], [0, 7, 7], [3, 3, 3], [5, 6, 7]]), pen.cpu().numpy())
    assert np.array_equal(good.cpu().numpy(), z)
    o, st = run([[-4, 0, 2 ** 40], [-2 ** 62, 2 ** 62, 2 ** 62], [3, 9, -1], [5, 6, 8]])
    assert st == 4 and torch.equal(o, good)
    o, st = run([[0, 0, 0]] * 4, bias_begin=torch.tensor([-5, 2, 1, 99, 99], device=d),
                bias_ids=torch.tensor([1, V, 1], dtype=torch.int32, device=d), bias_vals=torch.ones(3, device=d))
    want = x.clone()
    want[0, 1] += 1
    want[2, 1] += 1
    assert st == 4 and torch.equal(o, want)
    o, st = run([[0, 0, 0]] * 4, mask=torch.zeros((1, 2), dtype=torch.int32, device=d),
                mask_rows=torch.tensor([1, -7, 2 ** 31 - 1, 0], dtype=torch.int32, device=d))
    assert st == 4 and torch.equal(o[:3], x[:3]) and (o[3] == -float("inf")).all()
    ctx.close()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_columns_of_a_wider_tensor_in_place_and_out(dtype):
    d = _dev()
    rng = np.random.default_rng(1)
    M, V = 5, 1003
    c = _controls(rng, M, V, history=300, bias=9, masks=2)
    wide, wide_np = _logits(rng, M, V + 37, dtype, d)
    z, t = oracle(wide_np[:, 5:5 + V], **c)
    ctl = _dev_controls(c, d)
    big = torch.full((M, V + 3), 7.0, device=d)
    out, tok = ops.process_logits(wide[:, 5:5 + V], ctl, out=big[:, 1:1 + V])
    assert np.array_equal(out.cpu().numpy(), z) and np.array_equal(tok.cpu().numpy(), t)
    assert (big[:, 0] == 7).all() and (big[:, 1 + V:] == 7).all()
    if dtype == torch.float32:
        out, _ = ops.process_logits(wide[:, 5:5 + V], ctl, out=wide[:, 5:5 + V])
        assert np.array_equal(out.cpu().numpy(), z)
        assert np.array_equal(wide[:, :5].cpu().numpy(), wide_np[:, :5])
        assert np.array_equal(wide[:, 5 + V:].cpu().numpy(), wide_np[:, 5 + V:])


def test_captured_replayed_two_streams_and_equal_bits():
    d = _dev()
    rng = np.random.default_rng(2)
    M, V = 6, 9000
    c = _controls(rng, M, V, history=500, bias=30, masks=2, repeat=True)
    x, _ = _logits(rng, M, V, torch.bfloat16, d)
    ctl = _dev_controls(c, d)
    want = ops.process_logits(x, ctl)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.process_logits(x, ctl))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[0]) and torch.equal(b, want[1]) for a, b in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, tok = ops.process_logits(x, ctl)
    for n in range(3):
        y, y_np = _logits(rng, M, V, torch.bfloat16, d)
        x.copy_(y)
        ctl.spans[:, 2] = torch.clamp(ctl.spans[:, 2] - n, min=0).maximum(ctl.spans[:, 1])
        g.replay()
        c["spans"] = ctl.spans.cpu().numpy()
        z, t = oracle(y_np, **c)
        assert np.array_equal(out.cpu().numpy(), z) and np.array_equal(tok.cpu().numpy(), t)


def test_penalties_of_every_kind():
    """Zero, negative, infinite and NaN penalties act as the steps say."""
    d = _dev()
    rng = np.random.default_rng(4)
    vals = [0.0, -1.5, np.inf, -np.inf, np.nan, 1.0, 1e-38, 3e38]
    pen = np.array([[a, b, c] for a in vals for b in (0.0, np.inf, -2.0) for c in (0.0, np.nan, 1e30)], F32)
    M, V = len(pen), 90
    x, x_np = _logits(rng, M, V, torch.float32, d)
    x[:, 7], x_np[:, 7] = 0.0, 0.0
    tokens = rng.integers(0, V // 2, M * 20).astype(np.int32)
    at = 20 * np.arange(M)
    c = dict(tokens=tokens, spans=np.stack([at, at + 8, at + 20], 1).astype(np.int64), penalties=pen)
    out, tok = ops.process_logits(x, _dev_controls(c, d))
    with np.errstate(all="ignore"):
        z, t = oracle(x_np, **c)
    np.testing.assert_array_equal(out.cpu().numpy(), z)
    np.testing.assert_array_equal(tok.cpu().numpy(), t)


def test_thousands_of_rows():
    _run(3000, 130, history=40, bias=3, masks=7)


def test_no_rows():
    d = _dev()
    out, tok = ops.process_logits(torch.empty((0, 10), device=d))
    assert out.shape == (0, 10) and tok.shape == (0,)
