"""Cases of the per-request operators of a mixed serving batch: low-rank adapters beside a (quantised) projection,
and the controls of each request on its logits.

  lora    out[m] = y[m] + scale[id] * (x[m] A[id]^T) B[id]^T, id = ids[m]; a negative id leaves the row as it is
  gemm    out[m] = bf16(x[m] W^T + scale[id] * (x[m] A[id]^T) B[id]^T), W = GGUF rows (Q4_K, Q6_K, Q8_0, F16)
  logits  out[m] = mask(penalties(logits[m]) + bias[m]) and its greedy token

The plain forms are elementary torch operations in 32 bits; `exact` restates the definitions in 64 bits.
"""
import numpy as np
import torch

own = False

BLOCK = {"Q4_K": (256, 144), "Q6_K": (256, 210), "Q8_0": (32, 34), "F16": (1, 2)}
WTYPE = {"Q4_K": 0, "Q6_K": 1, "Q8_0": 2, "F16": 3}  # the library's type codes
WEIGHT_SIZE = {"Q4_K": 0.8, "Q6_K": 0.9, "Q8_0": 0.25, "F16": 0.02}  # root mean square of the weights made here
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------ cases
def lora(name, M, K, N, R, L, at="bf16", yt="bf16", order="mixed", none=0, ranks="same"):
    return {"name": name, "op": "lora", "M": M, "K": K, "N": N, "R": R, "L": L, "at": at, "yt": yt, "order": order,
            "none": none, "ranks": ranks}


def gemm(name, wt, M, K, N, R, L, order="mixed", none=0, ranks="same"):
    return {"name": name, "op": "gemm", "wt": wt, "M": M, "K": K, "N": N, "R": R, "L": L, "at": "bf16", "yt": "bf16",
            "order": order, "none": none, "ranks": ranks}


def logits(name, M, V, history, lt="bf16", shared=False, bias=0, masks=0):
    return {"name": name, "op": "logits", "M": M, "V": V, "history": history, "lt": lt, "shared": shared, "bias": bias,
            "masks": masks}


def listed():
    return [
        # one user's token through a square projection: latency
        lora("add 1 row", M=1, K=4096, N=4096, R=16, L=4),
        # a decode batch: many users, adapters of several ranks, some users without one
        lora("add 64 rows, 32 adapters", M=64, K=4096, N=4096, R=64, L=32, none=5, ranks="mixed"),
        # prompts of eight users packed behind one another
        lora("add 4096 rows in runs", M=4096, K=6144, N=2048, R=32, L=8, order="runs"),
        # odd sizes, half-precision adapters as an F16 file holds them, a 32-bit result kept
        lora("add 77 rows, odd sizes", M=77, K=1000, N=2051, R=13, L=5, at="fp16", yt="fp32", none=3),
        # the same beside a quantised projection: one token, a small batch, packed prompts, an odd width
        gemm("Q4_K 1 row", "Q4_K", M=1, K=4096, N=4096, R=16, L=4),
        gemm("Q6_K 8 rows", "Q6_K", M=8, K=2048, N=6144, R=32, L=8, none=1),
        gemm("Q4_K 2048 rows in runs", "Q4_K", M=2048, K=6144, N=2048, R=16, L=8, order="runs"),
        gemm("Q8_0 24 rows, odd width", "Q8_0", M=24, K=4096, N=1003, R=8, L=24, ranks="mixed"),
        # one chat with penalties; a verify pass of seven drafts under a grammar; a full decode batch; a wide batch
        # of an odd vocabulary in 32 bits
        logits("logits 1 row", M=1, V=32000, history=500),
        logits("logits 8 verify rows", M=8, V=128000, history=4000, shared=True, bias=40, masks=8),
        logits("logits 64 rows", M=64, V=128000, history=8000, bias=100, masks=3),
        logits("logits 256 rows, odd", M=256, V=50001, history=1000, lt="fp32", bias=10),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["lora", "gemm", "logits"])
    while True:
        if op == "logits":
            V = _log(rng, 1000, 160000)
            M = _log(rng, 1, 256)
            c = logits("", M, V, _log(rng, 1, 16000), lt=rng.choice(["bf16", "fp32"]), shared=rng.random() < 0.3 and M <= 16,
                       bias=rng.choice([0, 1, 17, 300]), masks=rng.choice([0, 1, M]))
            top = 100e6
        else:
            L = _log(rng, 1, 64)
            M = _log(rng, 1, 4096)
            a = dict(R=_log(rng, 1, 128), L=L, order=rng.choice(["mixed", "runs"]), none=rng.choice([0, M // 7]),
                     ranks=rng.choice(["same", "mixed"]))
            if op == "lora":
                K, N = _log(rng, 64, 8192), _log(rng, 64, 8192)
                if rng.random() < 0.7:
                    K, N = max(64, K // 64 * 64), max(64, N // 64 * 64)
                c = lora("", M, K, N, at=rng.choice(["bf16", "fp16"]), yt=rng.choice(["bf16", "fp32"]), **a)
                top = 88e6
            else:
                wt = rng.choice(list(BLOCK))
                K, N = 256 * _log(rng, 1, 32), _log(rng, 64, 8192)
                if rng.random() < 0.7:
                    N = max(64, N // 64 * 64)
                c = gemm("", wt, M, K, N, **a)
                top = 40e6
                # the library has its tensor-core prefill for Q4_K and Q6_K; the other types are for decode batches
                if (wt in ("Q8_0", "F16") and M > 32) or 2 * M * K * N > 2 * 2048 * 6144 * 2048:
                    continue
        if work(c)["bytes"] <= top:
            del c["name"]
            return c


# ------------------------------------------------------------------------------------------------ inputs
def _ranks(case):
    """The adapters' ranks: the padded rank, or that and its half and quarter in turn."""
    return [case["R"] if case["ranks"] == "same" else max(1, case["R"] >> (n % 3)) for n in range(case["L"])]


def _adapted(case):
    """Rows with an adapter; adapters 0 .. min(L, rows) - 1 all have one."""
    return case["M"] - case["none"]


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)


def _ids(case, g):
    n, L = _adapted(case), case["L"]
    if case["order"] == "runs":  # every adapter's rows behind one another, in runs of uneven lengths
        k = min(L, n)
        cuts = torch.randperm(max(n - 1, 1), device="cuda", generator=g)[:max(k - 1, 0)].add(1).sort().values
        ids = torch.bucketize(torch.arange(n, device="cuda"), cuts, right=True)
    else:
        ids = torch.arange(n, device="cuda") % L
        ids = ids[torch.randperm(n, device="cuda", generator=g)]
    at = torch.randperm(case["M"], device="cuda", generator=g)[:n].sort().values
    full = torch.full((case["M"],), -1, dtype=torch.int32, device="cuda")
    full[at] = ids.to(torch.int32)
    return full


def _rows(wt, N, K, g):
    """N rows of K weights in GGUF blocks: random codes, scales as the formats have them."""
    if wt == "F16":
        return _randn(g, N, K, std=0.02, dtype=torch.float16).view(torch.uint8)
    weights, size = BLOCK[wt]
    n = N * K // weights
    b = torch.randint(0, 256, (n, size), device="cuda", generator=g, dtype=torch.uint8)
    d = (torch.randn(n, 2, device="cuda", generator=g).abs() * 2.0 ** -8).to(torch.float16).view(torch.uint8)
    if wt == "Q4_K":
        b[:, 0:4] = d
    elif wt == "Q6_K":
        b[:, 192:208] = torch.randint(-32, 32, (n, 16), device="cuda", generator=g, dtype=torch.int8).view(torch.uint8)
        b[:, 208:210] = d[:, :2]
    else:
        b[:, 0:2] = d[:, :2]
    return b.view(N, -1)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": case}
    M = case["M"]
    if case["op"] != "logits":
        K, N, R, L = (case[k] for k in "KNRL")
        at, yt = DTYPE[case["at"]], DTYPE[case["yt"]]
        s["x"] = _randn(g, M, K)
        s["a"] = _randn(g, L, R, K, std=K ** -0.5, dtype=at)
        # the adapters' share of a result is about a third: large enough to tell in 16 bits
        size = 1.0 if case["op"] == "lora" else WEIGHT_SIZE[case["wt"]] * K ** 0.5
        s["b"] = _randn(g, L, N, R, std=0.3 * size * R ** -0.5, dtype=at)
        s["scale"] = torch.rand(L, device="cuda", generator=g) + 0.5
        s["ranks"] = torch.tensor(_ranks(case), dtype=torch.int32, device="cuda")
        s["ids"] = _ids(case, g)
        if case["op"] == "lora":
            s["y"] = _randn(g, M, N, dtype=yt)
        else:
            s["w"] = _rows(case["wt"], N, K, g)
        return s
    V, H = case["V"], case["history"]
    s["logits"] = _randn(g, M, V, std=3.0, dtype=DTYPE[case["lt"]])
    # contexts: skewed token frequencies; verify rows share one context that grows by a draft a row
    if case["shared"]:
        T = H + M
        begin = torch.zeros(M, dtype=torch.int64, device="cuda")
        end = H + torch.arange(M, device="cuda")
    else:
        lens = torch.randint(H // 2, H + 1, (M,), device="cuda", generator=g)
        end = lens.cumsum(0)
        begin, T = end - lens, H * M
    u = torch.rand(T, device="cuda", generator=g)
    s["tokens"] = ((V + 1.0) ** u - 1).to(torch.int32).clamp_(0, V - 1)
    half = (begin + end) // 2  # half prompt, half answer
    s["spans"] = torch.stack([begin, half, end], 1).contiguous()
    s["penalties"] = torch.rand(M, 3, device="cuda", generator=g) * 0.5 + torch.tensor([1.0, 0.0, 0.0], device="cuda")
    s["bias_begin"] = s["bias_ids"] = s["bias_vals"] = s["mask"] = s["mask_rows"] = None
    if case["bias"]:
        n = case["bias"]
        s["bias_begin"] = torch.arange(M + 1, device="cuda") * n
        ids = torch.rand(M, V, device="cuda", generator=g).topk(n, dim=1).indices  # distinct in a row, as a map's keys
        s["bias_ids"] = ids.reshape(-1).to(torch.int32)
        s["bias_vals"] = torch.randn(M * n, device="cuda", generator=g) * 2
    if case["masks"]:
        G, W = case["masks"], (V + 31) // 32
        p = torch.rand(G, 1, 1, device="cuda", generator=g)  # from nearly closed to nearly open grammars
        bits = torch.rand(G, W, 32, device="cuda", generator=g) < p
        words = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(2)
        s["mask"] = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
        s["mask_rows"] = (torch.arange(M, device="cuda") % (G + 1) - (1 if G < M else 0)).to(torch.int32)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _bytes_f16(b):
    return b.contiguous().view(torch.float16).to(torch.float32)


def _dequant(wt, w, N, K):
    """GGUF rows as fp32 [N, K]."""
    if wt == "F16":
        return w.view(torch.float16).to(torch.float32).view(N, K)
    weights, size = BLOCK[wt]
    b = w.view(-1, size)
    if wt == "Q8_0":
        return (_bytes_f16(b[:, 0:2]) * b[:, 2:].view(torch.int8).to(torch.float32)).view(N, K)
    if wt == "Q6_K":
        lo, hi = b[:, :128].view(-1, 2, 64), b[:, 128:192].view(-1, 2, 32)
        low = torch.cat([lo & 15, lo >> 4], 2)  # [block, half, 128]
        top = torch.cat([hi & 3, (hi >> 2) & 3, (hi >> 4) & 3, hi >> 6], 2)
        q = (low.to(torch.int16) + 16 * top.to(torch.int16) - 32).to(torch.float32).view(-1, 16, 16)
        sc = b[:, 192:208].view(torch.int8).to(torch.float32).unsqueeze(2)
        return (_bytes_f16(b[:, 208:210]).unsqueeze(2) * sc * q).view(N, K)
    t, q = b[:, 4:16], b[:, 16:].view(-1, 4, 32)
    sc = torch.cat([t[:, 0:4] & 63, (t[:, 8:12] & 15) | ((t[:, 0:4] >> 6) << 4)], 1).to(torch.float32)
    mn = torch.cat([t[:, 4:8] & 63, (t[:, 8:12] >> 4) | ((t[:, 4:8] >> 6) << 4)], 1).to(torch.float32)
    q = torch.stack([q & 15, q >> 4], 2).view(-1, 8, 32).to(torch.float32)
    return ((_bytes_f16(b[:, 0:2]) * sc).unsqueeze(2) * q - (_bytes_f16(b[:, 2:4]) * mn).unsqueeze(2)).view(N, K)


def _plain_delta(s):
    """scale * (x A^T) B^T of every row, fp32 [M, N]: the products with all adapters at once, those of other rows' adapters
    (and of the columns past an adapter's rank) set to zero in between."""
    c = s["case"]
    M, K, N, R, L = (c[k] for k in "MKNRL")
    h = (s["x"].to(torch.float32) @ s["a"].to(torch.float32).view(L * R, K).t()).view(M, L, R)
    one = torch.arange(L, device=h.device)
    keep = (s["ids"].view(M, 1) == one).unsqueeze(2) & (torch.arange(R, device=h.device) < s["ranks"].view(L, 1))
    h = torch.where(keep, h * s["scale"].view(L, 1), 0.0).view(M, L * R)
    return h @ s["b"].to(torch.float32).transpose(1, 2).reshape(L * R, N)


def _plain_logits(s):
    c = s["case"]
    M, V = c["M"], c["V"]
    z = s["logits"].to(torch.float32)
    begin, gen, end = s["spans"].unbind(1)
    pos = begin.view(M, 1) + torch.arange(c["history"] + M, device=z.device)
    inside = pos < end.view(M, 1)
    tok = s["tokens"][pos.clamp_max(s["tokens"].numel() - 1)].long() + V * torch.arange(M, device=z.device).view(M, 1)
    seen = torch.bincount(tok[inside], minlength=M * V).view(M, V) > 0
    count = torch.bincount(tok[inside & (pos >= gen.view(M, 1))], minlength=M * V).view(M, V).to(torch.float32)
    rep, pres, freq = (s["penalties"][:, n].view(M, 1) for n in range(3))
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - freq * count
    z = z - pres * (count > 0).to(torch.float32)
    if s["bias_ids"] is not None:
        row = torch.arange(M, device=z.device).repeat_interleave(s["bias_begin"].diff())
        z = z.index_put((row, s["bias_ids"].long()), s["bias_vals"], accumulate=True)
    if s["mask"] is not None:
        bits = (s["mask"].unsqueeze(2) >> torch.arange(32, device=z.device, dtype=torch.int32)) & 1
        allowed = bits.view(s["mask"].shape[0], -1)[:, :V] != 0
        rows = s["mask_rows"].long()
        z = torch.where(allowed[rows.clamp_min(0)] | (rows < 0).view(M, 1), z, float("-inf"))
    best = z.max(dim=1, keepdim=True).values
    first = torch.where(z == best, torch.arange(V, device=z.device), V).min(dim=1).values
    return z, torch.where(best.view(M) == float("-inf"), -1, first).to(torch.int32)


def run(s):
    c = s["case"]
    if own:
        from aipu_b200 import ops

        if c["op"] == "logits":
            ctl = ops.LogitControls(tokens=s["tokens"], spans=s["spans"], penalties=s["penalties"],
                                    bias_begin=s["bias_begin"], bias_ids=s["bias_ids"], bias_vals=s["bias_vals"],
                                    mask=s["mask"], mask_rows=s["mask_rows"])
            return ops.process_logits(s["logits"], ctl)
        ad = ops.LoraAdapters(a=s["a"], b=s["b"], scale=s["scale"], ranks=s["ranks"])
        if c["op"] == "lora":
            return ops.lora_add(ad, s["ids"], s["x"], s["y"])
        return ops.gemm_lora(WTYPE[c["wt"]], s["w"], c["N"], c["K"], s["x"], ad, s["ids"])
    if c["op"] == "logits":
        return _plain_logits(s)
    if c["op"] == "lora":
        return (s["y"].to(torch.float32) + _plain_delta(s)).to(s["y"].dtype)
    w = _dequant(c["wt"], s["w"], c["N"], c["K"])
    return (s["x"].to(torch.float32) @ w.t() + _plain_delta(s)).to(torch.bfloat16)


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_weights(wt, raw, N, K):
    """The formats' definitions weight by weight (in the order of a row), on a numpy array of the row bytes."""
    f16 = lambda b: np.ascontiguousarray(b).view(np.float16).astype(np.float64)  # noqa: E731
    if wt == "F16":
        return f16(raw).reshape(N, K)
    weights, size = BLOCK[wt]
    blk = raw.reshape(-1, size)
    p = np.arange(weights)
    if wt == "Q8_0":
        return (f16(blk[:, :2]) * blk[:, 2:].view(np.int8)).reshape(N, K)
    if wt == "Q6_K":
        half, run_, n = p // 128, p % 128 // 32, p % 32
        low = blk[:, 64 * half + 32 * (run_ % 2) + n] >> (4 * (run_ // 2)).astype(np.uint8) & 15
        top = blk[:, 128 + 32 * half + n] >> (2 * run_).astype(np.uint8) & 3
        q = low.astype(np.int32) + 16 * top.astype(np.int32) - 32
        return (f16(blk[:, 208:210]) * blk[:, 192 + p // 16].view(np.int8) * q).reshape(N, K)
    j = np.arange(8)
    t = blk[:, 4:16].astype(np.int32)
    near, far = t[:, j % 4], t[:, 4 + j % 4]
    both = t[:, 8 + j % 4]
    sc = np.where(j < 4, near & 63, (both & 15) + 16 * (near >> 6))
    mn = np.where(j < 4, far & 63, (both >> 4) + 16 * (far >> 6))
    sub = p // 32
    q = blk[:, 16 + 32 * (sub // 2) + p % 32] >> (4 * (sub % 2)).astype(np.uint8) & 15
    return (f16(blk[:, 0:2]) * sc[:, sub] * q - f16(blk[:, 2:4]) * mn[:, sub]).reshape(N, K)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] != "logits":
        x = s["x"].double()
        if case["op"] == "lora":
            out = s["y"].double()
        else:
            w = _exact_weights(case["wt"], s["w"].cpu().numpy(), case["N"], case["K"])
            out = x @ torch.from_numpy(np.ascontiguousarray(w)).cuda().t()
        for n, r in enumerate(_ranks(case)):
            m = (s["ids"] == n).nonzero().view(-1)
            h = x[m] @ s["a"][n, :r].double().t()
            out[m] += s["scale"][n].double() * (h @ s["b"][n, :, :r].double().t())
        return out
    z = s["logits"].double().cpu().numpy()
    host = {k: v.cpu().numpy() for k, v in s.items() if torch.is_tensor(v) and k != "logits"}
    V = case["V"]
    for m in range(case["M"]):
        b, g, e = host["spans"][m]
        rep, pres, freq = host["penalties"][m].astype(np.float64)
        ids = np.unique(host["tokens"][b:e])
        z[m, ids] = np.where(z[m, ids] > 0, z[m, ids] / rep, z[m, ids] * rep)
        ids, n = np.unique(host["tokens"][g:e], return_counts=True)
        z[m, ids] -= freq * n + pres
        if case["bias"]:
            i = slice(host["bias_begin"][m], host["bias_begin"][m + 1])
            np.add.at(z[m], host["bias_ids"][i], host["bias_vals"][i].astype(np.float64))
        if case["masks"] and host["mask_rows"][m] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_rows"][m]].view(np.uint8), bitorder="little")[:V]
            z[m, bits == 0] = -np.inf
    return torch.from_numpy(z), None  # which token is first goes by the 32-bit values


def work(case):
    M = case["M"]
    if case["op"] == "logits":
        V, H = case["V"], case["history"]
        size = 2 if case["lt"] == "bf16" else 4
        context = H + M if case["shared"] else M * H * 3 // 4
        b = M * V * (size + 4) + 4 * context + 8 * M * case["bias"] + min(case["masks"], M) * ((V + 31) // 32) * 4 + 40 * M
        return {"bytes": b, "flops": 6 * M * V + context}
    K, N = case["K"], case["N"]
    n = _adapted(case)
    ranks = _ranks(case)[:min(case["L"], n)]
    ysize = 2 if case["yt"] == "bf16" else 4
    b = 2 * M * K + sum(ranks) * (K + N) * 2 + 4 * M + ysize * M * N
    f = 2 * n * (K + N) * (sum(ranks) / max(len(ranks), 1))
    if case["op"] == "lora":
        return {"bytes": b + ysize * M * N, "flops": int(f)}
    weights, size = BLOCK[case["wt"]]
    return {"bytes": b + N * K // weights * size, "flops": int(f + 2 * M * N * K)}
