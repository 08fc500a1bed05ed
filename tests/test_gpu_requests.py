"""The per-request operators together, as a verify pass uses them: token rows, LM head, the request's head adapter, its
controls, the greedy token. Passes of K + 1 rows must commit the stream of decoding one row at a time, and the tokens
those of the definition in 64 bits."""
import numpy as np
import pytest
import torch

from aipu_b200 import ops
from aipu_b200.spec import Request, SpecVerifier

pytestmark = pytest.mark.gpu


def _verifier(V=1001, H=256, adapters=3, seed=0):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    d = torch.device("cuda", 0)
    g = torch.Generator().manual_seed(seed)

    def r(*s, std):
        return (torch.randn(s, generator=g) * std).to(torch.bfloat16).to(d)

    ad = ops.LoraAdapters(r(adapters, 16, H, std=H ** -0.5), r(adapters, V, 16, std=0.5))
    return SpecVerifier(r(V, H, std=1.0), r(V, H, std=0.1), lambda h: torch.tanh(h.float()).to(torch.bfloat16), head_adapters=ad)


def _definition(v, context, q, mask=None):
    """Processed logits of the token after `context`, in 64 bits."""
    h = torch.tanh(v.emb[context[-1]].float()).to(torch.bfloat16).double()
    z = v.lm_head.double() @ h
    if q.adapter >= 0:
        z = z + v.head_adapters.b[q.adapter].double() @ (v.head_adapters.a[q.adapter].double() @ h)
    z = z.cpu().numpy()
    ids = np.unique(context)
    z[ids] = np.where(z[ids] > 0, z[ids] / q.repetition, z[ids] * q.repetition)
    ids, n = np.unique(context[q.n_prompt:], return_counts=True)
    z[ids] -= q.frequency * n + q.presence
    for t, b in q.bias.items():
        z[t] += b
    if mask is not None:
        z[~mask] = -np.inf
    return z


def _grammar(V):
    """After a context of n tokens only those of the class n % 5 are allowed."""
    def allowed(n):
        return torch.arange(V) % 5 == n % 5
    return allowed, lambda context: ops.pack_mask(allowed(len(context))[None])[0]


def _request(V, kind):
    q = Request(context=[5, 17, 17, 3], n_prompt=3)
    if kind != "plain":
        q.repetition, q.presence, q.frequency, q.adapter = 1.3, 0.4, 0.2, 1
        q.bias = {7: 1.5, 900: -2.0, 3: 0.25}
    if kind == "grammar":
        q.mask = _grammar(V)[1]
    return q


@pytest.mark.parametrize("kind", ["plain", "controls", "grammar"])
@pytest.mark.parametrize("k", [0, 1, 4, 11])
def test_verify_passes_commit_the_stream_of_one_row_at_a_time(kind, k):
    v = _verifier()
    V = v.lm_head.shape[0]
    one, want = _request(V, kind), []
    for _ in range(24):
        (t,), _ = v.verify(one.context[-1], [], one)
        want.append(t)
    known = {}
    for a, b in zip([3] + want, want):
        known.setdefault(a, b)  # drafts that are right the first time a token comes

    def draft(tok, n):
        out = []
        for _ in range(n):
            tok = known.get(tok, 0)
            out.append(tok)
        return out

    q = _request(V, kind)
    assert v.generate(3, 24, draft, k, request=q) == want
    assert q.context == one.context == [5, 17, 17, 3] + want


@pytest.mark.parametrize("kind", ["plain", "controls", "grammar"])
def test_tokens_are_those_of_the_definition(kind):
    v = _verifier(seed=3)
    V = v.lm_head.shape[0]
    q = _request(V, kind)
    for _ in range(20):
        before = list(q.context)
        (t,), _ = v.verify(before[-1], [], q)
        mask = _grammar(V)[0](len(before)).numpy() if kind == "grammar" else None
        z = _definition(v, before, q, mask)
        # the logits are rounded to bf16 twice (head, adapter): 2^-8 each of at most the largest magnitude, and as much
        # again for the head's 32-bit sums rounding the other way; the chosen token can be this much below the best
        assert z[t] >= z.max() - 4 * 2.0 ** -8 * np.abs(z[np.isfinite(z)]).max()


def test_a_mask_that_leaves_nothing_ends_the_stream():
    v = _verifier()
    V = v.lm_head.shape[0]
    none = torch.zeros((V + 31) // 32, dtype=torch.int32)
    q = Request(context=[5, 3], mask=lambda c: none if len(c) >= 6 else None)
    out = v.generate(3, 50, lambda t, k: [0] * k, 3, request=q)
    assert len(out) == 4 and len(q.context) == 6


def test_requests_are_checked():
    v = _verifier()
    with pytest.raises(ValueError):
        v.verify(3, [], Request(context=[4]))
    with pytest.raises(ValueError):
        v.verify(3, [], Request(context=[]))
    with pytest.raises(ValueError):
        v.verify(3, [], Request(context=[3], adapter=3))
    assert v.stats.passes == 0


def test_pack_mask():
    allowed = torch.rand(3, 77) < 0.5
    w = ops.pack_mask(allowed)
    assert w.shape == (3, 3) and w.dtype == torch.int32
    assert torch.equal(torch.from_numpy(np.unpackbits(w.numpy().view(np.uint8), axis=1, bitorder="little")[:, :77]) != 0, allowed)
