"""What a Request's controls ask of its grammar and what a verify pass refuses, on the host."""
import pytest
import torch

from aipu_b200 import ops
from aipu_b200.spec import Request, SpecVerifier

V = 70


class Strict:
    """A matcher that follows contexts as a grammar does: after token t only t + 1 and t + 2 (mod V) may come, and a context
    that the grammar has refused cannot be asked about."""

    def __init__(self, free=()):
        self.asked, self.free = [], free  # free: lengths of contexts without a mask

    def __call__(self, context):
        self.asked.append(list(context))
        for a, b in zip(context, context[1:]):
            if (b - a) % V not in (1, 2):
                raise ValueError(f"the grammar does not know {list(context)}")
        if len(context) in self.free:
            return None
        ok = torch.zeros((1, V), dtype=torch.bool)
        ok[0, [(context[-1] + 1) % V, (context[-1] + 2) % V]] = True
        return ops.pack_mask(ok)[0]


@pytest.mark.parametrize("drafts,asked", [([6, 7, 9], 4), ([6, 9, 10], 2), ([5, 6], 1), ([6, 69, 0], 2), ([], 1), ([1000, 6], 1), ([-1, 6], 1)])
def test_masks_are_asked_for_up_to_the_first_refused_draft(drafts, asked):
    g = Strict()
    q = Request(context=[4, 5], mask=g)
    c = q.controls(drafts, "cpu")
    assert g.asked == [[4, 5] + drafts[:j] for j in range(asked)]
    assert c.mask.shape == (asked, 3) and c.mask.dtype == torch.int32
    assert c.mask_rows.tolist() == list(range(asked)) + [-1] * (len(drafts) + 1 - asked)


def test_a_context_without_a_mask_allows_every_draft():
    g = Strict(free=(2,))
    c = Request(context=[4, 5], mask=g).controls([6, 8, 11, 12], "cpu")
    assert len(g.asked) == 3 and c.mask_rows.tolist() == [-1, 0, 1, -1, -1]


def test_verify_rows_need_their_request():
    e = torch.zeros((V, 8), dtype=torch.bfloat16)
    v = SpecVerifier(e, e, lambda h: h)
    ad = ops.LoraAdapters(torch.zeros((2, 1, 8), dtype=torch.bfloat16), torch.zeros((2, V, 1), dtype=torch.bfloat16))
    w = SpecVerifier(e, e, lambda h: h, head_adapters=ad)
    for sv, q in ((v, Request(context=[4])), (v, Request(context=[])), (v, Request(context=[3], adapter=0)), (w, Request(context=[3], adapter=2))):
        for call in (lambda: sv.greedy_tokens([3, 5], q), lambda: sv.verify(3, [5], q)):
            with pytest.raises(ValueError, match="context must end with|does not have"):
                call()
    with pytest.raises(ValueError, match="n_prompt"):
        Request(context=[3], n_prompt=-1).controls([], "cpu")


@pytest.mark.parametrize("rows", [[V], [-1], [3, V], [3, 5, 1 << 40]])
def test_tokens_outside_the_embedding_are_refused(rows):
    """Before the device looks them up."""
    e = torch.zeros((V, 8), dtype=torch.bfloat16)
    v = SpecVerifier(e, e, lambda h: h)
    with pytest.raises(ValueError, match="outside"):
        v.greedy_tokens(rows)
    with pytest.raises(ValueError, match="outside"):
        v.verify(rows[0], rows[1:], Request(context=rows[:1]))


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1, 3, 9])
def test_drafts_that_the_grammar_refuses_change_nothing(k):
    """The stream of one row at a time, with drafts that are right, wrong and refused by the grammar."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    d, g = torch.device("cuda", 0), torch.Generator().manual_seed(1)
    emb, head = ((torch.randn((V, 64), generator=g) * s).to(torch.bfloat16).to(d) for s in (1.0, 0.1))
    v = SpecVerifier(emb, head, lambda h: torch.tanh(h.float()).to(torch.bfloat16))
    one, want = Request(context=[3], repetition=1.2, mask=Strict()), []
    for _ in range(20):
        want += v.verify(one.context[-1], [], one)[0]
    q, n = Request(context=[3], repetition=1.2, mask=Strict()), 0
    while len(q.context) <= 20:
        right = want[len(q.context) - 1:][:k]
        drafts = [t if (n + j) % 3 else (t + 7) % V for j, t in enumerate(right)]
        n += 1
        v.verify(q.context[-1], drafts, q)
    assert q.context[1:21] == want
