"""Bias lists with repeated tokens: their sums in list order, and their time."""
import numpy as np
import pytest
import torch

from aipu_b200 import ops

pytestmark = pytest.mark.gpu


def _lists(V, n, repeats, M=3):
    """Rows of n distinct tokens and values; `repeats` of the entries name an earlier token of the row again."""
    rng = np.random.default_rng(n + repeats)
    ids, vals = [], rng.standard_normal((M, n)).astype(np.float32)
    for _ in range(M):
        t = rng.permutation(V)[:n].astype(np.int32)
        at = rng.permutation(np.arange(1, n))[:repeats]
        for i in sorted(at):
            t[i] = t[rng.integers(0, i)]
        ids.append(t)
    d = torch.device("cuda", 0)
    return ids, vals, ops.LogitControls(bias_begin=torch.arange(M + 1, device=d) * n, bias_ids=torch.from_numpy(np.concatenate(ids)).to(d),
                                        bias_vals=torch.from_numpy(vals.reshape(-1)).to(d))


@pytest.mark.parametrize("n,repeats", [(2, 1), (50, 3), (1000, 40), (1000, 64), (1000, 65), (1000, 90), (3000, 1), (3000, 1500)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float32])
def test_entries_of_a_token_are_added_in_list_order(n, repeats, t):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    V = 5003
    ids, vals, ctl = _lists(V, n, repeats)
    x = torch.randn((3, V), generator=torch.Generator().manual_seed(n)).to(t).cuda()
    z = x.float().cpu().numpy()
    for m in range(3):
        for i, v in zip(ids[m], vals[m]):
            z[m, i] = np.float32(z[m, i] + v)
    out, token = ops.process_logits(x, ctl)
    assert np.array_equal(out.cpu().numpy().view(np.uint32), z.view(np.uint32))
    assert token.cpu().tolist() == z.argmax(1).tolist()
    assert torch.equal(ops.greedy_tokens(x, ctl), token)


def test_one_repeat_does_not_make_every_entry_look_through_the_list():
    """Twice the entries with one repeat take twice as long at most, not four times."""
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    x = torch.randn((3, 32000), device="cuda")
    times = []
    for n in (10000, 20000):
        _, _, ctl = _lists(32000, n, 1)
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.greedy_tokens(x, ctl)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
    assert times[1] < 3 * times[0], times
