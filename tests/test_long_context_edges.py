"""The long-context operators at the ends of what their arguments allow: lengths and windows at the type's limits, weights
far below the largest, infinite and NaN values behind ranges that weigh nothing, workspaces kept over differing batches,
layers whose graphs outlive a buffer.  Oracle and tolerances are those of test_long_context.py."""
import pytest
import torch

from test_long_context import F16, Cache, _inputs, check, oracle, score_err


# ---------------------------------------------------------------------------------------------------------------------
# lengths and windows
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("window", [0, 1, 40, (1 << 31) - 1])
@pytest.mark.parametrize("P", [0, 2500])
def test_gpu_negative_lengths_are_empty(P, window, m355, cuda):
    """A length below zero is an empty context, whatever the window: zeros, and no score moves; the other sequences keep
    their results."""
    c = Cache(3, [P + 70, P + 33, P + 5], 2, 64, 16, F16, prefix=P)
    q, _ = _inputs(c, 3, 16, 1, False)
    want, mag, weights = oracle(c, q, [1] * 3, 0.125, window=window)
    kc, vc, bt, cl = c.device(cuda)
    sc = c.scores.to(cuda)
    for length in (-1, -2, -100, -(1 << 31)):
        lens = cl.clone()
        lens[1] = length
        before = sc.clone()
        st = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=cuda)
        for got in (m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, lens, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window),
                    m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, lens, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window, seq_starts=st, max_q=1),
                    m355.paged_attn_decode_scored(q.to(cuda), kc, vc, sc, bt, lens, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window)):
            assert (got[1] == 0).all()
            check(got[[0, 2]], want[[0, 2]], mag[[0, 2]], F16, score_err(c, q, 0.125))
        moved = (sc != before).cpu()
        page, off = c.slots(1)
        assert not moved[page[P:], :, off[P:]].any()
        page, off = c.slots(0)
        seen = weights[0].t()[P:] > 1e-6
        assert moved[page[P:], :, off[P:]][seen].all()
    # several tokens of a sequence that is shorter than they are many: the ones in front of it see nothing
    n = [2, 2, 5]
    c = Cache(4, [P + 70, 0, 3], 2, 64, 16, F16, prefix=P)
    q, _ = _inputs(c, 9, 16, 2, False)
    want, mag, _ = oracle(c, q, n, 0.125, window=window)
    kc, vc, bt, cl = c.device(cuda)
    cl[1] = -5
    st = torch.tensor([0, 2, 4, 9], dtype=torch.int32, device=cuda)
    got = m355.shared_prefix_attn(q.to(cuda), kc, vc, bt, cl, prefix_len=P, max_ctx=P + 70, scale=0.125, window=window, seq_starts=st, max_q=5)
    check(got, want, mag, F16, score_err(c, q, 0.125))
    assert (got[2:6] == 0).all()
