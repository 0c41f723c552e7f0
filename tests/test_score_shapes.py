"""Token arrays and buffers of the right number of elements in another shape are refused, before anything needs a GPU."""
import pytest
import torch

from pcp_amd import scores
from pcp_amd._lib import PcpError

S, T, V, K = 3, 4, 10, 2


def arrays(*names, **other):
    return {n: other.get(n, torch.zeros(S, T)) for n in names}


@pytest.mark.parametrize("which", ["row_max", "log_sum", "entropy", "dlogp", "dentropy"])
@pytest.mark.parametrize("shape", [(T, S), (S * T,), (S, T, 1), (1, S * T), (2 * S, T // 2)])
def test_bwd_arrays(which, shape):
    x, ids = torch.zeros(S, T, V), torch.zeros(S, T, dtype=torch.int64)
    a = arrays("row_max", "log_sum", "entropy", "dlogp", "dentropy", **{which: torch.zeros(shape)})
    with pytest.raises(PcpError, match=r"must be \[S, TS\]"):
        scores.token_scores_bwd(x, ids, **a)


@pytest.mark.parametrize("which,shape", [("logp", (T, S)), ("entropy", (T, S)), ("row_max", (S * T,)), ("log_sum", (T, S)),
                                         ("top_logp", (T, S, K)), ("top_ids", (S, K, T)), ("top_ids", (S, T * K))])
def test_outputs_of_another_shape(which, shape):
    x, ids = torch.zeros(S, T, V), torch.zeros(S, T, dtype=torch.int64)
    out = scores.TokenScores(*(torch.zeros(S, T) for _ in range(4)), torch.zeros(S, T, K),
                             torch.zeros(S, T, K, dtype=torch.int32))
    setattr(out, which, torch.zeros(shape, dtype=getattr(out, which).dtype))
    with pytest.raises(PcpError, match="outputs do not fit"):
        scores.token_scores(x, ids, k=K, outputs=out)
