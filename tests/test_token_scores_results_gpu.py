"""What token_logprobs returns can be saved and copied."""
import io
import pickle

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from raptor_t_b200 import ops as _ops
    return _ops


@pytest.mark.parametrize("top", [0, 5])
@pytest.mark.parametrize("given", [False, True])
def test_scores_can_be_saved(ops, top, given):
    g = torch.Generator(device="cuda").manual_seed(1)
    z = torch.randn(7, 1000, device="cuda", generator=g)
    t = torch.arange(7, dtype=torch.int32, device="cuda") if given else None
    scores = ops.token_logprobs(z, t, top_k=top)
    file = io.BytesIO()
    torch.save(tuple(scores), file)
    file.seek(0)
    again = ops.TokenScores._make(torch.load(file))
    copy = pickle.loads(pickle.dumps(scores))
    for a, b, c in zip(scores, again, copy):
        if a is None:
            assert b is None and c is None
        else:
            assert a.dtype == b.dtype == c.dtype and torch.equal(a, b) and torch.equal(a, c)
