"""The 4-bit KV cache on the GPU, at the edges of its plans: cut units, scratch, strides, streams, refusals."""
import math

import pytest
import torch

from test_kv_fp4_gpu import attend, case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("q,seq", [(2000, 512), (5120, 576), (1500, 700), (2304, 513)])
@pytest.mark.parametrize("hq,d", [(1, 128), (2, 128), (1, 256), (1, 64)])
def test_more_new_tokens_than_keys_over_many_runs(q, seq, hq, d):
    """Rows before the first key weigh nothing: the few units that see keys are cut, every cut has its partial, and
    nothing of an earlier call's partials is merged."""
    cols = None if d == 128 else 4000  # a wide table says that the work may be large
    attend(case((700,), (9000,), 8, 1, d, seed=40, gain=4.0, cols=cols))  # leaves partials of every run behind
    c = case((q,), (seq,), hq, 1, d, seed=41, cols=cols)
    got = attend(c)
    check(c, got)
    assert (got[: q - seq] == 0).all()
    assert torch.equal(got, attend(c))
