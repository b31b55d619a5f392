"""GPU: the serving operators at the edges of what their documentation allows: scales at the ends of their range, values that are not finite
numbers, pages of very different scales, calls that the status word has to report, and inputs that lie elsewhere in memory than usual."""
import ctypes as C
import math

import pytest
import torch

from tests import serving_ref as ref
from tests.test_serving_gpu import _close, _packed, _pool, _prompt_reference, _starts

pytestmark = pytest.mark.gpu
NAN = float("nan")


@pytest.fixture(autouse=True)
def _status_is_clean():
    yield
    import flashmhf_b200 as fm
    fm.check_device_status()


@pytest.mark.parametrize("hd,scale,size", [(64, 2.0 ** -102, 2.0 ** 50), (96, -2.0 ** -111, 2.0 ** 55), (64, 0.0, 2.0 ** 58), (128, 2.0 ** -130, 2.0 ** 60),
                                           (64, 2.0 ** 100, 2.0 ** -52)])
def test_prompt_attention_scales_near_the_ends_of_their_range(hd, scale, size):
    """Large queries and keys under a scale that brings their scores back, and the other way round: the scale is taken as it is, however small.
    A score is off by the roundings that test_prompt_attention_scales_and_scores_that_grow counts, and three more: of the scale, of its product with
    log2(e), and of the score times it."""
    import flashmhf_b200 as fm
    n = [130, 40]
    q, k, v = _packed(sum(n), 4, hd, 1, size), _packed(sum(n), 2, hd, 2, size), _packed(sum(n), 2, hd, 3)
    want, want_lse, room = _prompt_reference(q, k, v, n, n, scale, True)
    most = float(q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()) * abs(scale)
    off = most * (hd / 16 * 2.0 ** -22 + 6 * 2.0 ** -24)
    o, lse = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), ref.ints(_starts(n)), scale=scale, return_lse=True)
    _close(o, want, room * (1 + 2 * off * 2.0 ** 8), lse, want_lse)


@pytest.mark.parametrize("lq,lk", [(300, 300), (300, 301), (300, 427), (300, 299), (130, 700)])
@pytest.mark.parametrize("bad", [0, 100, 255, 256, 290])
def test_prompt_attention_values_that_are_no_numbers_reach_127_rows_at_most(lq, lk, bad):
    """Whatever the difference between rows and keys: row r sees key c where c <= r + lk - lq, and a value at c that is not a number may reach
    the 127 rows before its own, no other row that does not see it."""
    import flashmhf_b200 as fm
    q, k, v = _packed(lq + 9, 2, 64, 1), _packed(lk + 9, 2, 64, 2), _packed(lk + 9, 2, 64, 3)
    cu_q, cu_k = ref.ints([0, lq, lq + 9]), ref.ints([0, lk, lk + 9])
    clean = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k)
    v[bad] = NAN
    o = fm.prompt_attention(q.cuda(), k.cuda(), v.cuda(), cu_q, cu_k)
    own = bad - (lk - lq)                      # the first row that sees it
    untouched = torch.ones(lq + 9, dtype=torch.bool)
    untouched[max(0, own - 127):lq] = False
    assert torch.equal(o.cpu()[untouched], clean.cpu()[untouched])
    assert bool(o.cpu()[max(0, own):lq].isnan().all())
