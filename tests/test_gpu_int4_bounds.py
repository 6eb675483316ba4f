"""paged_attention_int4: what max_query_len may be.  Helpers and tolerances of test_gpu_int4_attention.py."""
import pytest
import torch

from test_gpu_int4_attention import check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,s,Hq,Hkv,D", [([1] * 20, [3 + 41 * i for i in range(20)], 8, 1, 128), ([4, 1, 9, 0, 30], [100, 40, 9, 7, 500], 4, 2, 64),
                                          ([140, 3], [200, 90], 4, 2, 128), ([20, 5], [70, 300], 2, 2, 256)])
def test_any_bound_on_the_rows(n, s, Hq, Hkv, D):
    """One, too few, exact, the call's rows and far more: every plan is within the bound of the 64-bit result."""
    c = make(sum(s), n, s, Hq, Hkv, D, 32, "f16", extra_rows=1)
    for most in (1, max(2, max(n) // 2), max(n), c["T"], 100 * c["T"]):
        c["n"] = [most]                                  # (what the helper hands over as max_query_len)
        out = check(c)
        assert torch.equal(check(c), out)
