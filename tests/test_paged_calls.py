"""The calls of the paged cache without a GPU: arguments that never reach a kernel."""
import pytest

import einsummable_b200 as es
from einsummable_b200 import _lib
from test_paged import add_attention, attention, cache


@pytest.mark.parametrize("dtype,most", [("f16", 1e26), ("f32", 1e30)])
def test_scales_whose_scores_pass_f32_are_refused(dtype, most):
    """256 x 65504^2 x 10^26 x log2 e: an f16 score and its lse are finite."""
    for scale in (1e-30, most):
        add_attention(attention(cache(dtype=dtype), scale=scale))
    for scale in (most * 1.01, 1e31, 1e-31):
        with pytest.raises(es.es_error) as e:
            add_attention(attention(cache(dtype=dtype), scale=scale))
        assert e.value.status == _lib.ES_BAD_DESCRIPTOR
