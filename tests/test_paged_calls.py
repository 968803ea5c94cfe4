"""The calls of the paged cache without a GPU: arguments that never reach a kernel."""
import ctypes

import pytest

import einsummable_b200 as es
from einsummable_b200 import _lib
from test_paged import PTR, add_attention, append, attention, cache


@pytest.fixture
def km():
    m = es.kernel_manager_t.__new__(es.kernel_manager_t)  # no device: every call ends at the handle at the latest
    m._lib, m._h = _lib.load(), None
    yield m
    m._h = None


@pytest.mark.parametrize("missing", range(6))
def test_none_for_a_tensor_is_refused_by_the_library(km, missing):
    six = [None if i == missing else PTR for i in range(6)]
    for call in (lambda: km.paged_attention(attention(), None, *six), lambda: km.cache_append(append(), None, *six),
                 lambda: km.prefix_attention(attention(prefix_len=3), None, *six[:4], PTR, *six[4:])):
        with pytest.raises(es.es_error) as e:
            call()
        assert e.value.status == _lib.ES_BAD_ARGUMENT


def test_descriptors_are_not_taken_for_one_another(km):
    """A descriptor of the other kind is shorter or longer than what the library would read."""
    six = [PTR] * 6
    for call in (lambda: km.paged_attention(append(), None, *six), lambda: km.cache_append(attention(), None, *six),
                 lambda: km.prefix_attention(append(), None, *six, PTR), lambda: km.paged_attention_workspace(append())):
        with pytest.raises((TypeError, ctypes.ArgumentError)):
            call()


@pytest.mark.parametrize("dtype,most", [("f16", 1e26), ("f32", 1e30)])
def test_scales_whose_scores_pass_f32_are_refused(dtype, most):
    """256 x 65504^2 x 10^26 x log2 e: an f16 score and its lse are finite."""
    for scale in (1e-30, most):
        add_attention(attention(cache(dtype=dtype), scale=scale))
    for scale in (most * 1.01, 1e31, 1e-31):
        with pytest.raises(es.es_error) as e:
            add_attention(attention(cache(dtype=dtype), scale=scale))
        assert e.value.status == _lib.ES_BAD_DESCRIPTOR
