"""More refusals of the cached attention that the arguments alone decide."""
import math

import pytest

from raptor_t_b200 import capi
from test_answering_api_cpu import P, _cache

lib = capi.lib


def _attend(scale=0.125, out=2 * P, q=P, qs=128, tokens=8):
    return lib.rt_cached_attention(out, q, qs, _cache(), P, 4, P, P, 1, tokens, 8, 0, 2, scale, 0, 0, None)


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 3e38])
def test_scale_that_is_no_number(scale):
    assert _attend(scale=scale) == 1 and b"scale" in lib.rt_last_error()


@pytest.mark.parametrize("out,q,qs,tokens", [(P, P, 128, 8), (P, P, 128, 1), (P, P + 256, 128, 8), (P + 7 * 256, P, 128, 8), (P + 240, P, 128, 1),
                                             (P, P + 16, 0, 8), (P + 256, P, 384, 3)])
def test_output_over_the_queries(out, q, qs, tokens):
    """Rows of 256 bytes, the queries' 2 qs apart."""
    rows = [(q + 2 * qs * i, q + 2 * qs * i + 256) for i in range(tokens)]
    assert any(a < out + 256 * tokens and out < b for a, b in rows)
    assert _attend(out=out, q=q, qs=qs, tokens=tokens) == 1 and b"overlaps" in lib.rt_last_error()
