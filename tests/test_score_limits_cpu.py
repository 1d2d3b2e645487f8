"""CPU checks of the largest sizes of the token scores: what a kernel's 32-bit
row numbers cannot hold is refused before anything is launched."""
import pytest

from tests.test_paged_cpu import NULL, SCORE, SCORE_T, SHAPE, _call


@pytest.mark.parametrize("rows,rc", [((1 << 31) - 1, SHAPE), ((1 << 31) - 7, SHAPE), ((1 << 31) - 8, SHAPE), ((1 << 31) - 9, NULL)])
def test_rows_past_32_bits_of_the_last_cta_are_refused(rows, rc):
    """A CTA takes up to 8 rows: the last one counts up to rows + 7."""
    assert _call("fdl_token_logprobs", SCORE_T, SCORE, dict(rows=rows, x=None)) == rc
