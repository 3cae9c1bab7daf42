"""key_mass and cross_attention with several units per CTA (pair), in every form that walks them differently: against the formulas and bounds of
their own files."""
import pytest

import tests.test_cross_attention as cross
import tests.test_key_mass as weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,n_q,n_kv,hd,cap,lens,pad,decay", [
    (90, 20, 15, 1, 64, 600, None, True, 0.5),      # 300 query rows: two chunks, some 170 units on 74 pairs
    (100, 90, 4, 1, 128, 500, None, False, 1.0),    # 360
    (50, 40, 8, 1, 256, 1200, None, True, 0.5),     # 320: three chunks of 128
    (60, 100, 8, 1, 256, 700, None, False, 0.25),   # 800: seven, the groups' turns not a divisor
    (80, 50, 4, 1, 64, 900, None, False, 1.0),      # 200: one chunk of 256, two of the four parts in a group
    (120, 3, 8, 1, 256, 900, None, True, 0.5),      # one chunk that is one group's alone, more than four units per pair
    (300, 2, 6, 2, 64, 400, None, False, 1.0),
    (200, 1, 20, 5, 128, 300, None, True, 0.5),
])
def test_key_mass(B, S, n_q, n_kv, hd, cap, lens, pad, decay):
    weights.test_against_the_formula(B, S, n_q, n_kv, hd, cap, lens, pad, decay)


@pytest.mark.parametrize("B,S,n_q,n_kv,hd,cap,lens,pad", [
    (100, 50, 15, 5, 64, 241, None, True),     # 500 units on 148 CTAs: there, back and there again
    (250, 40, 8, 2, 128, 300, None, True),
    (200, 51, 8, 1, 256, 400, None, False),    # 400 units on 74 pairs
])
def test_cross_attention(B, S, n_q, n_kv, hd, cap, lens, pad):
    cross.test_against_the_formula(B, S, n_q, n_kv, hd, cap, lens, pad)
