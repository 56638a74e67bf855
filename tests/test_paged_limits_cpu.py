"""The number of steps that paged attention deals out is held in 32 bits, with the end of the last piece behind it."""
import ctypes

import landmark_attention_b200 as P
from landmark_attention_b200 import _lib as L


def attend(heads, max_pages):
    one, s = ctypes.c_void_p(256), L.I64x3(128 * heads, 128, 8)        # never dereferenced
    return P.lib().lmk_paged_attend(one, s, one, one, s, s, one, one, one, None, 1.0, None, 0, 1, heads, heads, 1, 8, 16, 4, max_pages, 0, 0, 0.5,
                                    L.LMK_BF16, None)


def test_lines_of_nearly_2_to_the_31_steps_are_refused():
    assert 32767 * 65538 == 2 ** 31 - 2
    assert attend(32767, 65538) == L.LMK_ERR_INVALID and b"too many for one call" in P.lib().lmk_last_error()
    assert attend(32767, 70000) == L.LMK_ERR_INVALID
