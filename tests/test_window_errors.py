"""Errors of the windowed prompt attention's C entry name that operator, those of the other the other."""
import ctypes
import math

from tests.test_prompt_refusals import Attention
from tests.test_serving_refusals import Window, lib  # noqa: F401


def test_errors_name_the_operator(lib):  # noqa: F811
    a = Window()
    a.prompt = Attention(*([4096] * 3), None, None, *([4096] * 3), None, None, 0, 1, 100, 100, 8, 8, 128, 1024, 128, 1024, 128, 1024, 128, 0, 0, 0, 0, 1024, 128, 0.1, 1, 0, 0)
    a.window = 5
    for field, value in (("b", 0), ("total_q", -1), ("heads", 7), ("d", 96), ("query_rope", 4096), ("softmax_scale", math.nan), ("query", None), ("key", 4104), ("query", 4097),
                         ("k_t", 1 << 40)):
        one = Window.from_buffer_copy(a)
        if field == "query_rope":
            one.prompt.d, one.prompt.key_rope = 64, 4096
        setattr(one.prompt, field, value)
        assert lib.pto_prompt_window_launch(ctypes.byref(one), None) == -1 and lib.pto_last_error().startswith(b"prompt_window_attention: "), (field, lib.pto_last_error())
        assert lib.pto_prompt_attention_launch(ctypes.byref(one.prompt), None) == -1 and lib.pto_last_error().startswith(b"prompt_attention: "), field
