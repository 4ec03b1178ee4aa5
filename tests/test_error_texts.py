"""The texts of the error codes name what each entry point's caller can look at."""

import pytest

from gdn_b200 import _lib


@pytest.mark.parametrize("code,words", [
    (_lib.GDN_ERR_SHAPE, ["128", "HV a multiple of H", "64, 128 or 256"]),
    (_lib.GDN_ERR_ALIAS, ["state and new_state", "overlap", "pool", "output"]),
    (_lib.GDN_ERR_ARG, ["rank or world", "scale", "window", "dtype", "eos_token"]),
    (_lib.GDN_ERR_LIMIT, ["0..63", "64 beams", "32 pools"]),
    (_lib.GDN_ERR_ALIGN, ["state", "16 B", "q/k 8 B"]),
])
def test_texts_name_the_arguments(gdn_lib, code, words):
    text = _lib.strerror(code)
    assert [w for w in words if w not in text] == []
