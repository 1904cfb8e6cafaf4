"""What an unsupported call is told: the head sizes of the kernels among it."""
import ctypes


def test_unsupported_names_head_sizes(lib):
    lib.ua_strerror.restype = ctypes.c_char_p
    text = lib.ua_strerror(-3).decode()
    assert "head_dim 128" in text and "64" in text and "softmax_scale" in text and "element type" in text
