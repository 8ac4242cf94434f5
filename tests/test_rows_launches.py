"""Sizes whose workgroups one launch cannot take are refused by name before the launch."""
import pytest
import torch


def _refused(native, code):
    assert code == -1 and 'too many' in native.odie_error().decode(), native.odie_error().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason='the addresses are made up')
def test_too_many_workgroups(native):
    big = 1 << 60
    # 32768 experts of 16 rows each and 2^20 columns; their weight gradients, their bias gradients
    _refused(native, native.odie_linear_forward(256, 1, 1 << 19, 256, None, None, 0, 256, 1 << 15, 1, 1 << 20, 1, 0, 256,
                                                1 << 20, None, 0))
    _refused(native, native.odie_linear_backward(256, 1 << 20, 256, 8, None, 1 << 19, None, 256, 1 << 15, 8, 1 << 20, 1, 0,
                                                 None, 256, None, 256, big, 0))
    _refused(native, native.odie_linear_backward(256, 1 << 20, 256, 8, None, 1 << 19, None, 256, 1 << 15, 8, 1 << 20, 1, 0,
                                                 None, None, 256, 256, big, 0))
    # 2^31 - 1 rows of 1 MB, looked up and brought back
    most = (1 << 31) - 1
    _refused(native, native.odie_embed_forward(256, 1 << 18, 100, 256, 4, most, 1.0, 1 << 18, 0, 256, 0))
    _refused(native, native.odie_rows_combine(256, 1 << 18, 256, None, most, 1, 1 << 18, 0, 256, 0))
    _refused(native, native.odie_embed_backward(256, 1 << 18, 256, 4, most, 100, 1.0, 1 << 18, 0, 256, 256, big, 0))
