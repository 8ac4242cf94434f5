"""The 4-bit entry points refuse what they cannot do before queuing any work (none of these calls reaches the GPU)."""
import pytest


def _refused(native, code, *words):
    assert code == -1
    message = native.odie_error().decode()
    for word in words:
        assert word in message, message


def test_quantize_refusals(native):
    def q(x=16, stride=40, rows=4, width=40, dtype=1, codes=16, scales=16):
        return native.odie_mx_quantize(x, stride, rows, width, dtype, codes, scales, 0)

    def d(codes=16, scales=16, rows=4, width=40, dtype=1, x=16, stride=40):
        return native.odie_mx_dequantize(codes, scales, rows, width, dtype, x, stride, 0)

    for call, what in ((q, 'odie_mx_quantize'), (d, 'odie_mx_dequantize')):
        _refused(native, call(dtype=3), what, 'dtype')
        _refused(native, call(rows=-1), what, 'rows')
        _refused(native, call(rows=1 << 31), what, 'rows')
        _refused(native, call(width=0), what, 'width')
        _refused(native, call(width=(1 << 20) + 1, stride=1 << 21), what, 'width')
        _refused(native, call(stride=39), what, 'overlap')
        _refused(native, call(x=None), what, 'null')
        _refused(native, call(codes=None), what, 'null')
        _refused(native, call(scales=None), what, 'null')
        _refused(native, call(codes=8), what, 'aligned')
        _refused(native, call(scales=18), what, 'aligned')
        assert call(rows=0) == 0


@pytest.mark.parametrize('change,word', [
    (dict(dtype=3), 'dtype'), (dict(activation=6), 'activation'), (dict(rows=-1), 'rows'), (dict(rows=1 << 31), 'rows'),
    (dict(inputs=0), 'inputs'), (dict(outputs=(1 << 20) + 1), 'outputs'), (dict(experts=0), 'experts'),
    (dict(experts=4), 'offsets'), (dict(experts=1 << 16, offsets=8), 'experts'), (dict(x=None), 'null'),
    (dict(out=None), 'null'), (dict(codes=None), 'null'), (dict(scales=None), 'null'), (dict(x_stride=15), 'overlap'),
    (dict(out_stride=7), 'overlap'), (dict(residual=8, residual_stride=7), 'overlap'), (dict(codes=8), 'aligned'),
    (dict(scales=18), 'aligned'), (dict(x=8, x_scales=16), 'aligned'), (dict(x_scales=18), 'aligned')])
def test_linear_refusals(native, change, word):
    a = dict(x=16, x_scales=None, x_stride=16, rows=10, codes=16, scales=16, bias=None, residual=None, residual_stride=8,
             offsets=None, experts=1, inputs=16, outputs=8, dtype=1, activation=0, out=8, out_stride=8, pre=None, stream=0)
    a.update(change)
    _refused(native, native.odie_mx_linear_forward(*a.values()), 'odie_mx_linear_forward', word)
    a.update(dict(x=16, x_scales=16, codes=16, scales=16, out=8, rows=0, dtype=1, activation=0, inputs=16, outputs=8, experts=1))
    assert native.odie_mx_linear_forward(*a.values()) == 0      # nothing to do
