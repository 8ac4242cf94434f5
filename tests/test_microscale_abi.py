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


@pytest.mark.parametrize('change,word', [
    (dict(dtype=-1), 'dtype'), (dict(activation=9), 'activation'), (dict(rows=-3), 'rows'), (dict(experts=2), 'offsets'),
    (dict(inputs=0), 'inputs'), (dict(outputs=1 << 21), 'outputs'), (dict(experts=1 << 15, outputs=1 << 20, offsets=8), 'below 2^31'),
    (dict(upstream=None), 'null'), (dict(pre=None), 'null'), (dict(codes=None), 'null'), (dict(scales=None), 'null'),
    (dict(upstream_stride=7), 'overlap'), (dict(codes=8), 'aligned'), (dict(scales=18), 'aligned'), (dict(workspace=None), 'workspace'),
    (dict(workspace=128), 'aligned'), (dict(workspace_bytes=10), 'workspace')])
def test_linear_backward_refusals(native, change, word):
    for rows in (10, 100000):       # apart, and in one pass
        a = dict(upstream=8, upstream_stride=8, pre=8, rows=rows, codes=16, scales=16, offsets=None, experts=1, inputs=16, outputs=8,
                 dtype=1, activation=1, dx=8, dbias=8, workspace=256, workspace_bytes=1 << 40, stream=0)
        a.update(change)
        _refused(native, native.odie_mx_linear_backward(*a.values()), 'odie_mx_linear_backward', word)


def test_linear_workspace(native):
    size = native.odie_mx_linear_workspace
    # the weight as fp16, in rows of whole 16 bytes
    assert size(10, 1, 0, 64, 48, 1, 0, 1, 0) == 64 * 48 * 2
    assert size(100000, 1, 0, 60, 48, 1, 4, 1, 0) == 64 * 48 * 2        # one pass
    assert size(100000, 1, 0, 60, 48, 1, 4, 1, 1) > 64 * 48 * 2         # and sums of the bias' gradient
    assert size(10, 1, 0, 64, 48, 1, 4, 1, 0) >= 64 * 48 * 2 + 10 * 48 * 2      # dz
    assert size(10, 1, 0, 64, 48, 1, 0, 0, 0) == 0
    assert size(-1, 1, 0, 64, 48, 1, 0, 1, 0) == -1 and size(10, 2, 0, 64, 48, 1, 0, 1, 0) == -1
