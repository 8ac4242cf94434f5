"""The row operators' C entry points refuse what they cannot do before queuing any work, and size their workspaces
(none of these calls reaches the GPU)."""
import pytest

BIG = 1 << 40


def _refused(native, code, *words):
    assert code == -1
    message = native.odie_error().decode()
    for word in words:
        assert word in message, message


def test_sort_refusals(native):
    call = native.odie_sort
    _refused(native, call(8, 2, 10, 4, 8, None, None, None, 8, BIG, 0), 'odie_sort', '4 or 8')
    _refused(native, call(8, 4, -1, 4, 8, None, None, None, 8, BIG, 0), 'count')
    _refused(native, call(8, 4, 1 << 31, 4, 8, None, None, None, 8, BIG, 0), 'count')
    _refused(native, call(8, 4, 10, 0, 8, None, None, None, 8, BIG, 0), 'buckets')
    _refused(native, call(8, 4, 10, (1 << 31) - 1, 8, None, None, None, 8, BIG, 0), 'buckets')
    _refused(native, call(None, 4, 10, 4, 8, None, None, None, 8, BIG, 0), 'null')
    _refused(native, call(8, 4, 10, 4, None, None, None, None, 8, BIG, 0), 'null')
    need = native.odie_sort_workspace(5000, 64)
    assert need > 0 and need % 4 == 0
    _refused(native, call(16, 4, 5000, 64, 16, None, None, None, 16, need - 1, 0), 'workspace', str(need))
    _refused(native, call(16, 4, 5000, 64, 16, None, None, None, 24, need, 0), 'aligned')
    _refused(native, call(16, 4, 5000, 64, 16, None, None, None, None, need, 0), 'workspace')
    assert call(None, 4, 0, 64, None, None, None, None, None, 0, 0) == 0          # nothing to do
    assert native.odie_sort_workspace(4096, 1 << 30) == 0 and native.odie_sort_workspace(-1, 4) == -1
    # a (position, key) pair twice for each key where one pass does not tell the buckets apart
    assert native.odie_sort_workspace(1 << 20, 1 << 20) >= 16 << 20


def test_row_moves_refusals(native):
    dispatch, combine, gradient = native.odie_rows_dispatch, native.odie_rows_combine, native.odie_rows_combine_backward
    _refused(native, dispatch(8, 4, 8, 8, 10, 2, 3, 4, 3, 8, 0), 'dtype')
    _refused(native, dispatch(8, 4, 8, 8, 10, 0, 3, 4, 0, 8, 0), 'choices')
    _refused(native, dispatch(8, 4, 8, 8, 1 << 30, 2, 3, 4, 0, 8, 0), 'choices')
    _refused(native, dispatch(8, 4, 8, 8, 10, 2, 0, 4, 0, 8, 0), 'experts')
    _refused(native, dispatch(8, 4, 8, 8, 10, 2, 3, 0, 0, 8, 0), 'width')
    _refused(native, dispatch(8, 3, 8, 8, 10, 2, 3, 4, 0, 8, 0), 'overlap')
    _refused(native, dispatch(None, 4, 8, 8, 10, 2, 3, 4, 0, 8, 0), 'null')
    _refused(native, combine(8, 4, None, None, 10, 2, 4, 0, 8, 0), 'null')
    _refused(native, combine(8, 3, 8, None, 10, 2, 4, 0, 8, 0), 'overlap')
    _refused(native, gradient(8, 4, None, 4, 8, None, 8, 10, 2, 3, 4, 0, 8, 8, 0), 'null')      # dweights without rows
    _refused(native, gradient(8, 4, 8, 4, 8, None, None, 10, 2, 3, 4, 0, 8, None, 0), 'null')   # drows without offsets
    _refused(native, gradient(8, 4, 8, 2, 8, None, 8, 10, 2, 3, 4, 0, 8, 8, 0), 'overlap')
    for call in (dispatch(None, 4, None, None, 0, 2, 3, 4, 0, None, 0), combine(None, 4, None, None, 0, 2, 4, 0, None, 0),
                 gradient(None, 4, None, 4, None, None, None, 10, 2, 3, 4, 0, None, None, 0)):
        assert call == 0


@pytest.mark.parametrize('change,word', [
    (dict(dtype=3), 'dtype'), (dict(activation=6), 'activation'), (dict(rows=-1), 'rows'), (dict(rows=1 << 31), 'rows'),
    (dict(inputs=0), 'inputs'), (dict(outputs=(1 << 20) + 1), 'outputs'), (dict(experts=0), 'experts'),
    (dict(experts=4), 'offsets'), (dict(experts=1 << 16, offsets=8), 'experts'), (dict(x=None), 'null'),
    (dict(out=None), 'null'), (dict(weight=None), 'null'), (dict(x_stride=15), 'overlap'), (dict(out_stride=7), 'overlap'),
    (dict(residual=8, residual_stride=7), 'overlap')])
def test_linear_forward_refusals(native, change, word):
    a = dict(x=8, x_stride=16, rows=10, weight=8, bias=None, residual=None, residual_stride=8, offsets=None, experts=1,
             inputs=16, outputs=8, dtype=1, activation=0, out=8, out_stride=8, pre=None, stream=0)
    a.update(change)
    _refused(native, native.odie_linear_forward(*a.values()), 'odie_linear_forward', word)


@pytest.mark.parametrize('change,word', [
    (dict(dtype=-1), 'dtype'), (dict(activation=9), 'activation'), (dict(rows=-3), 'rows'), (dict(experts=2), 'offsets'),
    (dict(upstream=None), 'null'), (dict(pre=None), 'null'), (dict(x=None), 'null'), (dict(weight=None), 'null'),
    (dict(upstream_stride=7), 'overlap'), (dict(x_stride=15), 'overlap'), (dict(workspace=None), 'workspace'),
    (dict(workspace=128), 'aligned'), (dict(workspace_bytes=10), 'workspace')])
def test_linear_backward_refusals(native, change, word):
    a = dict(upstream=8, upstream_stride=8, x=8, x_stride=16, pre=8, rows=10, weight=8, offsets=None, experts=1, inputs=16,
             outputs=8, dtype=1, activation=1, dx=8, dweight=8, dbias=8, workspace=256, workspace_bytes=BIG, stream=0)
    a.update(change)
    _refused(native, native.odie_linear_backward(*a.values()), 'odie_linear_backward', word)


def test_linear_workspace(native):
    size = native.odie_linear_workspace
    # no activation, no bias, rows that one workgroup's piece covers: nothing to keep
    assert size(100, 1, 0, 64, 64, 1, 0, 1, 0) == 0
    # dz in the tensors' type, and partial sums of the bias
    assert size(1000, 1, 0, 64, 48, 1, 1, 0, 0) == 1000 * 48 * 2
    assert size(1000, 1, 0, 64, 48, 0, 1, 0, 0) == 1000 * 48 * 4
    assert size(1000, 1, 0, 64, 48, 1, 0, 0, 1) > 0
    # partial weight sums stay below twice the operands' bytes, plus a piece for each expert
    for rows, inputs, outputs in ((65536, 1024, 4096), (4096, 1024, 1024), (65536, 64, 64), (1 << 20, 32, 64)):
        assert size(rows, 1, 0, inputs, outputs, 2, 0, 1, 0) <= 2 * 2 * rows * (inputs + outputs) + 4 * inputs * outputs
    assert size(-1, 1, 0, 64, 64, 1, 0, 1, 0) == -1 and size(10, 2, 0, 64, 64, 1, 0, 1, 0) == -1


def test_embed_refusals(native):
    forward, backward = native.odie_embed_forward, native.odie_embed_backward
    _refused(native, forward(8, 4, 100, 8, 4, 10, 1.0, 4, 7, 8, 0), 'dtype')
    _refused(native, forward(8, 4, 100, 8, 3, 10, 1.0, 4, 0, 8, 0), '4 or 8')
    _refused(native, forward(8, 4, 0, 8, 4, 10, 1.0, 4, 0, 8, 0), 'vocab')
    _refused(native, forward(8, 3, 100, 8, 4, 10, 1.0, 4, 0, 8, 0), 'overlap')
    _refused(native, forward(8, 4, 100, None, 4, 10, 1.0, 4, 0, 8, 0), 'null')
    _refused(native, backward(8, 4, 8, 4, 10, 100, 1.0, 0, 0, 8, 256, BIG, 0), 'width')
    _refused(native, backward(8, 4, 8, 4, 10, 100, 1.0, 4, 0, None, 256, BIG, 0), 'null')
    _refused(native, backward(8, 3, 8, 4, 10, 100, 1.0, 4, 0, 8, 256, BIG, 0), 'overlap')
    need = native.odie_embed_workspace(10, 100, 4, 0)
    assert need > 0
    _refused(native, backward(8, 4, 8, 4, 10, 100, 1.0, 4, 0, 8, 256, need - 1, 0), 'workspace', str(need))
    _refused(native, backward(8, 4, 8, 4, 10, 100, 1.0, 4, 0, 8, 128, need, 0), 'aligned')
    assert forward(None, 4, 100, None, 4, 0, 1.0, 4, 0, None, 0) == 0
    assert native.odie_embed_workspace(-1, 100, 4, 0) == -1
