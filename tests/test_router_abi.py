"""The router's C entry points refuse what they cannot do before queuing any work, and size their workspaces
(none of these calls reaches the GPU)."""
BIG = 1 << 40


def _refused(native, code, *words):
    assert code == -1
    message = native.odie_error().decode()
    for word in words:
        assert word in message, message


def test_choose_refusals(native):
    forward, backward = native.odie_choose_forward, native.odie_choose_backward

    def f(logits=8, stride=64, n=4, experts=64, choices=2, normalize=1, dtype=0, expert=8, weights=8, stats=None):
        return forward(logits, stride, n, experts, choices, normalize, dtype, expert, weights, stats, 0)

    def b(upstream=8, expert=8, weights=8, logits=8, stride=64, stats=8, n=4, experts=64, choices=2, dtype=0, out=8):
        return backward(upstream, expert, weights, logits, stride, stats, n, experts, choices, dtype, out, 0)

    for call, what in ((f, 'odie_choose_forward'), (b, 'odie_choose_backward')):
        _refused(native, call(dtype=3), what, 'dtype')
        _refused(native, call(experts=0), what, 'experts')
        _refused(native, call(experts=32769, stride=40000), what, 'experts')
        _refused(native, call(choices=0), what, 'choices')
        _refused(native, call(choices=65, experts=70, stride=70), what, 'choices')
        _refused(native, call(choices=9, experts=8), what, 'choices')
        _refused(native, call(n=-1), what, 'rows')
        _refused(native, call(n=1 << 30), what, 'rows')
        _refused(native, call(stride=63), what, 'overlap')
        _refused(native, call(expert=None), what, 'null')
        _refused(native, call(weights=None), what, 'null')
        assert call(n=0) == 0
    _refused(native, f(logits=None), 'null')
    _refused(native, f(stats=4), 'stats', 'aligned')
    _refused(native, b(stats=None), 'null')
    _refused(native, b(upstream=None), 'null')
    _refused(native, b(out=None), 'null')


def test_balance_refusals(native):
    def f(logits=8, stride=64, expert=8, n=4, choices=2, experts=64, dtype=0, loss=8, counts=8, stats=None, norm=8,
          workspace=8, size=BIG):
        return native.odie_balance_forward(logits, stride, expert, n, choices, experts, dtype, loss, counts, stats, norm,
                                           workspace, size, 0)

    def b(upstream=8, logits=8, stride=64, counts=8, stats=16, norm=8, n=4, experts=64, dtype=0, out=8):
        return native.odie_balance_backward(upstream, logits, stride, counts, stats, norm, n, experts, dtype, out, 0)

    for call, what in ((f, 'odie_balance_forward'), (b, 'odie_balance_backward')):
        _refused(native, call(dtype=-1), what, 'dtype')
        _refused(native, call(experts=0), what, 'experts')
        _refused(native, call(n=-1), what, 'rows')
        _refused(native, call(n=1 << 31), what, 'rows')
        _refused(native, call(stride=63), what, 'overlap')
        _refused(native, call(logits=None), what, 'null')
        _refused(native, call(counts=None), what, 'null')
        _refused(native, call(norm=None), what, 'null')
    _refused(native, f(choices=0), 'choices')
    _refused(native, f(expert=None), 'null')
    _refused(native, f(loss=None), 'null')
    need = native.odie_balance_workspace(4, 2, 64)
    assert need > 0
    _refused(native, f(size=need - 1), 'workspace', str(need))
    _refused(native, f(workspace=4), 'aligned')
    _refused(native, f(workspace=None), 'workspace')
    _refused(native, f(stats=8), 'stats', 'aligned')
    _refused(native, b(stats=8), 'stats', 'aligned')
    assert native.odie_balance_workspace(-1, 2, 64) == -1 and native.odie_balance_workspace(1 << 30, 4, 64) == -1
    assert native.odie_balance_workspace(1 << 28, 4, 64) < 1 << 20
    _refused(native, b(stats=None), 'null')
    _refused(native, b(upstream=None), 'null')
    _refused(native, b(out=None), 'null')
    assert b(n=0) == 0


def test_distill_refusals(native):
    def f(logits=8, stride=64, ids=8, id_bytes=8, teacher=8, teacher_dtype=0, n=4, classes=64, top=2, temperature=1.0,
          dtype=0, loss=8, stats=None, workspace=8, size=BIG):
        return native.odie_distill_forward(logits, stride, ids, id_bytes, teacher, teacher_dtype, n, classes, top,
                                           temperature, dtype, loss, stats, workspace, size, 0)

    def b(upstream=8, logits=8, stride=64, ids=8, id_bytes=8, teacher=8, teacher_dtype=0, stats=8, n=4, classes=64, top=2,
          temperature=1.0, dtype=0, out=8):
        return native.odie_distill_backward(upstream, logits, stride, ids, id_bytes, teacher, teacher_dtype, stats, n,
                                            classes, top, temperature, dtype, out, 0)

    for call, what in ((f, 'odie_distill_forward'), (b, 'odie_distill_backward')):
        _refused(native, call(dtype=3), what, 'dtype')
        _refused(native, call(teacher_dtype=3), what, 'teacher_dtype')
        _refused(native, call(id_bytes=2), what, '4 or 8')
        _refused(native, call(classes=0), what, 'classes')
        _refused(native, call(classes=(1 << 24) + 1, stride=1 << 25), what, 'classes')
        _refused(native, call(top=0), what, 'entries')
        _refused(native, call(top=1025), what, 'entries')
        _refused(native, call(n=-1), what, 'rows')
        _refused(native, call(n=1 << 31), what, 'rows')
        for temperature in (0.0, -1.0, float('nan'), float('inf'), 1e-45):
            _refused(native, call(temperature=temperature), what, 'temperature')
        _refused(native, call(stride=63), what, 'overlap')
        _refused(native, call(logits=None), what, 'null')
        _refused(native, call(ids=None), what, 'null')
        _refused(native, call(teacher=None), what, 'null')
        assert call(n=0) == 0
    _refused(native, f(loss=None), 'null')
    _refused(native, b(stats=None), 'null')
    _refused(native, b(upstream=None), 'null')
    _refused(native, b(out=None), 'null')
    # few long rows are cut into pieces, whose maxima and sums are kept
    need = native.odie_distill_workspace(3, 70000, 2)
    assert need > 0
    _refused(native, f(n=3, classes=70000, stride=70000, dtype=2, size=need - 1), 'workspace', str(need))
    _refused(native, f(n=3, classes=70000, stride=70000, dtype=2, workspace=4), 'aligned')
    assert native.odie_distill_workspace(1 << 20, 70000, 2) == 0 and native.odie_distill_workspace(4, 64, 2) == 0
    assert native.odie_distill_workspace(-1, 64, 2) == -1
