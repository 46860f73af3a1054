"""What drh_adamw decides on the host, over the stand-in for the HIP runtime: kernels do not run."""

from test_runtime_stand_in import program  # noqa: F401  (a fixture)

TENSORS = """
    a = np.zeros(1 << 16, np.float32)  # device memory
    steps = np.zeros(64, np.int64)

    def tensor(i, n=100, **places):  # the i-th tensor's arrays, 500 elements apart
        at = {k: addr(a) + 4 * (2500 * i + 500 * j) for j, k in enumerate(("param", "grad", "exp_avg", "exp_avg_sq"))}
        return _lib.AdamWTensor(**{**at, "step": addr(steps) + 8 * i, "n": n, **places})

    def call(*ts, dtype=0):
        f = lambda: _lib.check(_lib.lib().drh_adamw(ctx.handle, (_lib.AdamWTensor * len(ts))(*ts), len(ts), dtype, 32, .1, .9, .99, 0., 0., 0,
                                                    None, 0))
        return code(f)
"""


def test_a_gradient_that_is_written_is_refused(program):  # noqa: F811
    program(TENSORS + """
    t = [tensor(0), tensor(1)]
    assert launched(lambda: call(*t)) and call(*t) == 0
    for i in range(2):
        for where in ("param", "exp_avg", "exp_avg_sq"):
            for shift in (0, 99, -99):
                bad = tensor(1, grad=getattr(t[i], where) + 4 * shift)
                assert not launched(lambda: call(t[0], bad)) and call(t[0], bad) == 6, (i, where, shift)
                assert "gradient" in _lib.last_error()
            for shift in (100, -100):  # neighbours
                assert call(t[0], tensor(1, grad=getattr(t[i], where) + 4 * shift)) == 0
        assert call(t[0], tensor(1, grad=t[i].step - 4)) == 6 and call(t[0], tensor(1, grad=t[i].step + 4, n=1)) == 6
    assert call(t[0], tensor(1, grad=t[0].grad)) == 0  # two gradients
    assert call(t[0], tensor(1, grad=t[0].grad + 4 * 50)) == 0
    assert call(tensor(0), tensor(1, n=0, grad=t[0].param)) == 0  # of nothing
    # 16-bit elements: half as long
    assert call(tensor(0, n=200), tensor(1, grad=t[0].param + 200), dtype=1) == 6
    assert call(tensor(0, n=200), tensor(1, grad=t[0].param + 400), dtype=1) == 0
    """)


def test_no_memory_to_check_the_tensors(program):  # noqa: F811
    """An error, and no exception through the C entry."""
    program("""
    import resource
    n = 1 << 20
    table = (_lib.AdamWTensor * n)()
    steps = np.zeros(n, np.int64)
    np.frombuffer(table, np.int64).reshape(n, 8)[:, 6] = addr(steps) + 8 * np.arange(n)  # tensors of nothing
    call = lambda: code(lambda: _lib.check(_lib.lib().drh_adamw(ctx.handle, table, n, 0, 32, .1, .9, .99, 0., 0., 0, None, 0)))
    assert call() == 0
    used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
    resource.setrlimit(resource.RLIMIT_AS, (used + 4 * MIB, resource.RLIM_INFINITY))
    rc = call()
    resource.setrlimit(resource.RLIMIT_AS, (resource.RLIM_INFINITY, resource.RLIM_INFINITY))
    assert rc == 5 and "memory" in _lib.last_error(), rc
    assert call() == 0
    """)
