"""C entry points of the post-training operators: pointers off their type's boundary are
refused on the host (a kernel would fault on them)."""

import ctypes

from llm_training_b200 import _lib

ERR_DTYPE, ERR_ALIGN = 2, 3  # include/sqrtblock.h
OK_PTR = 1 << 12


def vp(v):
    return ctypes.c_void_p(v)


def refused(call, names, aligned, steps):
    """Each named pointer off its boundary by each of its `steps` alone is refused; with all on
    theirs the call gets as far as the dtype that `aligned` has wrong."""
    for name in names:
        for step in steps[name]:
            assert call(**{name: OK_PTR + step}) == ERR_ALIGN, (name, step)
    assert call(**aligned) == ERR_DTYPE


def test_losses():
    lib = _lib.lib()

    def logp(x=OK_PTR, t=OK_PTR, logp=OK_PTR, stats=OK_PTR, dtype=0):
        return lib.sqb_logp_fwd(vp(x), vp(t), vp(logp), vp(stats), 1, 4, 8, 32, 8, dtype, None)

    def grad(x=OK_PTR, t=OK_PTR, stats=OK_PTR, g=OK_PTR, scale=OK_PTR, dx=OK_PTR, dtype=0):
        return lib.sqb_logp_bwd(vp(x), vp(t), vp(stats), vp(g), vp(scale), vp(dx), 1, 4, 8, 32, 8,
                                32, 8, dtype, None)

    def preference(x=OK_PTR, t=OK_PTR, cu=OK_PTR, ref=OK_PTR, loss=OK_PTR, rewards=OK_PTR,
                   stats=OK_PTR, g=OK_PTR, ws=OK_PTR, dtype=0):
        return lib.sqb_preference_fwd(vp(x), vp(t), vp(cu), vp(ref), 2, .1, 0., vp(loss),
                                      vp(rewards), vp(stats), vp(g), 1, 4, 8, 32, 8, dtype,
                                      vp(ws), 1 << 20, None)

    def policy(x=OK_PTR, t=OK_PTR, cu=OK_PTR, old=OK_PTR, ref=OK_PTR, adv=OK_PTR, loss=OK_PTR,
               statistics=OK_PTR, logp=OK_PTR, stats=OK_PTR, g=OK_PTR, dx=OK_PTR, ws=OK_PTR,
               dtype=0):
        return lib.sqb_policy_fwd(vp(x), vp(t), vp(cu), 4, vp(old), vp(ref), vp(adv), 1, .2, .2,
                                  0., 0, vp(loss), vp(statistics), vp(logp), vp(stats), vp(g),
                                  vp(dx), 1., 1, 4, 8, 32, 8, 32, 8, dtype, vp(ws), 1 << 20, None)

    steps = {"t": (4,), "cu": (4,), "stats": (4,), "ws": (4,)}
    for call in (logp, grad, preference, policy):
        names = call.__code__.co_varnames[:call.__code__.co_argcount]
        pointers = [n for n in names if n != "dtype"]
        refused(call, pointers, {"dtype": 9}, {n: steps.get(n, (1, 2)) for n in pointers})
    # bf16 elements need no more than their own boundary
    assert logp(x=OK_PTR + 1, dtype=1) == ERR_ALIGN
    assert grad(dx=OK_PTR + 1, dtype=1) == ERR_ALIGN
    assert policy(dx=OK_PTR + 1, dtype=1) == ERR_ALIGN


def test_gradient_norm():
    lib = _lib.lib()
    one = lambda kind, v: (kind * 1)(v)  # noqa: E731
    p, n, d = (one(k, v) for k, v in ((ctypes.c_void_p, OK_PTR), (ctypes.c_int64, 4),
                                      (ctypes.c_int32, 0)))

    def norm(ws=OK_PTR, norm=OK_PTR):
        return lib.sqb_grad_norm(p, n, d, 1, vp(ws), 1 << 20, vp(norm), None)

    def clip(ws=OK_PTR, norm=OK_PTR):
        return lib.sqb_grad_clip(p, p, n, d, d, 1, 1.0, vp(ws), 1 << 20, vp(norm), None)

    for call in (norm, clip):
        assert call(ws=OK_PTR + 4) == ERR_ALIGN and call(norm=OK_PTR + 2) == ERR_ALIGN


def test_residual_step():
    lib = _lib.lib()

    def fwd(x=OK_PTR, h=OK_PTR, w=OK_PTR, b=OK_PTR, wp=OK_PTR, bp=OK_PTR, gate=OK_PTR, xo=OK_PTR,
            y=OK_PTR, stats=OK_PTR, dtype=0):
        return lib.sqb_residual_norm_fwd(vp(x), 0, vp(h), 0, vp(w), vp(b), vp(wp), vp(bp), vp(gate),
                                         1, 1., 1e-5, 0, vp(xo), vp(y), dtype, vp(stats), 4, 8,
                                         None)

    def bwd(dy=OK_PTR, dxo=OK_PTR, x=OK_PTR, h=OK_PTR, w=OK_PTR, b=OK_PTR, wp=OK_PTR, bp=OK_PTR,
            gate=OK_PTR, stats=OK_PTR, dx=OK_PTR, dh=OK_PTR, dw=OK_PTR, db=OK_PTR, dwp=OK_PTR,
            dbp=OK_PTR, dgate=OK_PTR, ws=OK_PTR, dtype=0):
        return lib.sqb_residual_norm_bwd(vp(dy), dtype, vp(dxo), vp(x), 0, vp(h), 0, vp(w), vp(b),
                                         vp(wp), vp(bp), vp(gate), 1, 1., 1e-5, 0, vp(stats),
                                         vp(dx), vp(dh), vp(dw), vp(db), vp(dwp), vp(dbp),
                                         vp(dgate), vp(ws), 1 << 20, 4, 8, None)

    steps = {"stats": (4, 8), "ws": (4, 8)}
    for call in (fwd, bwd):
        names = call.__code__.co_varnames[:call.__code__.co_argcount]
        pointers = [n for n in names if n != "dtype"]
        refused(call, pointers, {"dtype": 9}, {n: steps.get(n, (1, 2)) for n in pointers})
