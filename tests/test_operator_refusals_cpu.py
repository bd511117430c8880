"""The C entries of the gated delta rule, the sampled verification and the
expert routing refuse bad arguments before they touch a device (CPU only)."""

from __future__ import annotations

import ctypes

import pytest

P = ctypes.c_void_p(256)
ODD = ctypes.c_void_p(260)


def _rule(lib, **kw):
    a = dict(q=P, ldq=256, k=P, ldk=256, v=P, ldv=512, g=P, gv=0, beta=P, mask=None, cu=None, s=P, so=P, y=P,
             zero=1, B=2, T=4, Hv=4, Hk=2, Dv=128, Dk=128)
    a.update(kw)
    chunked = {k: x for k, x in a.items() if k != "gv"}
    return [lib.dfl_gdn_rule_recurrent(*a.values(), None), lib.dfl_gdn_rule_chunked(*chunked.values(), None, 0, None)]


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), 2), (dict(T=-1), 2), (dict(Hv=3), 2), (dict(Hk=0), 2), (dict(Dv=48), 2), (dict(Dv=0), 2),
    (dict(Dk=96), 2), (dict(Dk=0), 2), (dict(ldq=255), 2), (dict(ldk=128), 2), (dict(ldv=511), 2),
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(g=None), 1), (dict(beta=None), 1),
    (dict(s=None), 1), (dict(so=None), 1), (dict(y=None), 1),
    (dict(s=ODD), 3), (dict(so=ODD), 3), (dict(y=ODD), 3), (dict(B=0), 0),
    (dict(Hv=1 << 24, Hk=1 << 24, Dk=256, Dv=256), 2),
])
def test_gated_delta_rule(pkg, kw, status):
    from dflash_mlx_b200 import _lib

    assert set(_rule(_lib.load(), **kw)) == {status}


@pytest.mark.parametrize("kw,status", [
    (dict(Dk=256, ldq=512, ldk=512), 2), (dict(Dk=32), 2), (dict(ldq=257), 3), (dict(ldk=260), 3), (dict(ldv=513), 3),
    (dict(q=ODD), 3), (dict(k=ODD), 3), (dict(v=ODD), 3),
])
def test_chunked_form_alone(pkg, kw, status):
    from dflash_mlx_b200 import _lib

    assert _rule(_lib.load(), **kw)[1] == status


def _sampled(lib, **kw):
    a = dict(lg=P, dl=P, dtype=0, ids=P, u=P, s=P, temp=P, lens=None, sup=None, acc=P, tok=P, prob=P, ld=100,
             bs=400, ldd=100, bsd=300, B=2, T=4, V=100, ws=P, n=1 << 20)
    a.update(kw)
    return lib.dfl_verify_accept_sampled(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(B=-1), 2), (dict(T=0), 2), (dict(T=257), 2), (dict(V=0), 2), (dict(V=(1 << 24) + 1), 2),
    (dict(B=40000), 2), (dict(ld=1 << 41), 2), (dict(bsd=1 << 41), 2),
    (dict(dtype=3), 6), (dict(dtype=-1), 6), (dict(B=0), 0),
    (dict(lg=None), 1), (dict(s=None), 1), (dict(temp=None), 1), (dict(acc=None), 1), (dict(tok=None), 1),
    (dict(ids=None), 1), (dict(u=None), 1), (dict(prob=None), 1),
    (dict(lg=ctypes.c_void_p(257)), 3), (dict(dtype=2, dl=ctypes.c_void_p(258)), 3),
])
def test_sampled_verification(pkg, kw, status):
    from dflash_mlx_b200 import _lib

    assert _sampled(_lib.load(), **kw) == status


def test_sampled_workspace_shapes(pkg):
    from dflash_mlx_b200 import _lib

    st = ctypes.c_int(-1)
    assert _lib.load().dfl_verify_sampled_workspace_bytes(2, 0, 10, 1, ctypes.byref(st)) == 0 and st.value == 2


def _route(lib, **kw):
    a = dict(lg=P, dtype=2, ld=64, bias=None, T=4, E=64, k=8, groups=8, kept=4, flags=7, scale=1.0, w=P, ids=P)
    a.update(kw)
    return lib.dfl_moe_route_experts(*a.values(), None)


@pytest.mark.parametrize("kw,status", [
    (dict(T=-1), 2), (dict(E=0), 2), (dict(E=4097, ld=5000), 2), (dict(k=0), 2), (dict(k=33), 2),
    (dict(groups=0), 2), (dict(groups=5), 2), (dict(kept=0), 2), (dict(kept=9), 2), (dict(kept=1, k=9), 2),
    (dict(ld=63), 2), (dict(dtype=3), 6), (dict(flags=8), 6), (dict(T=0), 0), (dict(lg=None), 1),
    (dict(w=None), 1), (dict(ids=None), 1), (dict(lg=ctypes.c_void_p(258)), 3),
])
def test_expert_routing(pkg, kw, status):
    from dflash_mlx_b200 import _lib

    assert _route(_lib.load(), **kw) == status


@pytest.mark.parametrize("t,k,e,status", [(0, 8, 64, 2), (17, 8, 64, 2), (4, 17, 64, 2), (4, 0, 64, 2),
                                          (4, 8, 0, 2), (4, 8, 4097, 2)])
def test_route_table(pkg, t, k, e, status):
    from dflash_mlx_b200 import _lib

    assert _lib.load().dfl_moe_route_table(P, t, k, e, P, None) == status
    assert _lib.load().dfl_moe_route_table(None, 4, 8, 64, P, None) == 1
