"""What the entry points of the paged cache refuse, before anything is enqueued."""
import ctypes

import pytest

from spec_mcts_b200._lib import lib

NULL, SHAPE, ALIGN, WORKSPACE, UNSUPPORTED = -1, -2, -3, -4, -5
_buf = ctypes.create_string_buffer(4096)
A = (ctypes.addressof(_buf) + 255) // 256 * 256


def attn(tbl=A, idx=4, tstride=8, lens=A, q=A, qs=512, k=A, v=A, ks=A, vs=A, kind=1, o=A, P=128, B=2, L=128, H=4, Hkv=2, D=128, ps=16, w=0, s=0, ws=None, n=0):
    return lib.q40_attn_pages(tbl, idx, tstride, lens, q, qs, k, v, ks, vs, kind, o, P, B, L, H, Hkv, D, ps, w, s, ws, n, None)


def append(tbl=A, idx=4, tstride=8, width=8, pos=A, off=None, q=A, qs=512, qo=A, k=A, kst=256, v=A, vst=256, cos=A, sin=A, n_pos=64, kp=A, vp=A, ks=A, vs=A, kind=1, P=128, B=2, T=2,
           H=4, Hkv=2, D=128, ps=16):
    return lib.q40_page_append(tbl, idx, tstride, width, pos, off, q, qs, qo, k, kst, v, vst, cos, sin, n_pos, kp, vp, ks, vs, kind, P, B, T, H, Hkv, D, ps, None)


def window(q=A, ldq=512, k=A, ldk=256, v=A, ldv=256, o=A, ldo=512, S=4, H=4, Hkv=2, D=128, off=0, w=3, s=0, ws=None, n=0, err=A):
    return lib.q40_attn_causal_window(q, ldq, k, ldk, v, ldv, o, ldo, S, H, Hkv, D, off, w, s, ws, n, err, None)


@pytest.mark.parametrize("status,bad", [(NULL, dict(q=None)), (NULL, dict(tbl=None)), (NULL, dict(ks=None)), (NULL, dict(P=0)), (SHAPE, dict(H=5)), (SHAPE, dict(tstride=7)), (SHAPE, dict(P=100)),
                                        (SHAPE, dict(w=-1)), (SHAPE, dict(s=-1)), (SHAPE, dict(ps=0)), (SHAPE, dict(qs=511)), (SHAPE, dict(L=(1 << 30) + 1, tstride=1 << 40)),
                                        (ALIGN, dict(q=A + 8)), (ALIGN, dict(qs=516)), (ALIGN, dict(k=A + 8)), (ALIGN, dict(vs=A + 2)), (ALIGN, dict(lens=A + 2)), (ALIGN, dict(tbl=A + 2)),
                                        (UNSUPPORTED, dict(D=64)), (UNSUPPORTED, dict(idx=8)), (UNSUPPORTED, dict(kind=3)), (0, dict(B=0)),
                                        (WORKSPACE, dict(L=1 << 20, tstride=1 << 16)), (WORKSPACE, dict(L=1 << 20, tstride=1 << 16, ws=A, n=64)), (ALIGN, dict(L=1 << 20, tstride=1 << 16, ws=A + 4, n=1 << 30))])
def test_attention_refuses(status, bad):
    assert attn(**bad) == status


def test_attention_workspace():
    need = lambda *a: lib.q40_attn_pages_workspace_bytes(*a)
    assert need(1, 4, 4, 500, 0, 0) == 0 and need(0, 4, 4, 1 << 20, 0, 0) == 0 and need(2, 5, 4, 1 << 20, 0, 0) == 0
    one = need(4, 32, 8, 1 << 16, 0, 0)
    assert one > 0 and need(8, 32, 8, 1 << 16, 0, 0) > 0
    assert need(4, 32, 8, 1 << 16, 100, 4) == 0               # what a window leaves fits one chunk
    assert need(4, 32, 8, 1 << 16, 1 << 16, 0) == one and need(4, 32, 8, 1 << 16, 2 ** 31 - 1, 2 ** 31 - 1) == one


@pytest.mark.parametrize("status,bad", [(NULL, dict(k=None)), (NULL, dict(pos=None)), (NULL, dict(cos=None)), (NULL, dict(qo=None)), (NULL, dict(vs=None)), (NULL, dict(cos=None, sin=None)),
                                        (SHAPE, dict(T=3)), (SHAPE, dict(T=-1, off=A)), (SHAPE, dict(width=0)), (SHAPE, dict(width=9)), (SHAPE, dict(P=100)), (SHAPE, dict(kst=255)),
                                        (SHAPE, dict(n_pos=0)), (SHAPE, dict(H=0)), (SHAPE, dict(ps=0)), (SHAPE, dict(P=0)), (ALIGN, dict(kst=260)), (ALIGN, dict(k=A + 8)), (ALIGN, dict(kp=A + 8)),
                                        (ALIGN, dict(ks=A + 2)), (ALIGN, dict(off=A + 2)), (ALIGN, dict(sin=A + 8)), (UNSUPPORTED, dict(D=64)), (UNSUPPORTED, dict(kind=-1)), (UNSUPPORTED, dict(idx=1)),
                                        (0, dict(B=0, T=0)), (0, dict(T=0, off=A))])
def test_append_refuses(status, bad):
    assert append(**bad) == status


@pytest.mark.parametrize("status,bad", [(NULL, dict(o=None)), (UNSUPPORTED, dict(D=64)), (SHAPE, dict(H=5)), (SHAPE, dict(w=0)), (SHAPE, dict(s=-1)), (SHAPE, dict(off=-1)), (SHAPE, dict(off=1 << 30)),
                                        (SHAPE, dict(ldq=511)), (ALIGN, dict(ldk=260)), (ALIGN, dict(v=A + 8)), (ALIGN, dict(o=A + 2)), (0, dict(S=0)),
                                        (WORKSPACE, dict(S=100, off=4000, w=4000, ws=A, n=64)), (ALIGN, dict(S=100, off=4000, w=4000, ws=A + 4, n=1 << 30)), (ALIGN, dict(S=100, err=A + 2))])
def test_window_refuses(status, bad):
    assert window(**bad) == status


def test_window_workspace():
    need = lambda S, H, off, w, s=0: lib.q40_attn_causal_window_workspace_bytes(S, H, H, 128, off, w, s)
    row = 130 * 4
    assert need(1, 32, 0, 1) == need(100, 32, 0, 100) == need(0, 32, 5000, 5000) == need(100, 32, 5000, 0) == 0
    assert need(100, 32, 5000, 4096) == 4 * 100 * 32 * row                 # as many as leave each SM a CTA, for many tiles
    assert need(100, 32, 1000, 200) == 0                                   # few tiles
    assert need(100, 1, 1 << 20, 1 << 20) == 16 * 100 * row                # and 16 at most
    assert need(5000, 32, 5000, 4096) == need(512, 32, 0, 512) == 0
