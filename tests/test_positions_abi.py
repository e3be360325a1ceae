"""What the rotary, norm and paged-cache entry points refuse, without a GPU:
every check runs on the host before any HIP call."""
import pytest

import nova_hip as nh
from test_attention_abi import BF, EDTYPE, EINVAL, ERANGE, ESHAPE, ESTRIDE, F32, FAKE, HF, call, d

K, M = 1 << 20, 1 << 30
INF, NAN = float("inf"), float("nan")


def at(n, sizes, strides=None):
    """Operand n, far from the others."""
    return d(sizes, strides, ptr=FAKE + n * (1 << 36))


# ---- rotary -----------------------------------------------------------------------------

def rot(scale=1.0, inter=0, inv=0, dt=BF, **kw):
    o = dict(x=at(0, (10, 4, 64)), pos=at(1, (10,)), f=at(2, (32,)), out=at(3, (10, 4, 64)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_rotary", list(o.values()), scale, inter, inv, dt)


def norm(eps=1e-6, scale=1.0, inter=0, dt=BF, wdt=F32, **kw):
    o = dict(q=at(0, (10, 4, 64)), k=at(1, (10, 2, 64)), wq=at(2, (64,)), wk=at(3, (64,)), pos=at(4, (10,)),
             f=at(5, (32,)), qo=at(6, (10, 4, 64)), ko=at(7, (10, 2, 64)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_qk_norm_rotary", list(o.values()), eps, scale, inter, dt, wdt)


def back(eps=1e-6, scale=1.0, inter=0, dt=BF, wdt=F32, **kw):
    o = dict(gq=at(0, (10, 4, 64)), gk=at(1, (10, 2, 64)), q=at(2, (10, 4, 64)), k=at(3, (10, 2, 64)),
             wq=at(4, (64,)), wk=at(5, (64,)), pos=at(6, (10,)), f=at(7, (32,)), dq=at(8, (10, 4, 64)),
             dk=at(9, (10, 2, 64)), dwq=at(10, (64,)), dwk=at(11, (64,)), scratch=at(12, (K,)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_qk_norm_rotary_backward", list(o.values()), eps, scale, inter, dt, wdt)


@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(x=None)), (EINVAL, dict(pos=None)), (EINVAL, dict(f=None)), (EINVAL, dict(out=None)),
    (EINVAL, dict(scale=INF)), (EINVAL, dict(scale=NAN)), (EINVAL, dict(inter=2)), (EINVAL, dict(inv=-1)),
    (EINVAL, dict(x=d((10, 4, 64), ptr=0))), (EINVAL, dict(pos=d((10,), ptr=0))), (EINVAL, dict(f=d((32,), ptr=0))),
    (EDTYPE, dict(dt=3)), (EDTYPE, dict(dt=9)),
    (ESHAPE, dict(out=at(3, (10, 4, 32)))), (ESHAPE, dict(pos=at(1, (9,)))),
    (ERANGE, dict(f=at(2, (33,)))), (ERANGE, dict(f=at(2, (36,)))),    # beyond the head dim
    (ERANGE, dict(f=at(2, (6,)))),                                     # 12 values: no multiple of 8
    (ESTRIDE, dict(pos=at(1, (10,), (2,)))), (ESTRIDE, dict(f=at(2, (32,), (2,)))),
    (ESTRIDE, dict(x=at(0, (10, 4, 64), (512, 128, 2)))), (ESTRIDE, dict(x=at(0, (10, 4, 64), (260, 65, 1)))),
    (ESTRIDE, dict(x=d((10, 4, 64), ptr=FAKE + 2))), (ESTRIDE, dict(out=at(3, (10, 4, 64), (256, 32, 1)))),
    (ESTRIDE, dict(out=at(3, (10, 4, 64), (0, 64, 1)))),
    (EINVAL, dict(out=d((10, 4, 64), ptr=FAKE + 128))),                # over x, but not in its place
    (EINVAL, dict(out=d((10, 4, 64), (320, 64, 1)))),
    (EINVAL, dict(out=d((10, 4, 64), ptr=FAKE + (1 << 36) - 64))),     # over the positions
    (ERANGE, dict(x=at(0, (1 << 27, 1, 8)), out=at(3, (1 << 27, 1, 8)), pos=at(1, (1 << 27,)), f=at(2, (4,)))),
])
def test_rotary_refuses(want, kw):
    assert rot(**kw) == want, nh.lib().nova_hip_last_error()


@pytest.mark.parametrize("D", [4, 12, 264, 512])
def test_head_dims(D):
    st = (4 * 1024, 1024, 1)
    x, y = at(0, (10, 4, D), st), at(3, (10, 4, D), st)
    assert rot(x=x, out=y, f=at(2, (4,))) in (ERANGE,)
    assert norm(q=x, qo=y, k=at(1, (10, 4, D), st), ko=at(7, (10, 4, D), st), wq=at(2, (D,)), wk=at(3, (D,)),
                f=at(5, (4,))) == ERANGE


@pytest.mark.parametrize("f", [norm, back])
@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(q=None)), (EINVAL, dict(k=None)), (EINVAL, dict(wq=None)), (EINVAL, dict(pos=None)),
    (EINVAL, dict(f=None)), (EINVAL, dict(eps=-1.0)), (EINVAL, dict(eps=NAN)), (EINVAL, dict(eps=INF)),
    (EINVAL, dict(scale=-INF)), (EINVAL, dict(inter=3)), (EINVAL, dict(wk=d((64,), ptr=0))),
    (EDTYPE, dict(dt=7)), (EDTYPE, dict(wdt=HF)), (EDTYPE, dict(wdt=9)), (EDTYPE, dict(dt=F32, wdt=BF)),
    (ESHAPE, dict(wq=at(20, (32,)))), (ESHAPE, dict(wk=at(20, (65,)))), (ESHAPE, dict(pos=at(20, (11,)))),
    (ERANGE, dict(f=at(20, (40,)))), (ESTRIDE, dict(wq=at(20, (64,), (2,)))),
])
def test_norm_refuses(f, want, kw):
    assert f(**kw) == want, nh.lib().nova_hip_last_error()


def test_norm_shapes_and_overlaps():
    assert norm(k=at(1, (9, 2, 64)), ko=at(7, (9, 2, 64))) == ESHAPE
    assert norm(k=at(1, (10, 2, 32)), ko=at(7, (10, 2, 32))) == ESHAPE
    assert norm(qo=at(6, (10, 2, 64))) == ESHAPE and norm(ko=None) == EINVAL
    assert norm(qo=at(1, (10, 4, 64))) == EINVAL                       # over k
    assert norm(ko=at(6, (10, 2, 64))) == EINVAL                       # over q_out
    assert norm(qo=at(2, (10, 4, 64))) == EINVAL                       # over a weight
    assert norm(qo=at(0, (10, 4, 64), (256, 64, 1)), q=at(0, (10, 4, 64), (320, 64, 1))) == EINVAL
    assert back(dq=at(1, (10, 4, 64))) == EINVAL                       # over grad_k
    assert back(dk=at(2, (10, 2, 64))) == EINVAL                       # over q
    assert back(dk=at(8, (10, 2, 64))) == EINVAL                       # over dq
    assert back(dwq=at(11, (64,))) == EINVAL and back(dwq=at(8, (64,))) == EINVAL
    assert back(scratch=at(10, (K,))) == EINVAL and back(dwk=at(5, (64,))) == EINVAL


def test_backward_refuses_its_own():
    L = nh.lib()
    need = L.nova_hip_qk_norm_rotary_backward_scratch(10, 4, 2, 64)
    assert need == 2 * 10 * 64
    assert back(scratch=None) == EINVAL and back(scratch=at(12, (need - 1,))) == ESHAPE
    assert back(scratch=at(12, (K,), (2,))) == ESTRIDE
    assert back(gq=at(0, (10, 3, 64))) == ESHAPE and back(dk=at(9, (10, 2, 32))) == ESHAPE
    assert back(dwq=at(10, (32,))) == ESHAPE and back(dwk=None) == EINVAL
    # At most 1280 workgroups' sums of each operand, whatever the tokens.
    assert L.nova_hip_qk_norm_rotary_backward_scratch(1 << 20, 32, 8, 128) <= 2 * 1280 * 128
    assert L.nova_hip_qk_norm_rotary_backward_scratch(0, 4, 2, 64) == 0
    assert L.nova_hip_qk_norm_rotary_backward_scratch(-1, 4, 2, 64) == 0


def test_frequencies_refuse():
    def freq(f=at(0, (32,)), base=10000.0, factor=1.0, low=1.0, high=32.0, original=0):
        return call("_mlir_ciface_nova_hip_rotary_frequencies", [f], base, factor, low, high, original)
    assert freq(f=None) == EINVAL and freq(f=d((32,), ptr=0)) == EINVAL
    assert freq(f=at(0, (129,))) == ERANGE and freq(f=at(0, (32,), (2,))) == ESTRIDE
    for kw in (dict(base=0.0), dict(base=-1.0), dict(base=INF), dict(factor=0.0), dict(factor=NAN),
               dict(original=-1), dict(original=8, low=4.0, high=4.0), dict(original=8, high=INF)):
        assert freq(**kw) == EINVAL, kw
    assert freq(f=at(0, (0,))) == 0


# ---- pages ---------------------------------------------------------------------------------

PAGES = (50, 16, 2, 64)


def app(scale=1.0, inter=0, dt=BF, **kw):
    o = dict(k=at(0, (10, 2, 64)), v=at(1, (10, 2, 64)), kp=at(2, PAGES), vp=at(3, PAGES), off=at(4, (4,)),
             lens=at(5, (3,)), table=at(6, (3, 8)), f=at(7, (32,)), q=at(8, (10, 4, 64)), qo=at(9, (10, 4, 64)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_paged_append", list(o.values()), scale, inter, dt)


def att(scale=0.125, causal=1, most=0, dt=BF, **kw):
    o = dict(q=at(8, (10, 4, 64)), kp=at(2, PAGES), vp=at(3, PAGES), off=at(4, (4,)), lens=at(5, (3,)),
             table=at(6, (3, 8)), out=at(9, (10, 4, 64)), lse=at(10, (4, 10)), scratch=at(11, (M,)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_paged_attention", list(o.values()), scale, causal, most, dt)


@pytest.mark.parametrize("f", [app, att])
@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(kp=None)), (EINVAL, dict(vp=None)), (EINVAL, dict(off=None)), (EINVAL, dict(lens=None)),
    (EINVAL, dict(table=None)), (EINVAL, dict(scale=INF)), (EINVAL, dict(scale=NAN)),
    (EINVAL, dict(kp=d(PAGES, ptr=0))), (EINVAL, dict(off=d((4,), ptr=0))), (EINVAL, dict(lens=d((3,), ptr=0))),
    (EINVAL, dict(table=d((3, 8), ptr=0))), (EDTYPE, dict(dt=F32)), (EDTYPE, dict(dt=5)),
    (ESHAPE, dict(vp=at(3, (49, 16, 2, 64)))), (ESHAPE, dict(lens=at(5, (4,)))), (ESHAPE, dict(off=at(4, (0,)))),
    (ESHAPE, dict(table=at(6, (2, 8)))), (ESHAPE, dict(kp=at(2, (50, 16, 2, 32)), vp=at(3, (50, 16, 2, 32)))),
    (ESHAPE, dict(kp=at(2, (-1, 16, 2, 64)), vp=at(3, (-1, 16, 2, 64)))),
    (ESHAPE, dict(kp=at(2, (50, 16, 3, 64)), vp=at(3, (50, 16, 3, 64)))),
    (ESTRIDE, dict(kp=at(2, PAGES, (4096, 256, 128, 2)))), (ESTRIDE, dict(kp=d(PAGES, ptr=FAKE + 8))),
    (ESTRIDE, dict(vp=at(3, PAGES, (2052, 128, 64, 1)))), (ESTRIDE, dict(kp=at(2, PAGES, (-2048, 128, 64, 1)))),
    (ESTRIDE, dict(off=at(4, (4,), (2,)))), (ESTRIDE, dict(lens=at(5, (3,), (0,)))),
    (ESTRIDE, dict(table=at(6, (3, 8), (8, 2)))), (ESTRIDE, dict(table=at(6, (3, 8), (-8, 1)))),
    (ERANGE, dict(kp=at(2, (1 << 32, 16, 2, 64)), vp=at(3, (1 << 32, 16, 2, 64)))),
    (ERANGE, dict(table=at(6, (3, 1 << 28)))),
    (EINVAL, dict(q=None)),                                            # append: without q_out
])
def test_pages_refuse(f, want, kw):
    assert f(**kw) == want, nh.lib().nova_hip_last_error()


def test_append_refuses_its_own():
    assert app(k=None) == EINVAL and app(v=at(1, (10, 3, 64))) == ESHAPE and app(qo=None) == EINVAL
    assert app(q=at(8, (9, 4, 64)), qo=at(9, (9, 4, 64))) == ESHAPE
    assert app(inter=2) == EINVAL and app(f=at(7, (33,))) == ERANGE
    for st in ((2048, 128, 32, 1), (1024, 128, 64, 1), (0, 128, 64, 1), (2048, 0, 64, 1), (64, 64, 3200, 1)):
        assert app(kp=at(2, PAGES, st)) == ESTRIDE, st                  # rows of the pages overlap
    assert app(vp=at(2, PAGES)) == EINVAL                              # keys and values in one place
    both = (4096, 128, 64, 1)
    assert app(kp=at(2, PAGES, both), vp=d(PAGES, both, ptr=FAKE + 2 * (1 << 36) + 2048)) == EINVAL
    assert app(k=at(2, (10, 2, 64))) == EINVAL and app(q=at(3, (10, 4, 64))) == EINVAL
    assert app(qo=at(2, (10, 4, 64))) == EINVAL and app(qo=at(0, (10, 4, 64))) == EINVAL
    assert app(table=at(2, (3, 8))) == EINVAL and app(lens=at(3, (3,))) == EINVAL
    assert app(qo=d((10, 4, 64), ptr=FAKE + 8 * (1 << 36) + 128)) == EINVAL


def test_paged_attention_refuses_its_own():
    assert att(out=None) == EINVAL and att(out=at(9, (10, 3, 64))) == ESHAPE and att(lse=at(10, (10, 4))) == ESHAPE
    assert att(scale=0.0) == EINVAL and att(causal=2) == EINVAL and att(most=-1) == EINVAL
    assert att(q=at(8, (10, 3, 64)), out=at(9, (10, 3, 64)), lse=None) == ESHAPE     # 3 heads over 2
    big = (50, 16, 2, 136)
    assert att(q=at(8, (10, 4, 136)), out=at(9, (10, 4, 136)), kp=at(2, big), vp=at(3, big)) == ERANGE
    assert att(kp=at(2, PAGES, (1 << 29, (1 << 23) + 64, 64, 1))) == ERANGE
    assert att(out=at(8, (10, 4, 64))) == EINVAL and att(out=at(2, (10, 4, 64))) == EINVAL
    assert att(lse=at(9, (4, 10))) == EINVAL and att(lse=d((4, 10), (10, 2), ptr=FAKE)) == ESTRIDE
    wide = dict(table=at(6, (3, 800)))
    need = nh.lib().nova_hip_paged_attention_scratch(10, 3, 4, 2, 64, 12800, 10)
    assert need > 0
    assert att(scratch=None, **wide) == EINVAL and att(scratch=at(11, (need - 1,)), **wide) == ESHAPE
    assert att(scratch=d((M,), ptr=FAKE + 4), **wide) == ESTRIDE and att(scratch=at(11, (M,), (2,)), **wide) == ESTRIDE
    assert att(scratch=at(9, (M,)), **wide) == EINVAL
    n = 1 << 22  # 2^22 tokens of 512 heads
    q = dict(q=at(8, (n, 512, 8)), out=at(9, (n, 512, 8)), kp=at(2, (5, 16, 2, 8)), vp=at(3, (5, 16, 2, 8)), lse=None)
    assert att(**q) == ERANGE


def test_paged_scratch():
    f = nh.lib().nova_hip_paged_attention_scratch
    assert f(3, 3, 4, 2, 64, 64, 1) == 0                               # one split
    assert f(0, 3, 4, 2, 64, 64, 1) == 0 and f(3, 3, 5, 2, 64, 64, 1) == 0 and f(3, 3, 4, 2, 64, -1, 1) == 0
    assert (f(3, 3, 4, 2, 64, 12800, 1) - 2 * 3 * 4) % 66 == 0        # sums, and two numbers to a row
    # Single tokens: room for what fills the chip, or splits that are a grid's dimension.
    assert f(1, 1, 1, 1, 8, 2 ** 30, 1) <= 1536 * 32 * 10 + 4
    assert f(100, 100, 1, 1, 8, 2 ** 30, 1) <= 100 * 32768 * 10 + 200
    # Chunks: room for what fills the chip twice, whatever the tokens and rows.
    assert 0 < f(1 << 16, 4, 32, 8, 128, 131072, 1 << 16) <= 2 * 512 * 128 * 130
    assert f(1 << 16, 4, 32, 8, 128, 256, 1 << 16) == 0                # one split
    assert f(1 << 16, 100, 32, 8, 128, 131072, 1 << 16) == 0           # many tiles of many sequences
    assert att(table=at(6, (3, (1 << 26) + 1)), scratch=at(11, (1 << 33,))) == ERANGE


def test_empty_calls_do_nothing():
    none = dict(x=d((0, 4, 64), ptr=0), pos=d((0,), ptr=0), out=d((0, 4, 64), ptr=0))
    assert rot(**none) == 0
    e, e2 = d((0, 4, 64), ptr=0), d((0, 2, 64), ptr=0)
    assert norm(q=e, k=e2, qo=e, ko=e2, pos=d((0,), ptr=0)) == 0
    assert app(k=e2, v=e2, q=e, qo=e) == 0
    assert att(q=e, out=e, lse=None) == 0
    assert att(off=at(4, (1,)), lens=d((0,), ptr=0), table=d((0, 8), ptr=0)) == 0    # no sequence


@pytest.mark.parametrize("st", [(1 << 35, 64, 1), (256, 1 << 35, 1)])
def test_rows_too_far_apart(st):
    """Strides of 2^36 bytes."""
    assert rot(x=at(20, (2, 4, 64), st), out=at(3, (2, 4, 64)), pos=at(1, (2,))) == ERANGE
    two = dict(q=at(20, (2, 4, 64), st), k=at(40, (2, 4, 64)), pos=at(60, (2,)))
    assert norm(qo=at(6, (2, 4, 64)), ko=at(7, (2, 4, 64)), **two) == ERANGE
    assert back(gq=at(0, (2, 4, 64)), gk=at(1, (2, 4, 64)), dq=at(8, (2, 4, 64)), dk=at(9, (2, 4, 64)),
                **two) == ERANGE
