"""What the attention and token-loss entry points refuse, without a GPU:
every check runs on the host before any HIP call."""
import pytest

import nova_hip as nh

FAKE = 1 << 40  # never dereferenced
BF, HF, F32 = nh.DT_BF16, nh.DT_F16, nh.DT_F32
EINVAL, ESHAPE, ESTRIDE, EDTYPE, ERANGE = 1, 2, 3, 4, 5


def d(sizes, strides=None, ptr=FAKE):
    if strides is None:
        strides, n = [], 1
        for s in reversed(sizes):
            strides.insert(0, n)
            n *= s
    return nh.make_memref(ptr, sizes, strides)


def call(name, descs, *args):
    return getattr(nh.lib(), name)(*[nh.ref(x) for x in descs], *args)


# ---- attention -----------------------------------------------------------------------

def fwd(scale=0.125, causal=1, dt=BF, **kw):
    o = dict(q=d((10, 4, 64)), k=d((12, 2, 64)), v=d((12, 2, 64)), qo=d((3,)), ko=d((3,)),
             out=d((10, 4, 64)), lse=d((4, 10)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_attention", list(o.values()), scale, causal, dt)


def bwd(scale=0.125, causal=1, dt=BF, **kw):
    o = dict(go=d((10, 4, 64)), q=d((10, 4, 64)), k=d((12, 2, 64)), v=d((12, 2, 64)),
             out=d((10, 4, 64)), lse=d((4, 10)), qo=d((3,)), ko=d((3,)), dq=d((10, 4, 64)),
             dk=d((12, 2, 64)), dv=d((12, 2, 64)), scratch=d((10 ** 6,)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_attention_backward", list(o.values()), scale, causal, dt)


@pytest.mark.parametrize("f", [fwd, bwd])
@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(q=None)), (EINVAL, dict(v=None)), (EINVAL, dict(qo=None)), (EINVAL, dict(out=None)),
    (EINVAL, dict(q=d((10, 4, 64), ptr=0))), (EINVAL, dict(ko=d((3,), ptr=0))),
    (EINVAL, dict(lse=d((4, 10), ptr=0))),
    (EINVAL, dict(scale=0.0)), (EINVAL, dict(scale=-1.0)), (EINVAL, dict(scale=float("nan"))),
    (EINVAL, dict(scale=float("inf"))), (EINVAL, dict(causal=2)),
    (EDTYPE, dict(dt=F32)), (EDTYPE, dict(dt=7)),
    (ESHAPE, dict(k=d((12, 2, 32)))), (ESHAPE, dict(v=d((11, 2, 64)))), (ESHAPE, dict(v=d((12, 4, 64)))),
    (ESHAPE, dict(k=d((12, 3, 64)), v=d((12, 3, 64)))),    # 4 heads over 3
    (ESHAPE, dict(qo=d((4,)))), (ESHAPE, dict(qo=d((0,)), ko=d((0,)))),
    (ESHAPE, dict(out=d((10, 4, 32)))), (ESHAPE, dict(lse=d((10, 4)))),
    (ESHAPE, dict(q=d((-1, 4, 64)))),
    (ESTRIDE, dict(q=d((10, 4, 64), (512, 128, 2)))),      # no unit stride on D
    (ESTRIDE, dict(k=d((12, 2, 64), (32, 1024, 1)))),      # rows overlap
    (ESTRIDE, dict(k=d((12, 2, 64), (0, 64, 1)))),         # broadcast over tokens
    (ESTRIDE, dict(q=d((10, 4, 64), (260, 65, 1)))),       # rows not 16-byte aligned
    (ESTRIDE, dict(q=d((10, 4, 64), ptr=FAKE + 2))),
    (ESTRIDE, dict(lse=d((4, 10), (10, 2)))), (ESTRIDE, dict(lse=d((4, 10), (5, 1)))),
    (ESTRIDE, dict(qo=d((3,), (2,)))),
    (ERANGE, dict(k=d((12, 2, 64), ((1 << 23) + 8, 64, 1)))),
])
def test_attention_refuses(f, want, kw):
    assert f(**kw) == want, nh.lib().nova_hip_last_error()


@pytest.mark.parametrize("strides", [(256, 32, 1), (128, 64, 1), (256, 0, 1), (640, 32, 1)])
def test_attention_results_must_not_overlap(strides):
    x = d((10, 4, 64), strides)
    assert fwd(out=x) == ESTRIDE and bwd(dq=x) == ESTRIDE


@pytest.mark.parametrize("D,want", [(12, ERANGE), (136, ERANGE), (256, ERANGE), (1, ERANGE)])
def test_attention_head_dim(D, want):
    st = (4 * 256, 256, 1)  # aligned rows whatever D
    q = d((10, 4, D), st)
    k = d((12, 2, D), (512, 256, 1))
    assert fwd(q=q, k=k, v=k, out=q) == want


def test_attention_backward_refuses_its_own():
    assert bwd(lse=None) == EINVAL and bwd(scratch=None) == EINVAL and bwd(go=None) == EINVAL
    assert bwd(scratch=d((79,))) == ESHAPE and bwd(scratch=d((10 ** 6,), (2,))) == ESTRIDE
    assert bwd(dk=d((12, 4, 64))) == ESHAPE and bwd(dq=d((9, 4, 64))) == ESHAPE
    assert bwd(dv=d((12, 2, 64), (128, 8, 1))) == ESTRIDE
    L = nh.lib()
    # Without splits the rows' two constants; the splits' sums on top.
    assert L.nova_hip_attention_backward_scratch(10, 12, 2, 4, 2, 64, 1) == 80
    assert L.nova_hip_attention_backward_scratch(8192, 8192, 1, 8, 8, 64, 0) == 2 * 8 * 8192
    one = L.nova_hip_attention_backward_scratch(4096, 4096, 1, 4, 1, 128, 0)
    assert one > 2 * 4 * 4096 and (one - 2 * 4 * 4096) % (33 * 4 * 64 * 128) == 0
    assert L.nova_hip_attention_backward_scratch(-1, 4096, 1, 4, 1, 128, 0) == 0


def test_calls_beyond_a_grid_are_refused():
    # 2^20 one-token sequences of 32 heads: 2^25 tiles.
    n = 1 << 20
    q, off = d((n, 32, 64)), d((n + 1,))
    kw = dict(q=q, k=d((n, 2, 64)), v=d((n, 2, 64)), qo=off, ko=off, out=q, lse=d((32, n)))
    assert fwd(**kw) == ERANGE
    assert bwd(**kw, go=q, dq=q, dk=d((n, 2, 64)), dv=d((n, 2, 64)), scratch=d((1 << 40,))) == ERANGE
    assert logp(x=d((1 << 26, 4)), y=d((1 << 26,)), logp=d((1 << 26,))) == ERANGE
    assert logp(x=d((1 << 22, 5000)), y=d((1 << 22,)), logp=d((1 << 22,))) == ERANGE


def test_attention_empty_calls_do_nothing():
    none = dict(q=d((0, 4, 64), ptr=0), out=d((0, 4, 64), ptr=0), lse=d((4, 0), ptr=0))
    assert fwd(**none) == 0
    assert fwd(qo=d((1,)), ko=d((1,))) == 0  # no sequence


# ---- decode ----------------------------------------------------------------------------

def dec(scale=0.125, dt=BF, **kw):
    o = dict(q=d((3, 4, 64)), k=d((3, 2000, 2, 64)), v=d((3, 2000, 2, 64)), lens=d((3,)),
             out=d((3, 4, 64)), lse=None, scratch=d((10 ** 6,)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_attention_decode", list(o.values()), scale, dt)


@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(q=None)), (EINVAL, dict(lens=None)), (EINVAL, dict(scale=0.0)),
    (EINVAL, dict(k=d((3, 2000, 2, 64), ptr=0))), (EINVAL, dict(lens=d((3,), ptr=0))),
    (EINVAL, dict(scratch=None)), (EINVAL, dict(lse=d((3, 4), ptr=0))),
    (EDTYPE, dict(dt=F32)),
    (ESHAPE, dict(v=d((3, 1999, 2, 64)))), (ESHAPE, dict(lens=d((2,)))), (ESHAPE, dict(out=d((3, 2, 64)))),
    (ESHAPE, dict(k=d((2, 2000, 2, 64)), v=d((2, 2000, 2, 64)))),
    (ESHAPE, dict(k=d((3, 2000, 3, 64)), v=d((3, 2000, 3, 64)))), (ESHAPE, dict(lse=d((4, 3)))),
    (ESHAPE, dict(scratch=d((10,)))),
    (ESTRIDE, dict(k=d((3, 2000, 2, 64), (256000, 32, 64000, 1)))),
    (ESTRIDE, dict(k=d((3, 2000, 2, 64), (256000, 128, 64, 2)))),
    (ESTRIDE, dict(k=d((3, 2000, 2, 64), ptr=FAKE + 8))),
    (ESTRIDE, dict(v=d((3, 2000, 2, 64), (256004, 128, 64, 1)))),
    (ESTRIDE, dict(q=d((3, 4, 64), (256, 0, 1)))), (ESTRIDE, dict(out=d((3, 4, 64), (64, 64, 1)))),
    (ESTRIDE, dict(lens=d((3,), (2,)))), (ESTRIDE, dict(scratch=d((10 ** 6,), ptr=FAKE + 4))),
    (ESTRIDE, dict(lse=d((3, 4), (2, 1)))),
    (ERANGE, dict(k=d((3, 2000, 2, 64), (1 << 32, (1 << 23) + 64, 64, 1)))),
    (ERANGE, dict(q=d((3, 4, 136)), out=d((3, 4, 136)), k=d((3, 2000, 2, 136)), v=d((3, 2000, 2, 136)))),
])
def test_decode_refuses(want, kw):
    assert dec(**kw) == want, nh.lib().nova_hip_last_error()


def test_decode_scratch_and_empty_calls():
    L = nh.lib()
    assert L.nova_hip_attention_decode_scratch(3, 1024, 4, 2, 64) == 0  # one workgroup's work
    assert L.nova_hip_attention_decode_scratch(3, 1025, 4, 2, 64) == 3 * 4 * 17 * 66
    assert L.nova_hip_attention_decode_scratch(0, 2000, 4, 2, 64) == 0
    # At most 32768 splits whatever the cache.
    most = L.nova_hip_attention_decode_scratch(1, 2 ** 31 - 2 ** 20, 1, 1, 8)
    assert most <= 32768 * 10
    assert dec(q=d((0, 4, 64), ptr=0), out=d((0, 4, 64), ptr=0), lens=d((0,), ptr=0),
               k=d((0, 2000, 2, 64), ptr=0), v=d((0, 2000, 2, 64), ptr=0)) == 0


# ---- losses over token log-probabilities --------------------------------------------------

def logp(dt=F32, **kw):
    o = dict(x=d((6, 100)), y=d((6,)), logp=d((6,)), lse=None)
    o.update(kw)
    return call("_mlir_ciface_nova_hip_token_logp", list(o.values()), dt)


def policy(clip=(0.2, 0.2), kl=0.0, scale=1.0, dt=F32, **kw):
    o = dict(x=d((6, 100)), y=d((6,)), old=d((6,)), ref=None, adv=d((6,)), w=d((6,)), loss=d((1,)),
             logp=d((6,)), row=d((6,)), grad=d((6, 100)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_policy_loss", list(o.values()), clip[0], clip[1], kl, scale, dt)


def pref(beta=0.1, eps=0.0, scale=1.0, dt=F32, **kw):
    o = dict(x=d((6, 100)), y=d((6,)), off=d((5,)), ref=d((4,)), loss=d((1,)), seq=d((4,)),
             pair=d((2,)), token=d((3, 6)), grad=d((6, 100)))
    o.update(kw)
    return call("_mlir_ciface_nova_hip_preference_loss", list(o.values()), beta, eps, scale, dt)


@pytest.mark.parametrize("f", [logp, policy, pref])
@pytest.mark.parametrize("want,kw", [
    (EINVAL, dict(x=None)), (EINVAL, dict(y=None)), (EINVAL, dict(x=d((6, 100), ptr=0))),
    (EINVAL, dict(y=d((6,), ptr=0))), (EDTYPE, dict(dt=nh.DT_I32)),
    (ESHAPE, dict(y=d((5,)))), (ESHAPE, dict(x=d((6, 0)))),
    (ESTRIDE, dict(x=d((6, 100), (200, 2)))), (ESTRIDE, dict(x=d((6, 100), (99, 1)))),
    (ESTRIDE, dict(y=d((6,), (2,)))),
])
def test_losses_refuse(f, want, kw):
    assert f(**kw) == want, nh.lib().nova_hip_last_error()


@pytest.mark.parametrize("f,want,kw", [
    (logp, EINVAL, dict(logp=None)), (logp, ESHAPE, dict(logp=d((5,)))), (logp, ESHAPE, dict(lse=d((7,)))),
    (logp, ESTRIDE, dict(lse=d((6,), (2,)))),
    (policy, EINVAL, dict(old=None)), (policy, EINVAL, dict(row=None)), (policy, EINVAL, dict(loss=None)),
    (policy, ESHAPE, dict(adv=d((5,)))), (policy, ESHAPE, dict(loss=d((2,)))),
    (policy, ESHAPE, dict(grad=d((6, 99)))), (policy, ESTRIDE, dict(w=d((6,), (0,)))),
    (policy, ESTRIDE, dict(grad=d((6, 100), (50, 1)))),
    (policy, EINVAL, dict(kl=0.1)),                 # a KL term without ref_logp
    (policy, EINVAL, dict(clip=(-0.1, 0.2))), (policy, EINVAL, dict(clip=(1.5, 0.2))),
    (policy, EINVAL, dict(clip=(0.2, -1.0))), (policy, EINVAL, dict(clip=(0.2, float("inf")))),
    (policy, EINVAL, dict(kl=float("nan"))), (policy, EINVAL, dict(scale=float("inf"))),
    (pref, EINVAL, dict(off=None)), (pref, EINVAL, dict(token=None)), (pref, EINVAL, dict(ref=None)),
    (pref, ESHAPE, dict(off=d((1,)))), (pref, ESHAPE, dict(off=d((4,)))), (pref, ESHAPE, dict(off=d((0,)))),
    (pref, ESHAPE, dict(ref=d((3,)))), (pref, ESHAPE, dict(pair=d((1,)))), (pref, ESHAPE, dict(token=d((2, 6)))),
    (pref, ESTRIDE, dict(token=d((3, 6), (5, 1)))), (pref, ESTRIDE, dict(off=d((5,), (2,)))),
    (pref, EINVAL, dict(beta=0.0)), (pref, EINVAL, dict(beta=float("nan"))), (pref, EINVAL, dict(eps=1.5)),
    (pref, EINVAL, dict(scale=float("nan"))),
])
def test_losses_refuse_their_own(f, want, kw):
    assert f(**kw) == want, nh.lib().nova_hip_last_error()


@pytest.mark.parametrize("f", [policy, pref])
@pytest.mark.parametrize("kw", [
    dict(grad=d((6, 100))), dict(grad=d((6, 100), ptr=FAKE + 4 * 599)),
    dict(x=d((6, 100), ptr=FAKE + 4 * 599)),
    dict(grad=d((6, 100), (150, 1), ptr=FAKE + 400)),            # other row strides
    dict(x=d((6, 100), (200, 1)), grad=d((6, 100), (200, 1), ptr=FAKE + 4 * 99)),
    dict(x=d((6, 100), (200, 1)), grad=d((6, 100), (200, 1), ptr=FAKE + 4 * 101)),
    dict(x=d((6, 100), (200, 1), ptr=FAKE + 4 * 301), grad=d((6, 100), (200, 1))),
])
def test_gradients_on_the_logits_are_refused(f, kw):
    assert f(**kw) == EINVAL and b"overlaps" in nh.lib().nova_hip_last_error()


# ---- the Python wrappers' own checks ---------------------------------------------------------

def test_wrappers_refuse_before_the_call():
    import torch
    bf, f = torch.bfloat16, torch.float32
    q = torch.zeros(4, 2, 64, dtype=bf)
    off = torch.tensor([0, 4], dtype=torch.int32)

    def code(fn, *a, **k):
        with pytest.raises(nh.NovaHipError) as e:
            fn(*a, **k)
        return e.value.code

    assert code(nh.attention, q, q.float(), q, off, off) == EDTYPE
    assert code(nh.attention, q, q, q, off.long(), off) == EDTYPE
    assert code(nh.attention, q[0], q, q, off, off) == ESHAPE      # rank
    assert code(nh.attention, q, q, q, off[None], off) == ESHAPE
    assert code(nh.attention, q, q, q, off, off) == EINVAL         # not on a GPU
    assert code(nh.attention_backward, q, q, q, q, q, torch.zeros(2, 4, dtype=bf), off, off) == EDTYPE
    kv = torch.zeros(4, 8, 2, 64, dtype=bf)
    assert code(nh.attention_decode, q, kv[0], kv, off) == ESHAPE
    assert code(nh.attention_decode, q, kv, kv, off.float()) == EDTYPE
    x, y = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int32)
    v = torch.zeros(3)
    assert code(nh.token_logp, x, y.long()) == EDTYPE
    assert code(nh.token_logp, x[0], y) == ESHAPE
    assert code(nh.policy_loss, x, y, v.double(), v, v) == EDTYPE
    assert code(nh.policy_loss, x, y, v, v, v, grad=x.to(bf)) == EDTYPE
    assert code(nh.preference_loss, x, y, off, v.to(bf)) == EDTYPE
    assert code(nh.preference_loss, x, y, off, v) == EINVAL


# ---- results on operands ---------------------------------------------------------------------

def shifted(sizes, at, strides=None):
    """A view `at` elements of 2 bytes behind FAKE."""
    return d(sizes, strides, ptr=FAKE + 2 * at)


def refused(rc):
    return rc == EINVAL and b"overlaps" in nh.lib().nova_hip_last_error()


FAR = 1 << 24
Q, K = (10, 4, 64), (12, 2, 64)


def fwd_at(**kw):
    o = dict(q=shifted(Q, 0), k=shifted(K, FAR), v=shifted(K, 2 * FAR), out=shifted(Q, 3 * FAR),
             lse=shifted((4, 10), 4 * FAR))
    o.update(kw)
    return fwd(**o)


def bwd_at(**kw):
    o = dict(q=shifted(Q, 0), k=shifted(K, FAR), v=shifted(K, 2 * FAR), out=shifted(Q, 3 * FAR),
             lse=shifted((4, 10), 4 * FAR), go=shifted(Q, 5 * FAR), dq=shifted(Q, 6 * FAR),
             dk=shifted(K, 7 * FAR), dv=shifted(K, 8 * FAR), scratch=d((10 ** 6,), ptr=FAKE + 18 * FAR))
    o.update(kw)
    return bwd(**o)


def dec_at(**kw):
    o = dict(q=shifted((3, 4, 64), 0), k=shifted((3, 2000, 2, 64), FAR), v=shifted((3, 2000, 2, 64), 2 * FAR),
             out=shifted((3, 4, 64), 3 * FAR), lse=shifted((3, 4), 4 * FAR),
             scratch=d((10 ** 6,), ptr=FAKE + 10 * FAR))
    o.update(kw)
    return dec(**o)


@pytest.mark.parametrize("at", [0, 8, 2560 - 8, -(2560 - 8)])
def test_results_on_operands_are_refused(at):
    assert refused(fwd_at(out=shifted(Q, at)))
    assert refused(fwd_at(out=shifted(Q, FAR + min(at, 1536 - 8))))
    assert refused(fwd_at(lse=shifted((4, 10), max(-72, min(at, 2400)))))
    for i in (0, 3, 5):  # q, out, grad_out
        assert refused(bwd_at(dq=shifted(Q, i * FAR + at)))
    at = max(-(1536 - 8), min(at, 1536 - 8))
    for i in (1, 2):  # k, v
        assert refused(bwd_at(dk=shifted(K, i * FAR + at))) and refused(bwd_at(dv=shifted(K, i * FAR + at)))
    assert refused(bwd_at(dv=shifted(K, 7 * FAR + at))) and refused(bwd_at(dk=shifted(K, 6 * FAR)))
    assert refused(bwd_at(dq=shifted(Q, 4 * FAR)))
    for i in (0, 1, 2):
        assert refused(dec_at(out=shifted((3, 4, 64), i * FAR + max(at, 0) % 768 // 8 * 8)))
    assert refused(dec_at(lse=shifted((3, 4), 3 * FAR)))


@pytest.mark.parametrize("view,strides", [
    # Views of one buffer that share bytes: heads of one projection that
    # overlap by one, halves of rows by eight values, tokens by one.
    (256 - 64, (640, 64, 1)), (64 - 8, (640, 128, 1)), (9 * 256, (256, 64, 1)),
    (64, (128, 1280, 1)),  # every second token, but from the heads' side the same rows
])
def test_views_that_share_bytes_are_refused(view, strides):
    other = strides if strides != (128, 1280, 1) else (128, 1344, 1)
    assert refused(fwd_at(q=shifted(Q, 0, strides), out=shifted(Q, view, other)))
    assert refused(bwd_at(q=shifted(Q, 0, strides), dq=shifted(Q, view, other)))


@pytest.mark.parametrize("view,strides", [
    (256, (640, 64, 1)),       # heads beside each other in one projection's rows
    (-256, (640, 64, 1)), (640 - 256, (640, 64, 1)),
    (64, (512, 128, 1)),       # halves of each head's row
    (64, (128, 1280, 1)),      # tokens in turn, heads outermost
    (2560, (256, 64, 1)),      # one behind the other
    (640, (64, 1280, 1)),      # heads in turn
])
def test_views_beside_each_other_pass(view, strides):
    """(What comes behind the check, a launch without a GPU, fails otherwise.)"""
    assert not refused(fwd_at(q=shifted(Q, 0, strides), out=shifted(Q, view, strides)))
    assert not refused(bwd_at(q=shifted(Q, 0, strides), dq=shifted(Q, view, strides)))
    kv = strides[0] // 2 // 64 * 64 if strides == (640, 64, 1) else None
    if kv:  # dq, dk and dv as the three parts of a fused projection's gradient
        assert not refused(bwd_at(dq=shifted(Q, 6 * FAR, (512, 64, 1)), dk=shifted(K, 6 * FAR + 256, (512, 64, 1)),
                                  dv=shifted(K, 6 * FAR + 384, (512, 64, 1))))


def test_runs_of_queries_follow_tokens_and_sequences():
    """Scratch for runs where two runs of 16 tiles of 64 queries (three of 8 for few
    tiles, or heads of more than 64) fit the likely longest sequence, and by no
    other sign of a batch: between a little under and a little over the bound the
    answer changes once."""
    def runs(T, B, H, D, causal=1):
        return nh.lib().nova_hip_attention_backward_scratch(T, T, B, H, H, D, causal) > 2 * H * T
    # sqrt(T / 64 * T / B / 64) tiles in the likely longest.
    for H, D, B, tiles in ((6, 64, 8, 32), (6, 64, 9, 32), (12, 64, 4, 32), (1, 64, 4, 24), (3, 128, 8, 24),
                           (8, 128, 8, 32)):
        least = int(64 * tiles * B ** 0.5)
        assert [runs(T, B, H, D) for T in (least // 2, least - 1, least + 64, 2 * least)] == [0, 0, 1, 1], (H, D, B)
    # Equal and unequal sequences of the same number and tokens have the same bound.
    assert runs(8192, 8, 6, 64) and runs(8120, 8, 6, 64) and runs(9216, 9, 6, 64)
