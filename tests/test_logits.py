"""oadp_amd.clip.logits without a GPU: what the operators refuse, in Python and at the C entries (nothing here launches)."""
import ctypes as C

import pytest
import torch

from oadp_amd import _lib
from oadp_amd.clip.logits import distill_top_logits, label_logits, token_logprobs
from oadp_amd.dp import TopLogitsDistillation

X = torch.zeros(3, 7)
IDS = torch.zeros(3, 2, dtype=torch.int64)
LP = torch.zeros(3, 2)


@pytest.mark.parametrize('error, call', [
    (RuntimeError, lambda: token_logprobs(X)),                                         # CPU tensors: no fallback
    (TypeError, lambda: token_logprobs(X.double())),
    (TypeError, lambda: token_logprobs(X.int())),
    (ValueError, lambda: token_logprobs(X[:, :0])),                                    # no vocabulary
    (ValueError, lambda: token_logprobs(torch.tensor(1.0))),
    (ValueError, lambda: token_logprobs(X, top=-1)),
    (ValueError, lambda: token_logprobs(X, top=129)),
    (ValueError, lambda: token_logprobs(X, scale=0.0)),
    (ValueError, lambda: token_logprobs(X, scale=-1.0)),
    (ValueError, lambda: token_logprobs(X, scale=float('inf'))),
    (ValueError, lambda: token_logprobs(X, scale=float('nan'))),
    (TypeError, lambda: token_logprobs(X, torch.zeros(3))),                            # targets of another type
    (TypeError, lambda: token_logprobs(X, torch.zeros(3, dtype=torch.int16))),
    (ValueError, lambda: token_logprobs(X, torch.zeros(4, dtype=torch.int64))),
    (ValueError, lambda: token_logprobs(X, torch.zeros(3, 2, 2, dtype=torch.int64))),
    (ValueError, lambda: token_logprobs(X, torch.zeros(3, 1025, dtype=torch.int64))),
    (TypeError, lambda: token_logprobs(X, mask=torch.ones(7))),
    (ValueError, lambda: token_logprobs(X, mask=torch.ones(6, dtype=torch.bool))),
    (ValueError, lambda: token_logprobs(X, mask=torch.ones(3, 1, dtype=torch.bool))),
    (ValueError, lambda: token_logprobs(X, mask=torch.ones(2, 7, dtype=torch.bool))),
    (ValueError, lambda: token_logprobs(X, mask=torch.ones(1, 3, 7, dtype=torch.bool))),
    (RuntimeError, lambda: distill_top_logits(X, IDS, LP)),
    (TypeError, lambda: distill_top_logits(X, IDS.float(), LP)),
    (TypeError, lambda: distill_top_logits(X, IDS, LP.double())),
    (TypeError, lambda: distill_top_logits(X.double(), IDS, LP)),
    (ValueError, lambda: distill_top_logits(X, IDS, LP[:, :1])),
    (ValueError, lambda: distill_top_logits(X, IDS[:2], LP[:2])),
    (ValueError, lambda: distill_top_logits(X, IDS[:, 0], LP[:, 0])),
    (ValueError, lambda: distill_top_logits(X, IDS, LP, scale=0)),
    (ValueError, lambda: distill_top_logits(X, IDS, LP.clone().requires_grad_())),     # the teacher is frozen
    (ValueError, lambda: distill_top_logits(X, torch.zeros(3, 1025, dtype=torch.int32), torch.zeros(3, 1025))),
    (ValueError, lambda: label_logits(torch.zeros(2, 8), torch.zeros(5, 9))),
    (ValueError, lambda: label_logits(torch.zeros(2, 8), torch.zeros(8))),
    (ValueError, lambda: TopLogitsDistillation(torch.zeros(8))),
    (ValueError, lambda: TopLogitsDistillation(torch.zeros(5, 8), temperature=0)),
    (ValueError, lambda: TopLogitsDistillation(torch.zeros(5, 8))(torch.zeros(2, 5))),
    (ValueError, lambda: TopLogitsDistillation(torch.zeros(5, 8))(torch.zeros(2, 4), torch.zeros(2, 8))),
    (RuntimeError, lambda: TopLogitsDistillation(torch.zeros(5, 8))(torch.zeros(2, 5), torch.zeros(2, 8))),
])
def test_python_refusals(error, call):
    with pytest.raises(error):
        call()


def test_c_refusals(lib):
    """Every refusal comes before the first HIP call: host addresses stand in for device memory and are never read."""
    buf = C.create_string_buffer(4096)
    p = C.addressof(buf) + (-C.addressof(buf)) % 64

    def score(x=p, dtype=_lib.OAKE_F32, rows=3, vocab=7, stride=7, scale=1.0, mask=None, mstride=0, ids=p,
              index=_lib.OAKE_I64, n=1, top=1, lp=p, lse=p, ent=p, top_lp=p, top_ids=p, stats=p):
        return lib.oake_token_logprobs(x, dtype, rows, vocab, stride, scale, mask, mstride, ids, index, n, top, lp, lse, ent,
                                       top_lp, top_ids, stats, None, 0, None)

    def score_grad(x=p, dtype=_lib.OAKE_F32, rows=3, vocab=7, scale=1.0, ids=p, index=_lib.OAKE_I64, n=1, tids=p, top=1,
                   stats=p, g=p, grad=p, gstride=7):
        return lib.oake_token_logprobs_backward(x, dtype, rows, vocab, 7, scale, None, 0, ids, index, n, tids, top, stats,
                                                g, g, g, g, grad, gstride, None)

    def distill(x=p, dtype=_lib.OAKE_F32, rows=3, vocab=7, scale=1.0, ids=p, index=_lib.OAKE_I64, v=p, top=1, loss=p, stats=p):
        return lib.oake_distill_top_logits(x, dtype, rows, vocab, 7, scale, ids, index, v, top, 0, loss, stats, None, 0, None)

    def distill_grad(x=p, dtype=_lib.OAKE_F32, rows=3, vocab=7, ids=p, index=_lib.OAKE_I64, v=p, top=1, stats=p, g=p, grad=p,
                     gstride=7):
        return lib.oake_distill_top_logits_backward(x, dtype, rows, vocab, 7, 1.0, ids, index, v, top, 0, stats, g, grad,
                                                    gstride, None)

    bad = [
        (score, [dict(x=None), dict(x=p + 2), dict(dtype=_lib.OAKE_U8), dict(dtype=9), dict(rows=-1), dict(rows=2 ** 31),
                 dict(vocab=0), dict(vocab=2 ** 31), dict(stride=-7), dict(scale=0.0), dict(scale=-1.0),
                 dict(scale=float('nan')), dict(scale=float('inf')), dict(mask=p, mstride=-1), dict(ids=None), dict(index=0),
                 dict(ids=p + 4), dict(n=-1), dict(n=1025), dict(top=-1), dict(top=129), dict(lp=None), dict(top_lp=None),
                 dict(top_ids=None)]),
        (score_grad, [dict(x=None), dict(dtype=_lib.OAKE_U8), dict(rows=-1), dict(vocab=0), dict(scale=0.0), dict(ids=None),
                      dict(index=1), dict(n=1025), dict(tids=None), dict(tids=p + 4), dict(top=129), dict(stats=None),
                      dict(grad=None), dict(grad=p + 1), dict(gstride=6)]),
        (distill, [dict(x=None), dict(dtype=_lib.OAKE_I64), dict(rows=-1), dict(vocab=0), dict(scale=-0.0), dict(ids=None),
                   dict(index=2), dict(v=None), dict(top=-1), dict(top=1025), dict(loss=None), dict(stats=None)]),
        (distill_grad, [dict(x=None), dict(dtype=_lib.OAKE_I32), dict(rows=-1), dict(vocab=0), dict(ids=None), dict(index=3),
                        dict(v=None), dict(top=1025), dict(stats=None), dict(g=None), dict(grad=None), dict(grad=p + 2),
                        dict(gstride=0)]),
    ]
    for call, cases in bad:
        for case in cases:
            assert call(**case) == _lib.OAKE_ERR_INVALID, (call.__name__, case)
            assert lib.oake_last_error(None).startswith(b'oake_'), (call.__name__, case)
        assert call(rows=0) == _lib.OAKE_OK  # nothing to do
    n = C.c_size_t(7)
    assert lib.oake_logits_workspace(4, 100, _lib.OAKE_F16, 5, C.byref(n)) == _lib.OAKE_OK
    for args in [(-1, 100, _lib.OAKE_F16, 5), (4, 0, _lib.OAKE_F16, 5), (4, 100, _lib.OAKE_U8, 5), (4, 100, _lib.OAKE_F16, 129)]:
        assert lib.oake_logits_workspace(*args, C.byref(n)) == _lib.OAKE_ERR_INVALID
    assert lib.oake_logits_workspace(4, 100, _lib.OAKE_F16, 5, None) == _lib.OAKE_ERR_INVALID


def test_label_logits_under_autocast():
    """The cosines stay fp32: rounded to 16 bits and times CLIP's scale they would be off by 0.2 and more."""
    e, labels = torch.randn(4, 16, generator=torch.Generator().manual_seed(0)), torch.eye(16)[:5] + 0.1
    want = label_logits(e, labels)
    with torch.autocast('cpu', dtype=torch.bfloat16):
        got = label_logits(e, labels)
        assert torch.is_autocast_enabled('cpu')
    assert got.dtype == torch.float32 and torch.equal(got, want)


@pytest.mark.parametrize('options', [dict(top=0), dict(top=-3), dict(top=129), dict(scale=0.0), dict(scale=float('nan')),
                                     dict(temperature=float('nan')), dict(temperature=float('inf')),
                                     dict(mask=torch.ones(4, dtype=torch.bool)), dict(mask=torch.ones(5))])
def test_distillation_refuses_before_the_first_batch(options):
    with pytest.raises((ValueError, TypeError)):
        TopLogitsDistillation(torch.zeros(5, 8), **options)
    with pytest.raises(ValueError):
        TopLogitsDistillation(torch.zeros(0, 8))
    assert TopLogitsDistillation(torch.zeros(5, 8), top=128).top == 5


def test_a_learnt_scale_is_refused():
    """A scale that wants a gradient would silently get none; without one, or without grad mode, it is a number."""
    learnt = torch.nn.Parameter(torch.tensor(2.0))
    for call in (lambda s: token_logprobs(X, scale=s), lambda s: distill_top_logits(X, IDS, LP, scale=s)):
        for scale in (learnt, learnt.exp()):
            with pytest.raises(ValueError, match='scale'):
                call(scale)
        with pytest.raises(RuntimeError, match='GPU'):  # past the checks of arguments
            call(learnt.detach())
        with torch.no_grad(), pytest.raises(RuntimeError, match='GPU'):
            call(learnt)


def test_a_forward_mode_tangent_is_refused():
    """Outputs without a tangent would say that nothing depends on the input."""
    from torch.autograd import forward_ad as fw
    with fw.dual_level():
        dual = fw.make_dual(X.clone(), torch.ones_like(X))
        lp = fw.make_dual(LP.clone(), torch.ones_like(LP))
        scale = fw.make_dual(torch.tensor(2.0), torch.tensor(1.0))
        for call in (lambda: token_logprobs(dual), lambda: token_logprobs(dual.clone().requires_grad_()),
                     lambda: token_logprobs(X, scale=scale), lambda: distill_top_logits(dual, IDS, LP),
                     lambda: distill_top_logits(X, IDS, lp), lambda: distill_top_logits(X, IDS, LP, scale=scale)):
            with pytest.raises(ValueError, match='tangent'):
                call()
        for call in (lambda: token_logprobs(X, IDS), lambda: distill_top_logits(X, IDS, LP)):  # no tangent: past the checks
            with pytest.raises(RuntimeError, match='GPU'):
                call()
    with pytest.raises(RuntimeError, match='GPU'):
        token_logprobs(X)


def test_refusals_say_why(lib):
    """The text of a refusal is the library's own and names what was wrong."""
    buf, n = C.create_string_buffer(4096), C.c_size_t(0)
    p = C.addressof(buf) + (-C.addressof(buf)) % 64

    def why(rc):
        with pytest.raises(_lib.OakeError) as e:
            _lib.check(lib, None, rc, 'a call')
        return str(e.value)

    assert 'top must be 0 .. 128' in why(lib.oake_logits_workspace(1, 1, _lib.OAKE_F32, 500, C.byref(n)))
    for scale in (0.0, 1e-60, 2e38):  # (1e-60 is 0 in fp32)
        assert 'scale must be positive and at most 1e38' in why(lib.oake_token_logprobs(
            p, _lib.OAKE_F32, 3, 7, 7, scale, None, 0, None, 0, 0, 0, None, p, p, None, None, None, None, 0, None))
        assert 'scale must be positive and at most 1e38' in why(lib.oake_distill_top_logits(
            p, _lib.OAKE_F32, 3, 7, 7, scale, p, _lib.OAKE_I64, p, 1, 0, p, p, None, 0, None))
    assert 'n_targets must be 0 .. 1024' in why(lib.oake_token_logprobs(
        p, _lib.OAKE_F32, 3, 7, 7, 1.0, None, 0, p, _lib.OAKE_I64, 1025, 0, p, p, p, None, None, None, None, 0, None))
