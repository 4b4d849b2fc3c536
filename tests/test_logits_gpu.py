"""oadp_amd.clip.logits on the GPU against the definitions in 64 bits: log probabilities, entropy and top alternatives,
distillation from top logits, the gradients of both.

Tolerances (E = 2^-24, half an fp32 step), for z = scale * x, d = z - max z <= 0, p = softmax(z):
  e^d         x - max x, times scale * log2(e), exp2: 3 roundings scale with |d|, exp2 is off by at most 2E   (3|d| + 2) E
  S           sum of them over threads of V / 64 values at most, then a tree                       (V / 64 + 24) E more
  log S       so  tol_S = (3 sum p|d| + V / 64 + 32) E    (log itself: 2 steps of log S, which is at most 18)
  log p       tol_S + 4 |d| E + |log p| E
  entropy     log S - sum p d: each term of the second sum as e^d times |d|        tol_S (1 + sum p|d|) + 4 sum p d^2 E
  gradient    scale * (p * (a0 - g_H (log p + H)) + w): p is off by (3|d| + 3 log S + 4) E + tol_S, the bracket by a few
              E of its parts and g_H times what log p and H are off; half a step of the type for the rounding at the end
Each is doubled for what this leaves out (second orders, the rounding of scale * log2(e))."""
import threading

import pytest
import torch

from oadp_amd import _lib, clip
from oadp_amd.clip.logits import distill_top_logits, label_logits, token_logprobs
from oadp_amd.dp import TopLogitsDistillation
from oadp_amd.weights import synthetic_images, synthetic_state_dict

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
INF = float('inf')
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def half_step(t, dtype):
    """What rounding t to dtype may move it."""
    info = torch.finfo(dtype)
    return t.abs() * (info.eps / 2) + info.tiny * info.eps


def close(got, want, tol, what=''):
    got, want, tol = got.detach().double().cpu(), want.double().cpu(), tol.double().cpu().expand(want.shape)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = (got - want).abs()[fine] / tol[fine].clamp_min(1e-300)
    assert off.numel() == 0 or off.max() <= 1, (what, off.max().item(), (got - want).abs()[fine].max().item())


class Score:
    """Everything token_logprobs returns, and its gradient, in 64 bits."""

    def __init__(self, x, targets=None, top=0, mask=None, scale=1.0):
        self.x, self.scale, self.targets, self.top = x, scale, targets, top
        raw = x.detach().float()
        if mask is not None:
            raw = raw.masked_fill(~mask, -INF)
        z = raw.double() * scale
        self.n, self.vocab = z.shape
        nan = (torch.isnan(z) | (z == INF)).any(1, keepdim=True)
        self.empty = (z == -INF).all(1, keepdim=True)
        self.dead = self.empty | nan
        peak = z.amax(1, keepdim=True).masked_fill(self.dead, 0)
        self.d = (z - peak).masked_fill(self.dead, -INF)
        e = self.d.exp()
        total = e.sum(1, keepdim=True).masked_fill(self.dead, 1)
        self.log_s = total.log()
        self.p = e / total
        # no log probability in a NaN row, none but -inf in an empty one
        self.logp = (self.d - self.log_s).masked_fill(nan, float('nan'))
        self.lse = (peak + self.log_s).masked_fill(self.empty, -INF).masked_fill(nan, float('nan'))[:, 0]
        self.ad = self.d.masked_fill(self.d == -INF, 0).abs()
        self.mean_d = (self.p * self.ad).sum(1, keepdim=True)
        h = self.log_s + self.mean_d
        self.h = h.masked_fill(self.empty, 0).masked_fill(nan, float('nan'))[:, 0]
        self.tol_s = 2 * E * (3 * self.mean_d + self.vocab / 64 + 32)
        self.tol_logp = self.tol_s + 2 * E * (4 * self.ad + self.logp.masked_fill(~torch.isfinite(self.logp), 0).abs())
        self.tol_h = self.tol_s * (1 + self.mean_d) + 8 * E * (self.p * self.ad ** 2).sum(1, keepdim=True)
        self.tol_lse = self.tol_s[:, 0] + 2 * E * self.lse.abs().masked_fill(self.dead[:, 0], 0) + 2 * E * peak[:, 0].abs()
        self.raw = raw
        if top:
            k = min(top, self.vocab)
            order = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :k]
            value = raw.gather(1, order)
            self.top_indices = order.masked_fill(value == -INF, -1)
            self.top_logprobs = self.logp.gather(1, order).masked_fill(value == -INF, -INF)
            self.tol_top = self.tol_logp.gather(1, order)
            pad = (0, top - k)
            self.top_indices = torch.nn.functional.pad(self.top_indices, pad, value=-1)
            self.top_logprobs = torch.nn.functional.pad(self.top_logprobs, pad, value=-INF)
            self.tol_top = torch.nn.functional.pad(self.tol_top, pad)
        if targets is not None:
            t = targets.long()
            inside = t.clamp(0, self.vocab - 1)
            self.logprobs = self.logp.gather(1, inside).masked_fill(t < 0, 0).masked_fill(t >= self.vocab, float('nan'))
            self.tol_given = self.tol_logp.gather(1, inside)

    def check(self, got):
        close(got.lse, self.lse, self.tol_lse, 'lse')
        close(got.entropy, self.h, self.tol_h[:, 0], 'entropy')
        if self.targets is not None:
            close(got.logprobs, self.logprobs, self.tol_given, 'logprobs')
        if self.top:
            assert got.top_indices.dtype == torch.int64
            assert torch.equal(got.top_indices, self.top_indices), 'top_indices'
            close(got.top_logprobs, self.top_logprobs, self.tol_top, 'top_logprobs')

    def grad(self, g_logprobs=None, g_lse=None, g_entropy=None, g_top=None):
        """(gradient, how far off it may be)."""
        w, a0 = torch.zeros_like(self.p), torch.zeros_like(self.log_s)
        parts = torch.zeros_like(a0)
        for g, ids, value in ((g_logprobs, self.targets, getattr(self, 'logprobs', None)),
                              (g_top, getattr(self, 'top_indices', None), getattr(self, 'top_logprobs', None))):
            if g is not None:
                g = g.double().masked_fill((ids < 0) | (value == -INF), 0)
                w.scatter_add_(1, ids.long().clamp(0, self.vocab - 1), g)
                a0, parts = a0 - g.sum(1, keepdim=True), parts + g.abs().sum(1, keepdim=True)
        if g_lse is not None:
            a0, parts = a0 + g_lse.double()[:, None], parts + g_lse.double().abs()[:, None]
        gh = torch.zeros_like(a0) if g_entropy is None else g_entropy.double()[:, None]
        logp = self.logp.masked_fill(self.d == -INF, 0)
        bracket = a0 - gh * (logp + self.h[:, None])
        grad = (self.scale * (self.p * bracket + w)).masked_fill(self.empty, 0)
        off_p = 2 * E * (3 * self.ad + 3 * self.log_s + 4) + self.tol_s
        size = parts + gh.abs() * (logp.abs() + self.h[:, None].abs())
        tol = self.p * (size * (off_p + 16 * E) + gh.abs() * (self.tol_logp + self.tol_h)) + 8 * E * (w.abs() + self.p * parts)
        tol = self.scale * tol
        return grad, tol + half_step(grad.abs() + tol, self.x.dtype)


def logits_of(rows, vocab, dtype, seed=0, spread=3.0, dev='cuda'):
    g = torch.Generator(device='cuda').manual_seed(seed * 1000003 + rows * 7919 + vocab)
    return (torch.randn(rows, vocab, generator=g, device='cuda') * spread).to(dtype)


def some_targets(rows, vocab, n, seed=0, dtype=torch.int64):
    g = torch.Generator(device='cuda').manual_seed(seed + 17 * rows + vocab)
    t = torch.randint(vocab, (rows, n), generator=g, device='cuda').to(dtype)
    t.view(-1)[::7] = -1 - (seed % 3) * 50
    return t


# lengths around a wave's, a vector's and a thread block's edges; the text tower's vocabulary; beyond one block's share
VOCABS = [1, 2, 7, 8, 9, 63, 64, 65, 257, 511, 1203, 2048, 2049, 4099, 8192, 8193, 16384, 16385, 32769, 49408, 65536,
          65543, 131073, 300007]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', VOCABS)
def test_scores_over_lengths(cuda, vocab, dtype):
    rows = 5 if vocab < 20000 else 3
    for top, n, index in ((0, 1, torch.int64), (5, 3, torch.int32), (64, 0, torch.int64), (128, 2, torch.int64)):
        x = logits_of(rows, vocab, dtype, seed=top)
        t = some_targets(rows, vocab, n, top, index) if n else None
        Score(x, t, top).check(token_logprobs(x, t, top=top))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, top', [(1, 65, 5), (1, 1203, 20), (1, 49408, 5), (1, 151936, 128), (2, 49408, 64),
                                              (17, 20001, 10), (300, 65, 8), (700, 1203, 33), (1300, 4097, 7), (600, 9999, 1), (2500, 2049, 20),
                                              (2500, 4096, 32), (2050, 3001, 128), (400, 1999, 128), (400, 1203, 100)])
def test_scores_over_rows(cuda, rows, vocab, top, dtype):
    x = logits_of(rows, vocab, dtype, seed=3)
    t = some_targets(rows, vocab, 1)
    Score(x, t, top, scale=0.7).check(token_logprobs(x, t, top=top, scale=0.7))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [1, 7, 65, 1203, 5000, 49409, 140001])
@pytest.mark.parametrize('shared', [True, False])
def test_masks(cuda, vocab, dtype, shared):
    """Masked places hold NaN, infinities and the largest values; one row has nothing allowed, one a single place."""
    rows = 6
    x = logits_of(rows, vocab, dtype, seed=5)
    g = torch.Generator(device='cuda').manual_seed(vocab)
    mask = torch.rand(vocab if shared else (rows, vocab), generator=g, device='cuda') < 0.5
    if not shared:
        mask[1] = False
        mask[2] = False
        mask[2, vocab // 2] = True
        mask[3] = True
    full = mask.expand(rows, vocab)
    junk = torch.tensor([float('nan'), INF, -INF, torch.finfo(dtype).max, torch.finfo(dtype).min], device='cuda').to(dtype)
    which = torch.randint(5, (rows, vocab), generator=g, device='cuda')
    x = torch.where(full, x, junk[which])
    t = some_targets(rows, vocab, 2)
    for top in (0, 4, 100):
        Score(x, t, top, mask=full).check(token_logprobs(x, t, top=top, mask=mask))
    x.requires_grad_()
    out = token_logprobs(x, t, top=4, mask=mask)
    up = [torch.randn(o.shape, generator=g, device='cuda') for o in (out.logprobs, out.entropy, out.top_logprobs)]
    grad, = torch.autograd.grad([out.logprobs, out.entropy, out.top_logprobs], [x], up)
    want, tol = Score(x, t, 4, mask=full).grad(g_logprobs=up[0], g_entropy=up[1], g_top=up[2])
    close(grad, want, tol)
    assert (grad[~full] == 0).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [5, 700, 9000, 200001])
def test_special_rows(cuda, vocab, dtype):
    lowest = torch.finfo(dtype).min
    x = logits_of(12, vocab, dtype, seed=9)
    x[0] = -INF                               # nothing
    x[1] = lowest                             # a mask of the type's lowest value that leaves nothing: uniform
    x[2, 1:] = lowest                         # ... that leaves one
    x[3] = 0                                  # all equal: the lowest indices
    x[4, vocab // 2] = float('nan')
    x[5, vocab - 1] = INF
    x[6] = torch.arange(vocab, device='cuda').to(dtype) / 8           # ascending: the best are last
    x[7] = -x[6]
    x[8] = (torch.arange(vocab, device='cuda') % 2).to(dtype) * -0.0  # +0 and -0 are equal
    x[9] = -INF
    x[9, vocab - 2] = 1.5                     # one place
    x[10] = float('nan')
    x[11, 0] = 60                             # one place has nearly all
    t = torch.tensor([0, vocab - 1, vocab, 2 ** 40], device='cuda').expand(12, 4)
    for top in (0, 3, 128):
        Score(x, t, top).check(token_logprobs(x, t, top=top))
    assert token_logprobs(x, top=3).top_indices[4, 0] == vocab // 2   # NaN stands above all


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [300, 5000, 49408])
def test_many_equal_logits(cuda, vocab, dtype):
    """Coarse values: ties at every border, decided by the index."""
    g = torch.Generator(device='cuda').manual_seed(1)
    for levels in (2, 5, 40):
        x = torch.randint(levels, (9, vocab), generator=g, device='cuda').to(dtype)
        for top in (1, 20, 128):
            Score(x, None, top).check(token_logprobs(x, top=top))
    # everything that counts in one stretch, as a vocabulary sorted by frequency has it
    x = logits_of(4, vocab, dtype)
    x[0, :200] += 40
    x[1, -200:] += 40
    x[2, 100:228] = 50
    x[3, ::vocab // 130] = 45
    Score(x, None, 128).check(token_logprobs(x, top=128))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [700, 2000, 3500, 9000, 49408, 140001])
def test_crowded_rows(cuda, vocab, dtype):
    """More places at the border than any list holds: equal values in a stretch, in the whole row, at its end, NaN among them,
    and the same among masked places."""
    g = torch.Generator(device='cuda').manual_seed(vocab)
    x = logits_of(8, vocab, dtype, spread=1.0)
    x[0] = -3.5                                                    # all equal and negative
    x[1, vocab // 3:] = 9                                          # ... behind a third of the row
    x[2, vocab // 2:] = torch.finfo(dtype).max
    x[3, :40] = 30                                                 # fewer than asked for above, the rest equal
    x[3, 40:] = -2
    x[4, torch.randperm(vocab, generator=g, device='cuda')[:vocab // 2]] = float('nan')
    x[5, :50] = float('nan')                                       # fewer NaN than asked for, then equal ones
    x[5, 50:] = 1
    x[6, :] = -INF
    x[6, vocab - 300:] = 0.125
    x[7] = torch.arange(vocab, device='cuda').to(dtype) * 1e-3     # (16 bits: steps of many places)
    mask = torch.rand(8, vocab, generator=g, device='cuda') < 0.6
    for top in (1, 20, 64, 128):
        Score(x, None, top).check(token_logprobs(x, top=top))
        Score(x, None, top, mask=mask).check(token_logprobs(x, top=top, mask=mask))
    if vocab < 4096:  # as many rows as another share of the work takes
        x, mask = x.repeat(256, 1), mask.repeat(256, 1)
        Score(x, None, 20, mask=mask).check(token_logprobs(x, top=20, mask=mask))


@pytest.mark.parametrize('vocab', [300, 6000, 60000])
def test_sizes_of_values(cuda, vocab):
    """Logits whose scaled size leaves no digits for their differences, that differ by many powers of ten, or that run
    through zero: log probabilities of d = scale * (x - max x), alternatives in the order of x."""
    x = logits_of(7, vocab, torch.float32)
    x[0] += 1e6                                                    # differences of whole steps of 1 / 16
    x[1] *= 1e20
    x[2] = x[2].abs() * 10 ** (torch.arange(vocab, device='cuda') % 30 - 15.0)
    x[3] = -x[3].abs() * 10 ** (torch.arange(vocab, device='cuda') % 30 - 15.0)
    x[4] *= 1e-30
    x[5, ::3] = -3e38
    x[6] = -torch.rand(vocab, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda') * 1e-6
    for scale in (1.0, 1e-3, 50.0):
        ours, ref = token_logprobs(x, top=100, scale=scale), Score(x, None, 100, scale=scale)
        assert torch.equal(ours.top_indices, ref.top_indices)
        # (z = scale * x in 64 bits has all digits of the fp32 product that lse is)
        close(ours.entropy, ref.h, ref.tol_h[:, 0] + 1e-9)
        close(ours.top_logprobs, ref.top_logprobs, ref.tol_top + 4 * E * ref.top_logprobs.abs())


def test_lists_of_many_chunks(cuda):
    """A vocabulary of 37 chunks with the longest lists: more keys than the join holds at once."""
    x = logits_of(3, 1200007, torch.float32)
    x[1] = 1.5  # every chunk's list is full of equal values
    t = some_targets(3, 1200007, 3)
    Score(x, t, 128).check(token_logprobs(x, t, top=128))
    ids, v = a_teacher(3, 1200007, 128)
    leaf = x.requires_grad_()
    up = torch.rand(3, device=cuda)
    loss = distill_top_logits(leaf, ids, v, tail=True)
    grad, = torch.autograd.grad([loss], [leaf], [up])
    Distill(leaf, ids, v, 1.0, True).check(loss, grad, up)


def test_large_logits_past_the_cache(cuda):
    """Logits of 300 MB and their gradient, read and written past the cache, row by row what a small call gives."""
    x = logits_of(1600, 49153, torch.float32).requires_grad_()
    t = some_targets(1600, 49153, 1)
    w = torch.rand(1600, 1, generator=torch.Generator().manual_seed(0)).to(cuda)
    out = token_logprobs(x, t, top=4)
    grad, = torch.autograd.grad([out.logprobs], [x], [w])
    ids, v = out.top_indices, out.top_logprobs.detach()
    g2, = torch.autograd.grad([distill_top_logits(x, ids, v, scale=0.5, tail=True)], [x], [w[:, 0]])
    for rows in (slice(0, 3), slice(797, 800), slice(1597, 1600)):
        s = x.detach()[rows].requires_grad_()
        small = token_logprobs(s, t[rows], top=4)
        assert all(torch.equal(a[rows], b) for a, b in zip(out, small))
        assert torch.equal(grad[rows], torch.autograd.grad([small.logprobs], [s], [w[rows]])[0])
        loss = distill_top_logits(s, ids[rows], v[rows], scale=0.5, tail=True)
        assert torch.equal(g2[rows], torch.autograd.grad([loss], [s], [w[rows, 0]])[0])


def test_clip_scale(cuda):
    """Cosines at CLIP's scale: the log probabilities keep their digits."""
    x = (logits_of(50, 1203, torch.float32, spread=0.03) + 0.2)
    t = some_targets(50, 1203, 1)
    Score(x, t, 20, scale=100.0).check(token_logprobs(x, t, top=20, scale=100.0))


def test_layouts(cuda):
    """Leading dimensions, strides, orders and offsets; every view gives what its copy gives, bit for bit."""
    base = logits_of(6, 1210, torch.float16, seed=2)
    views = [base[:, 3:1206], base[:, :1203], base[::2, 5:1208], base[1:2, :1203].expand(4, 1203),
             logits_of(1203, 6, torch.float16).t(), logits_of(2, 3 * 1203, torch.float16).view(2, 3, 1203),
             logits_of(24, 1203, torch.float16).view(2, 3, 4, 1203).permute(2, 0, 1, 3), base[0, 7:1210]]
    for v in views:
        t = torch.randint(1203, v.shape[:-1], device=cuda)
        got = token_logprobs(v, t, top=6)
        flat = v.reshape(-1, 1203).clone(memory_format=torch.contiguous_format)
        want = token_logprobs(flat, t.reshape(-1), top=6)
        Score(flat, t.reshape(-1, 1), 6).check(want._replace(logprobs=want.logprobs[:, None]))
        for a, b, more in zip(got, want, ((), (), (), (6,), (6,))):
            assert a.shape == v.shape[:-1] + more and torch.equal(a.reshape(b.shape), b)
        leaf = v.detach().requires_grad_()
        grad, = torch.autograd.grad(token_logprobs(leaf, t).logprobs.sum(), [leaf])
        fleaf = flat.requires_grad_()
        fgrad, = torch.autograd.grad(token_logprobs(fleaf, t.reshape(-1)).logprobs.sum(), [fleaf])
        assert torch.equal(grad.reshape(fgrad.shape), fgrad)
    # a mask with rows of its own stride, and one that repeats over leading dimensions
    x = logits_of(12, 100, torch.float32).view(3, 4, 100)
    wide = torch.rand(3, 4, 131, device=cuda) < 0.6
    for mask in (wide[..., 11:111], wide[:1, :, :100], wide[:, :1, 31:], wide[0, 0, :100]):
        got = token_logprobs(x, top=9, mask=mask)
        want = token_logprobs(x, top=9, mask=mask.expand(3, 4, 100).contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


def test_empty_shapes(cuda):
    out = token_logprobs(torch.empty(0, 9, device=cuda, requires_grad=True), torch.empty(0, 2, dtype=torch.int64, device=cuda), top=3)
    assert out.logprobs.shape == (0, 2) and out.lse.shape == (0,) and out.top_indices.shape == (0, 3)
    x = torch.randn(4, 9, device=cuda, requires_grad=True)
    out = token_logprobs(x, torch.empty(4, 0, dtype=torch.int64, device=cuda))
    assert out.logprobs.shape == (4, 0) and out.top_indices is None
    assert torch.equal(distill_top_logits(torch.empty(0, 9, device=cuda), torch.empty(0, 2, dtype=torch.int64, device=cuda),
                                          torch.empty(0, 2, device=cuda)), torch.empty(0, device=cuda))
    loss = distill_top_logits(x, torch.empty(4, 0, dtype=torch.int64, device=cuda), torch.empty(4, 0, device=cuda))
    grad, = torch.autograd.grad(loss.sum(), [x])
    assert (loss == 0).all() and (grad == 0).all()
    one = token_logprobs(torch.tensor([2.5], device=cuda), torch.tensor(0, device=cuda), top=1)
    assert one.logprobs == 0 and one.entropy == 0 and one.lse == 2.5 and one.top_indices.tolist() == [0]


def test_offsets_past_32_bits(cuda):
    """Rows more than 2^31 elements apart, forward and backward."""
    stride = 2 ** 30 + 24
    buf = torch.zeros(2 * stride + 1300, dtype=torch.float16, device=cuda)
    x = buf.as_strided((3, 1203), (stride, 1))
    small = logits_of(3, 1203, torch.float16, seed=4)
    x.copy_(small)
    t = some_targets(3, 1203, 2)
    for a, b in zip(token_logprobs(x, t, top=7), token_logprobs(small, t, top=7)):
        assert torch.equal(a, b)
    ids, lp = token_logprobs(small, top=9, scale=0.5).top_indices, token_logprobs(small, top=9, scale=0.5).top_logprobs
    grads = []
    for v in (x, small):
        leaf = v.detach().requires_grad_()
        loss = token_logprobs(leaf, t).logprobs.sum() + distill_top_logits(leaf, ids, lp, tail=True).sum()
        grads += torch.autograd.grad(loss, [leaf])
    assert torch.equal(*grads)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab', [(4, 1), (5, 9), (300, 65), (3, 511), (40, 1203), (6, 5001), (3, 49408), (2, 131073)])
def test_score_gradients(cuda, rows, vocab, dtype):
    x = logits_of(rows, vocab, dtype, seed=6).requires_grad_()
    t = some_targets(rows, vocab, 5, dtype=torch.int32)
    t[:, 1] = t[:, 0]  # the same token twice
    top = min(12, vocab + 2)
    g = torch.Generator(device='cuda').manual_seed(rows)
    out = token_logprobs(x, t, top=top, scale=1.3)
    ref = Score(x, t, top, scale=1.3)
    ref.check(out)
    named = dict(g_logprobs=out.logprobs, g_lse=out.lse, g_entropy=out.entropy, g_top=out.top_logprobs)
    ups = {k: torch.randn(o.shape, generator=g, device='cuda') for k, o in named.items()}
    for use in (['g_logprobs'], ['g_lse'], ['g_entropy'], ['g_top'], list(named)):
        grad, = torch.autograd.grad([named[k] for k in use], [x], [ups[k] for k in use], retain_graph=True)
        assert grad.dtype == dtype
        close(grad, *ref.grad(**{k: ups[k] for k in use}), what=use)


def test_out_of_range_targets_are_loud(cuda):
    x = logits_of(3, 50, torch.float32).requires_grad_()
    t = torch.tensor([4, 50, 49], device=cuda)
    out = token_logprobs(x, t)
    assert torch.isnan(out.logprobs).tolist() == [False, True, False]
    grad, = torch.autograd.grad(out.logprobs.sum(), [x])
    assert torch.isnan(grad).any(1).tolist() == [False, True, False]


class Distill:
    """The loss and its gradient in 64 bits."""

    def __init__(self, x, ids, v, scale=1.0, tail=False):
        s = Score(x, scale=scale)
        self.s, self.x, self.scale = s, x, scale
        ids, v = ids.long(), v.double()
        here = (ids >= 0) & (v > -INF)
        v = v.masked_fill(~here, -INF)
        self.none = ~here.any(1, keepdim=True)
        best = v.amax(1, keepdim=True).masked_fill(self.none, 0)
        if tail:
            self.q, log_q = v.exp(), v
        else:
            norm = best + (v - best).exp().sum(1, keepdim=True).masked_fill(self.none, 1).log()
            log_q = v - norm
            self.q = log_q.exp()
        at = ids.clamp_min(0)
        held = torch.zeros_like(s.p).scatter_add_(1, at, here.double()) > 0
        logp = s.logp.gather(1, at)
        term = (self.q * (log_q - logp)).masked_fill(self.q == 0, 0)
        loss = term.sum(1, keepdim=True)
        q_sum = self.q.sum(1, keepdim=True)
        self.rest = torch.zeros_like(loss)
        do = s.d.masked_fill(held, -INF)
        peak_o = do.amax(1, keepdim=True)
        none_o = peak_o == -INF
        eo = (do - peak_o.masked_fill(none_o, 0)).exp()
        so = eo.sum(1, keepdim=True).masked_fill(none_o, 1)
        log_po = peak_o.masked_fill(none_o, 0) + so.log() - s.log_s
        if tail:
            self.rest = (1 - q_sum).clamp_min(0).masked_fill(none_o, 0)
            loss = loss + (self.rest * (self.rest.clamp_min(1e-300).log() - log_po)).masked_fill(self.rest == 0, 0)
        self.loss = loss.masked_fill(self.none, 0).masked_fill(s.empty & ~self.none, INF)
        self.po, self.inside = log_po.exp(), eo / so
        grad = s.p * (q_sum + self.rest) - self.rest * self.inside * (~none_o)
        grad = grad.scatter_add(1, at, -self.q)
        self.grad = grad.masked_fill(self.none | s.empty, 0)
        self.w = torch.zeros_like(s.p).scatter_add(1, at, self.q)
        # |v| E for e^v, the sum of the terms, and what log p and the bucket's logarithm are off
        size = (self.q * (log_q.abs() + logp.abs())).masked_fill(self.q == 0, 0).masked_fill(s.dead, 0).sum(1, keepdim=True)
        off = (self.q * s.tol_logp.gather(1, at)).sum(1, keepdim=True)
        v_off = (self.q * v.masked_fill(~here, 0).abs()).sum(1, keepdim=True)
        bucket = (self.rest * (self.rest.clamp_min(1e-300).log().abs() + log_po.abs())).masked_fill(self.rest == 0, 0)
        self.tol = 2 * (off + E * (20 + ids.shape[1] / 64) * (size + v_off + bucket + q_sum)
                        + self.rest * (2 * s.tol_s + 4 * E * log_po.abs()) + 2 * E * q_sum)
        self.off_p = 2 * E * (3 * s.ad + 3 * s.log_s + 4) + s.tol_s

    def check(self, loss, grad, up):
        close(loss[:, None], self.loss, self.tol, 'loss')
        u = up.double()[:, None] * self.scale
        want = self.grad * u
        # outside the list e^(z - lse_o) (p_o q - rest): both products are off as p is, p_o by what two sums are
        size = self.s.p + self.rest * self.inside
        tol = u.abs() * (size * (2 * self.off_p + 4 * self.s.tol_s + 40 * E) + 16 * E * (self.w * (1 + self.w.clamp_min(1e-30).log().abs()) + self.s.p))
        close(grad, want, tol + half_step(want.abs() + tol, self.x.dtype), 'grad')


def a_teacher(rows, vocab, k, seed=0, index=torch.int64):
    """Distinct places of a teacher that has seen something like the student's logits."""
    z = logits_of(rows, vocab, torch.float32, seed=seed + 50)
    t = token_logprobs(z, top=min(k, 128))
    ids, v = t.top_indices.to(index), t.top_logprobs
    if k > 128:  # longer lists come from elsewhere
        ids = torch.argsort(z, 1, descending=True)[:, :k].to(index)
        v = torch.log_softmax(z, 1).gather(1, ids.long())
    return ids, v


@pytest.mark.parametrize('tail', [False, True])
@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, k', [(3, 1, 1), (4, 2, 1), (5, 9, 4), (5, 9, 9), (5, 9, 12), (300, 65, 8), (3, 511, 1),
                                            (40, 1203, 20), (7, 1203, 300), (6, 5001, 64), (3, 49408, 128), (2, 140001, 1000), (2100, 2301, 20)])
def test_distillation(cuda, rows, vocab, k, dtype, tail):
    x = logits_of(rows, vocab, dtype, seed=8).requires_grad_()
    ids, v = a_teacher(rows, vocab, k, index=torch.int32 if k % 2 else torch.int64)
    up = torch.rand(rows, device=cuda) + 0.5
    for scale in (1.0, 0.25):
        loss = distill_top_logits(x, ids, v, scale=scale, tail=tail)
        grad, = torch.autograd.grad([loss], [x], [up])
        assert grad.dtype == dtype
        Distill(x, ids, v, scale, tail).check(loss, grad, up)
        with torch.no_grad():
            assert torch.equal(distill_top_logits(x, ids, v, scale=scale, tail=tail), loss)


@pytest.mark.parametrize('tail', [False, True])
@pytest.mark.parametrize('vocab', [90, 3000, 70001])
def test_distillation_special_rows(cuda, vocab, tail):
    x = logits_of(9, vocab, torch.float32, seed=3)
    ids, v = (t.clone() for t in a_teacher(9, vocab, 16))
    ids[0] = -1                                  # no teacher: the index says so
    v[1] = -INF                                  # ... the log probability does
    ids[2, ::2] = -7                             # half a list
    ids[3, 4:8] = ids[3, 0]                      # an index five times over
    x[4] = -INF                                  # a student with one place, which the list has
    x[4, ids[4, 0]] = 2
    v[4, 1:] = -INF
    v[4, 0] = -0.25                              # (tail: the rest has nowhere to go and is left out)
    x[5, ids[5]] += 60                           # the student is sure of the list: its bucket is 1e-25
    x[6, ids[6]] -= 120                          # ... of the rest
    v[7] -= 40                                   # a teacher that gives the list nothing (tail), or any constant
    up = torch.rand(9, device=cuda) + 0.5
    leaf = x.requires_grad_()
    loss = distill_top_logits(leaf, ids, v, tail=tail)
    grad, = torch.autograd.grad([loss], [leaf], [up])
    Distill(x, ids, v, 1.0, tail).check(loss, grad, up)
    assert (loss[:2] == 0).all() and (grad[:2] == 0).all()


def test_distillation_infinite_and_not_a_number(cuda):
    x = logits_of(5, 100, torch.float32)
    ids, v = a_teacher(5, 100, 6)
    x[0, ids[0, 2]] = -INF                       # the student rules out what the teacher lists
    x[1] = -INF                                  # a student with nothing
    x[2, 7] = float('nan')
    ids = ids.clone()
    ids[3, 1] = 100                              # no such place
    leaf = x.requires_grad_()
    loss = distill_top_logits(leaf, ids, v)
    grad, = torch.autograd.grad(loss.sum(), [leaf])
    assert loss[0] == INF and loss[1] == INF and torch.isnan(loss[2:4]).all() and torch.isfinite(loss[4])
    want = torch.softmax(x.detach()[0].double(), 0).index_add(0, ids[0], -torch.softmax(v[0].double(), 0))
    torch.testing.assert_close(grad[0].double(), want, rtol=1e-5, atol=1e-6)
    assert (grad[1] == 0).all() and torch.isnan(grad[2:4]).any(1).all() and torch.isfinite(grad[4]).all()


def test_gradients_against_differences(cuda):
    """Central differences of the 64-bit definitions: the formulas, not only their evaluation.  With step h the quotient
    is off by h^2 / 6 times a third derivative of order 1."""
    h, x = 1e-4, logits_of(3, 40, torch.float32, seed=1)
    t = some_targets(3, 40, 2)
    t[0] = t[0].clamp_min(0)
    ids, v = a_teacher(3, 40, 7)
    functions = [
        (lambda a: token_logprobs(a, t, top=3, scale=1.5), lambda a: (lambda s: (s.logprobs, s.h, s.lse, s.top_logprobs))(Score(a, t, 3, scale=1.5))),
        (lambda a: (distill_top_logits(a, ids, v, scale=0.8),), lambda a: (Distill(a, ids, v, 0.8).loss[:, 0],)),
        (lambda a: (distill_top_logits(a, ids, v, scale=0.8, tail=True),), lambda a: (Distill(a, ids, v, 0.8, True).loss[:, 0],))]
    for ours, exact in functions:
        leaf = x.clone().requires_grad_()
        outs = [o for o in ours(leaf) if o is not None and o.dtype == torch.float32]
        ups = [torch.randn(o.shape, generator=torch.Generator().manual_seed(i)).to(cuda) for i, o in enumerate(outs)]
        grad, = torch.autograd.grad(outs, [leaf], ups)

        def value(z):
            return sum((o * u.double()).sum() for o, u in zip(exact(_Exact(z)), ups))
        for j in range(40):
            step = torch.zeros(3, 40, dtype=torch.float64, device=cuda)
            for r in range(3):
                step.zero_()[r, j] = h
                slope = (value(x.double() + step) - value(x.double() - step)) / (2 * h)
                assert abs(slope.item() - grad[r, j].item()) < 1e-5 * (1 + abs(slope.item())) * 5


class _Exact:
    """64-bit logits where Score and Distill take tensors of the operators' types."""

    def __init__(self, z):
        self.z, self.dtype = z, torch.float64

    def detach(self):
        return self

    def float(self):
        return self.z


def test_answers_do_not_depend_on_the_batch(cuda):
    """A row's values are those of the row alone, and repeat bit for bit."""
    for vocab, rows in ((65, 300), (1203, 64), (49408, 600)):
        x = logits_of(rows, vocab, torch.bfloat16, seed=7)
        t = some_targets(rows, vocab, 1)
        a, b = token_logprobs(x, t, top=10), token_logprobs(x, t, top=10)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
        one = token_logprobs(x[5:6], t[5:6], top=10)
        assert torch.equal(one.top_indices, a.top_indices[5:6])
        Score(x[5:6], t[5:6], 10).check(one)


def test_streams_devices_and_threads(cuda):
    """Another stream than the default one, and calls from two threads on two streams at once."""
    x = logits_of(64, 20000, torch.float16)
    t = some_targets(64, 20000, 1)
    want = token_logprobs(x, t, top=12)
    torch.cuda.synchronize()
    results = {}

    def work(name):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            results[name] = [token_logprobs(x, t, top=12) for _ in range(20)]
        s.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [th.start() for th in threads]
    [th.join() for th in threads]
    for r in results.values():
        assert len(r) == 20 and all(torch.equal(a, b) for got in r for a, b in zip(got, want))
    s = torch.cuda.Stream()
    leaf = x.clone().requires_grad_()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g1, = torch.autograd.grad(token_logprobs(leaf, t).logprobs.sum(), [leaf])
    s.synchronize()
    g2, = torch.autograd.grad(token_logprobs(leaf, t).logprobs.sum(), [leaf])
    assert torch.equal(g1, g2)


@pytest.mark.parametrize('rows, vocab', [(1, 49408), (300, 65), (40, 140001)])
def test_captured_and_replayed(cuda, rows, vocab):
    """A teacher's call, the student's loss and the gradient in one graph, and a second graph of the same calls: replayed in
    turn with eager work between, on new inputs each time."""
    teacher, student = logits_of(rows, vocab, torch.float16), logits_of(rows, vocab, torch.float16)
    t = some_targets(rows, vocab, 1)
    up = torch.full((rows,), 0.25, device=cuda)

    def step(a, b):
        b = b.detach().requires_grad_()
        with torch.no_grad():
            best = token_logprobs(a, t, top=16)
        loss = distill_top_logits(b, best.top_indices, best.top_logprobs, tail=True)
        grad, = torch.autograd.grad([loss], [b], [up])
        own = token_logprobs(b, t)
        g2, = torch.autograd.grad([own.logprobs, own.entropy], [b], [up[:, None], up])
        return best.top_indices, best.top_logprobs, loss.detach(), grad, own.lse.detach(), g2

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(teacher, student)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(teacher, student)
        graphs.append((g, out))
    for seed in range(4):
        teacher.copy_(logits_of(rows, vocab, torch.float16, seed=seed + 20))
        student.copy_(logits_of(rows, vocab, torch.float16, seed=seed + 40))
        want = [w.clone() for w in step(teacher, student)]
        for g, out in graphs:
            for o in out:
                o.fill_(0)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals_on_the_device(cuda):
    x = torch.randn(3, 7, device=cuda)
    with pytest.raises(ValueError):
        token_logprobs(x, torch.zeros(3, dtype=torch.int64))             # targets on the CPU
    with pytest.raises(ValueError):
        token_logprobs(x, mask=torch.ones(7, dtype=torch.bool))
    with pytest.raises(ValueError):
        distill_top_logits(x, torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2))
    lib = _lib.load()
    with pytest.raises(_lib.OakeError, match='scale'):
        _lib.check(lib, None, lib.oake_logits_workspace(1, 1, 0, 500, None), 'scale')
    leaf = x.clone().requires_grad_()
    out = token_logprobs(leaf)
    g, = torch.autograd.grad(out.lse.sum(), [leaf], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), [leaf])                             # differentiable once


def test_classify(cuda):
    """CLIP.classify: crops through the encoder, against label embeddings, answered."""
    model, _ = clip.load(synthetic_state_dict(width=128, layers=2, heads=2, mlp_dim=256, embed_dim=64), max_batch=8)
    x = synthetic_images(6, seed=3).to(cuda)
    labels = torch.randn(65, 64, generator=torch.Generator().manual_seed(0)).to(cuda) * 3
    mask = torch.ones(65, dtype=torch.bool, device=cuda)
    mask[48:] = False
    t = torch.tensor([0, 1, 2, 47, 48, -1], device=cuda)
    got = model.classify(x, labels, targets=t, top=4, mask=mask)
    e = model.encode_image(x, normalize=True, out_dtype=torch.float32)
    logits = label_logits(e, labels)
    cos = torch.nn.functional.normalize(e.double(), dim=1) @ torch.nn.functional.normalize(labels.double(), dim=1).t()
    close(logits, cos, torch.full_like(cos, 2 * (64 + 8) * E))  # 64 products and two norms
    want = Score(logits, t[:, None], 4, mask=mask, scale=100.0)
    want.check(got._replace(logprobs=got.logprobs[:, None]))
    assert got.logprobs[4] == -INF and got.logprobs[5] == 0 and (got.top_indices < 48).all()


@pytest.mark.parametrize('temperature', [1.0, 4.0])
@pytest.mark.parametrize('n, top, tail', [(65, 8, False), (65, 100, True), (1203, 20, True)])
def test_teacher_and_student(cuda, n, top, tail, temperature):
    """TopLogitsDistillation: stored embeddings -> the teacher's lists -> the student's loss and its logits' gradient, as
    one step and from a stored list; a student that answers as the teacher does has nothing to learn."""
    g = torch.Generator().manual_seed(n)
    labels = torch.randn(n, 512, generator=g).to(cuda)
    embeddings = (torch.randn(2, 40, 512, generator=g).to(cuda) + labels[torch.randint(n, (2, 40), generator=g)]).half()
    head = TopLogitsDistillation(labels, top=top, scale=50.0, temperature=temperature, tail=tail)
    student = torch.randn(2, 40, n, generator=g).to(cuda).requires_grad_()
    loss = head(student, embeddings)
    up = torch.rand(2, 40, generator=g).to(cuda)
    grad, = torch.autograd.grad([loss], [student], [up])
    ids, v = head.teacher(embeddings)
    assert ids.shape == (2, 40, min(top, n)) and not v.requires_grad
    stored = head(student, teacher=(ids, v))
    assert torch.equal(loss, stored)
    ref = Distill(student.detach().reshape(80, n), ids.reshape(80, -1), v.reshape(80, -1), 1 / temperature, tail)
    ref.tol = ref.tol + 4 * E * ref.loss.abs()  # (divided and multiplied by T^2: 16, exact; T itself: exact)
    ref.check(loss.reshape(80) / temperature ** 2, grad.reshape(80, n), up.reshape(80) * temperature ** 2)
    same = (label_logits(embeddings, head.labels) * 50.0).requires_grad_()
    learnt = head(same, embeddings)
    grad, = torch.autograd.grad(learnt.sum(), [same])
    if tail or top >= n:  # (a renormalised list differs from the teacher's whole distribution)
        # the logits 50 cos are rounded once more than the teacher's, each by 50 E at most: p moves by 100 E p, the loss
        # by its second order; the rest is what the loss and p may be off anyway
        ref = Distill(same.detach().reshape(80, n), ids.reshape(80, -1), v.reshape(80, -1), 1 / temperature, tail)
        assert (learnt.reshape(80, 1).abs() <= temperature ** 2 * (ref.tol + 8 * E)).all()
        assert grad.abs().max() <= temperature * (2 * ref.off_p.max() + 200 * E)


@pytest.mark.parametrize('dtype', (torch.float16, torch.bfloat16, torch.float32))
@pytest.mark.parametrize('vocab', (1, 7, 9, 2056, 8192, 16385, 16392, 33288, 49407, 65536, 65537, 131071, 200003))
def test_rows_at_any_element(cuda, dtype, vocab):
    """The same rows from an even and from an odd element on, NaN before, between and behind them: the same bits."""
    x = logits_of(3, vocab, dtype)
    outs = []
    for offset, gap in ((0, 8 - vocab % 8), (1, 1 + vocab % 2), (3, 8 - vocab % 8), (2, 1 + vocab % 2), (0, 1 - vocab % 2 + 1)):
        buf = torch.full((offset + 3 * (vocab + gap) + 8,), float('nan'), dtype=dtype, device=cuda)
        rows = torch.as_strided(buf, (3, vocab), (vocab + gap, 1), offset)
        rows.copy_(x)
        a = token_logprobs(rows, torch.tensor([0, vocab - 1, vocab // 2], device=cuda), top=min(vocab, 24))
        losses = [distill_top_logits(rows, a.top_indices, a.top_logprobs, scale=0.7, tail=tail) for tail in (False, True)]
        leaf = rows.detach().requires_grad_()
        grad, = torch.autograd.grad(token_logprobs(leaf).entropy.sum(), [leaf])
        outs.append([*a, *losses, grad])
    assert not outs[0][2].isnan().any()
    for other in outs[1:]:
        assert all(torch.equal(w, o) for w, o in zip(outs[0], other))


@pytest.mark.parametrize('rows, vocab', [(5, 1), (7, 65), (6, 1203), (3, 49409)])
def test_saved_tensors_that_come_back_packed(cuda, rows, vocab):
    """Logits and a mask with rows of their own strides, moved to the host and back between the two passes."""
    base = logits_of(rows, vocab + 13, torch.float16)
    allowed = torch.rand(rows, vocab + 70, device=cuda) < 0.7
    allowed[:, 11] = True
    x, mask, t = base[:, 5:5 + vocab], allowed[:, 11:11 + vocab], some_targets(rows, vocab, 2)
    up = torch.randn(rows, device=cuda)

    def step():
        leaf = x.detach().requires_grad_()
        a = token_logprobs(leaf, t, top=3, mask=mask)
        loss = distill_top_logits(leaf, a.top_indices, a.top_logprobs.detach(), scale=0.5, tail=True)
        return torch.autograd.grad([a.logprobs, a.entropy, a.top_logprobs, loss], [leaf],
                                   [up[:, None].expand(rows, 2), up, up[:, None].expand(rows, 3), up])[0]

    want = step()
    with torch.autograd.graph.save_on_cpu():
        got = step()
    assert torch.equal(got, want)
    assert vocab == 1 or want.abs().sum() > 0


@pytest.mark.parametrize('tail', [False, True])
@pytest.mark.parametrize('vocab, k', [(1, 1), (2, 2), (3, 3), (3, 2), (9, 4), (33, 33), (64, 20)])
def test_nearly_equal_distributions(cuda, vocab, k, tail):
    """Few classes, a student that has nearly learnt its teacher: the loss is 1e-4 and less, and right relative to its terms.

    Tolerance, relative to sum q |log q - log p|: e^(v - log norm) 2^-21 (an argument of up to 16) and 2^-22, the logarithms'
    difference and the product 2^-24 each, a sum of up to 64 terms over lanes 7 * 2^-24: less than 2^-19 together.  The bucket
    is rounded to fp32: its own 2^-24, and that of the product with its logarithm."""
    x = logits_of(512, vocab, torch.float32, seed=4)
    noise = torch.randn(512, vocab, generator=torch.Generator().manual_seed(5)).to(cuda) * 0.01
    best = token_logprobs(x + noise, top=k)
    loss = distill_top_logits(x, best.top_indices, best.top_logprobs, tail=tail).double()
    logp = torch.log_softmax(x.double(), 1)
    v, lp = best.top_logprobs.double(), logp.gather(1, best.top_indices)
    log_q = v if tail else v - torch.logsumexp(v, 1, keepdim=True)
    terms = log_q.exp() * (log_q - lp)
    want, tol = terms.sum(1), 2.0 ** -19 * terms.abs().sum(1) + 1e-14
    if tail and k < vocab:
        rest = (1 - log_q.exp().sum(1)).clamp_min(0)
        p_o = logp.exp().scatter(1, best.top_indices, 0).sum(1)
        last = torch.where(rest > 0, rest * (rest.clamp_min(1e-300).log() - p_o.log()), torch.zeros_like(rest))
        want, tol = want + last, tol + 2.0 ** -19 * last.abs() + 2.0 ** -23 * rest
    assert ((loss - want).abs() <= tol).all(), ((loss - want).abs() / tol).max()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [1, 2, 65, 1203, 3001, 9000, 49408, 140001])
def test_a_single_place_leaves_nothing_open(cuda, vocab, dtype):
    """One place with a probability: entropy and log probability are 0, not about 0."""
    at = vocab // 2
    x = logits_of(40, vocab, dtype, seed=11)
    mask = torch.zeros(vocab, dtype=torch.bool, device=cuda)
    mask[at] = True
    alone = x.masked_fill(~mask, -INF)
    t = torch.full((40,), at, device=cuda)
    for scale in (1.0, 0.7, 100.0):
        for out in (token_logprobs(x, t, top=2, mask=mask, scale=scale), token_logprobs(alone, t, top=2, scale=scale)):
            assert (out.entropy == 0).all() and (out.logprobs == 0).all() and (out.top_logprobs[:, 0] == 0).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab, n', [(1, 1), (2, 1), (65, 1), (65, 70), (3001, 1), (9000, 1), (140001, 1)])
def test_a_single_place_has_nothing_to_learn(cuda, vocab, n, dtype):
    """A student with one place and a teacher that lists it: loss and gradient are 0, not about 0."""
    at = vocab // 2
    x = logits_of(40, vocab, dtype, seed=11)
    x[:, :at] = x[:, at + 1:] = -INF
    ids = torch.full((40, n), -1, device=cuda)
    ids[:, n // 2] = at
    for scale in (1.0, 0.7, 100.0):
        for tail, v in ((True, 0.0), (False, 0.0), (False, -3.7)):
            leaf = x.clone().requires_grad_()
            loss = distill_top_logits(leaf, ids, torch.full((40, n), v, device=cuda), scale=scale, tail=tail)
            grad, = torch.autograd.grad(loss.sum(), [leaf])
            assert (loss == 0).all() and (grad == 0).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows, vocab, step', [(4, 9, 1), (7, 9, 2), (5, 65, 1), (6, 1203, 1), (3, 9000, 1), (3, 140001, 1)])
def test_gradients_of_rows_that_overlap(cuda, rows, vocab, step, dtype):
    """Sliding windows over one buffer: every row's gradient is what a copy's is, bit for bit."""
    buf = logits_of(1, vocab + (rows - 1) * step, dtype, seed=12)[0]
    views = [buf.unfold(0, vocab, step), buf.as_strided((rows, vocab), (step, 1))]
    allowed = (torch.arange(vocab + rows, device=cuda) % 3 > 0).unfold(0, vocab, 1)[:rows]
    t = some_targets(rows, vocab, 2)
    ids, v = a_teacher(rows, vocab, min(8, vocab))
    up = torch.rand(rows, generator=torch.Generator().manual_seed(0)).to(cuda) + 0.5
    for view in views:
        assert view.shape == (rows, vocab) and view.stride() == (step, 1)
        grads = []
        for x in (view, view.clone(memory_format=torch.contiguous_format)):
            leaf = x.detach().requires_grad_()
            a = token_logprobs(leaf, t, top=3, mask=allowed)
            loss = distill_top_logits(leaf, ids, v, scale=0.5, tail=True)
            grads.append((*torch.autograd.grad([a.logprobs, a.entropy, a.top_logprobs], [leaf],
                                               [up[:, None].expand(rows, 2), up, up[:, None].expand(rows, 3)]),
                          *torch.autograd.grad([loss], [leaf], [up])))
        for ours, copy in zip(*grads):
            assert torch.equal(ours, copy) and copy.abs().sum() > 0
        want, tol = Score(view, t, 3, mask=allowed).grad(g_logprobs=up[:, None].expand(rows, 2), g_entropy=up,
                                                         g_top=up[:, None].expand(rows, 3))
        close(grads[0][0], want, tol)


@pytest.mark.parametrize('shift', [0.0, 30.0, -300.0, 1e3, -1e5])
@pytest.mark.parametrize('vocab, k', [(65, 8), (1203, 64), (5000, 200), (140001, 100)])
def test_teachers_up_to_a_constant(cuda, vocab, k, shift):
    """A renormalised list may stand at any height: loss and gradient are those of its differences.  (The reference takes the
    shifted entries as they came out in fp32, less the shift: exact in 64 bits.)"""
    x = logits_of(6, vocab, torch.float32, seed=13).requires_grad_()
    ids, v = a_teacher(6, vocab, k)
    v = v + shift
    up = torch.rand(6, generator=torch.Generator().manual_seed(0)).to(cuda) + 0.5
    loss = distill_top_logits(x, ids, v)
    grad, = torch.autograd.grad([loss], [x], [up])
    Distill(x, ids, v.double() - shift).check(loss, grad, up)
    # p and q both sum to 1: each of the 2 k terms p_j - q_j and the sum of the others is off by 16 steps of its size at most
    assert (grad.double().sum(1).abs() <= 32 * E * 2 * up).all()


def nearly_equal(vocab, k, pad, tail, rows=512):
    """(loss, 64-bit loss) of a student that has nearly learnt its teacher; lists padded to k + pad."""
    x = logits_of(rows, vocab, torch.float32, seed=4)
    noise = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(5)).cuda() * 0.01
    best = token_logprobs(x + noise, top=k)
    ids = torch.nn.functional.pad(best.top_indices, (0, pad), value=-1)
    loss = distill_top_logits(x, ids, torch.nn.functional.pad(best.top_logprobs, (0, pad), value=-INF), tail=tail).double()
    logp = torch.log_softmax(x.double(), 1)
    v, lp = best.top_logprobs.double(), logp.gather(1, best.top_indices)
    log_q = v if tail else v - torch.logsumexp(v, 1, keepdim=True)
    terms = log_q.exp() * (log_q - lp)
    if tail and k < vocab:
        rest = (1 - log_q.exp().sum(1, keepdim=True)).clamp_min(0)
        p_o = logp.exp().scatter(1, best.top_indices, 0).sum(1, keepdim=True)
        terms = torch.cat([terms, torch.where(rest > 0, rest * (rest.clamp_min(1e-300).log() - p_o.log()), torch.zeros_like(rest))], 1)
    return loss, terms.sum(1)


@pytest.mark.parametrize('tail', [False, True])
@pytest.mark.parametrize('vocab, k', [(2, 1), (3, 3), (9, 4), (13, 1), (23, 5), (33, 33), (52, 50), (64, 20)])
def test_small_losses_have_all_their_digits(cuda, vocab, k, tail):
    """Tolerance: the loss is rounded once, 2^-24 of it, doubled; e^y in 64 bits is off by 1e-13 of terms of 1e-2."""
    loss, want = nearly_equal(vocab, k, 0, tail)
    assert ((loss - want).abs() <= 2.0 ** -23 * want.abs() + 1e-14).all(), ((loss - want) / want).abs().max()


@pytest.mark.parametrize('tail', [False, True])
@pytest.mark.parametrize('vocab, k, pad', [(65, 8, 0), (65, 65, 0), (65, 8, 60), (100, 20, 0), (128, 128, 0), (7, 7, 93), (7, 3, 1000),
                                           (2, 2, 63), (64, 20, 280), (128, 100, 0)])
def test_sums_of_short_rows_whatever_the_list(cuda, vocab, k, pad, tail):
    """Rows of up to 128 places have the same digits whatever the length of the list.  Tolerance as above."""
    loss, want = nearly_equal(vocab, k, pad, tail)
    assert ((loss - want).abs() <= 2.0 ** -23 * want.abs() + 1e-14).all(), ((loss - want) / want).abs().max()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('vocab', [65, 1203, 2049, 3000, 4096, 9000, 49408, 140001])
def test_bits_do_not_depend_on_the_batch(cuda, vocab, dtype):
    """Every output and gradient of a row is the same, bit for bit, alone, among a few rows and among many."""
    many = 2100 if vocab < 5000 else 300
    x = logits_of(many, vocab, dtype, seed=14)
    t = some_targets(many, vocab, 2)
    up = torch.rand(many, generator=torch.Generator().manual_seed(0)).to(cuda) + 0.5
    ids, v = a_teacher(many, vocab, 20)

    def step(rows, top, tail):
        leaf = x[rows].detach().requires_grad_()
        n, u = leaf.shape[0], up[rows]
        a = token_logprobs(leaf, t[rows], top=top, scale=0.9)
        loss = distill_top_logits(leaf, ids[rows], v[rows], scale=0.5, tail=tail)
        return [*a, loss, *torch.autograd.grad([a.logprobs, a.entropy], [leaf], [u[:, None].expand(n, 2), u]),
                *torch.autograd.grad([loss], [leaf], [u])]

    for top, tail in ((20, False), (33, True)):
        whole = step(slice(0, many), top, tail)
        for rows in (slice(5, 6), slice(3, 10), slice(0, many - 60)):
            for name, (a, b) in enumerate(zip(step(rows, top, tail), whole)):
                assert torch.equal(a, b[rows]), (rows, top, name)
