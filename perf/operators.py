"""Cases that time the operators on logits (``oadp_amd.clip.logits``) and compare them with a plain form.

Two operators, each forward and backward:

* ``token_logprobs``: over every row of logits, the log probabilities of given tokens (labels), the entropy, the log of
  the partition sum and the top alternatives - what a classifier answers, and what a teacher leaves behind for a student;
* ``distill_top_logits``: the loss of a student's logits against such a teacher's list, with its gradient.

``own`` selects the framework's kernels; otherwise ``run`` is elementary torch in 32 bits, rounded once at the end.
"""
import torch

own = False

DTYPES = dict(f32=torch.float32, f16=torch.float16, bf16=torch.bfloat16)
SIZE = dict(f32=4, f16=2, bf16=2)
INF = float('inf')
MOST_BYTES = 2048 * 131071 * 2  # of logits, in any case


def listed():
    def case(name, kind, rows, vocab, dtype, **more):
        return dict(dict(name=name, kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=0, given=1, mask='none', pad=0,
                         cosine=False, tail=False), **more)

    return [
        # the 300 proposals of one image against the 65 OV-COCO labels, the dataset's own ones allowed: latency
        case('proposals-65', 'score', 300, 65, 'f32', top=5, mask='labels', cosine=True),
        # one new token, or one caption's next word, over the text tower's vocabulary: a single row
        case('one-row-49408', 'score', 1, 49408, 'f16', top=5),
        # the 1728 block crops of a flush of 64 images over LVIS' labels (an odd row length), allowed labels per image
        case('blocks-1203', 'score', 1728, 1203, 'f16', top=20, given=3, mask='rows', cosine=True),
        # a few rows at a time over a long odd vocabulary, with long lists: single steps of a batch
        case('few-rows-200003', 'score', 16, 200003, 'f32', top=100, given=2),
        # scoring a batch of texts token by token
        case('texts-49408', 'score', 4096, 49408, 'bf16', top=20),
        # a teacher's lists for a long vocabulary: the largest
        case('teacher-131071', 'score', 2048, 131071, 'bf16', top=64, given=0),
        # training on log probabilities with an entropy bonus, several labels a crop, rows behind each other with a gap
        case('train-1203', 'train', 777, 1203, 'f32', given=4, mask='rows', pad=5),
        # the same over the text vocabulary
        case('train-49408', 'train', 2048, 49408, 'f16', top=8),
        # a detector head's proposals distilled from an image's teacher: the smallest training call
        case('distill-65', 'distill', 300, 65, 'f32', top=8),
        # 8 images of 300 proposals over LVIS' labels, what the list leaves out held in one bucket
        case('distill-1203', 'distill', 2400, 1203, 'f16', top=20, tail=True),
        # text tokens, lists renormalised
        case('distill-49408', 'distill', 4096, 49408, 'bf16', top=64),
        # a long odd vocabulary in 32 bits, with the bucket
        case('distill-100003', 'distill', 1024, 100003, 'f32', top=32, tail=True),
    ]


def draw(rng):
    kind = rng.choice(('score', 'score', 'train', 'distill', 'distill'))
    dtype = rng.choice(sorted(DTYPES))
    vocab = int(2 ** rng.uniform(0, 18)) | rng.choice((0, 1))
    most = MOST_BYTES // (SIZE[dtype] * vocab * (1 if kind == 'score' else 2))
    rows = max(1, int(2 ** rng.uniform(0, 13)))
    rows = max(1, min(rows, most))
    top = rng.choice((1, 3, 5, 8, 20, 50, 64, 100, 128))
    if kind != 'distill' and rng.random() < 0.25:
        top = 0
    return dict(kind=kind, rows=rows, vocab=vocab, dtype=dtype, top=top, given=rng.choice((1, 1, 2, 5)),
                mask=rng.choice(('none', 'none', 'labels', 'rows')) if kind != 'distill' else 'none',
                pad=rng.choice((0, 0, 0, 1, 8, 61)), cosine=rng.random() < 0.3,
                tail=kind == 'distill' and rng.random() < 0.5)


def prepare(case, seed):
    rows, vocab, dtype = case['rows'], case['vocab'], DTYPES[case['dtype']]
    dev = torch.device('cuda')
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *s: torch.rand(*s, generator=g, device=dev)  # noqa: E731
    buf = torch.randn(rows, vocab + case['pad'], generator=g, device=dev)
    if case['cosine']:  # cosines of normalised embeddings, answered at CLIP's scale
        buf = buf.mul_(0.03).add_(0.2)
        scale = 100.0
    else:               # a language model's: broad, with a few tokens that stand out in each row
        buf = buf.mul_(2.0).sub_(3.0)
        peaks = torch.randint(vocab, (rows, 6), generator=g, device=dev)
        buf.scatter_add_(1, peaks, 4 + 8 * rand(rows, 6))
        scale = 1.0
    buf = buf.to(dtype)
    logits = buf[:, :vocab]
    state = dict(kind=case['kind'], scale=scale, top=case['top'], tail=case['tail'], mask=None, targets=None)

    if case['mask'] != 'none':
        shape = (vocab,) if case['mask'] == 'labels' else (rows, vocab)
        mask = rand(*shape) < 0.7
        if case['mask'] == 'labels':
            mask[torch.randint(vocab, (1,), generator=g, device=dev)] = True
        elif rows > 3:
            mask[2] = False  # a row that is padding: nothing is allowed
        state['mask'] = mask
        # what stands in masked places is not to be read: some of it is no number
        logits.masked_fill_(~mask & (rand(rows, vocab) < 0.1), float('nan'))
    if case['kind'] != 'distill' and case['given']:
        targets = torch.randint(vocab, (rows, case['given']), generator=g, device=dev)
        if rows > 3:
            targets[1] = -1  # padding
        state['targets'] = targets
    if case['kind'] == 'train':
        state['g_logprobs'] = torch.randn(rows, case['given'], generator=g, device=dev) / rows
        state['g_entropy'] = torch.randn(rows, generator=g, device=dev) * 0.1 / rows
    if case['kind'] == 'distill':
        k = min(case['top'], vocab)
        z = logits.float() * scale
        z += torch.randn(rows, vocab, generator=g, device=dev)
        values, ids = torch.topk(torch.log_softmax(z, 1), k, 1)
        if case['top'] > k:  # lists longer than the vocabulary are filled up
            values = torch.nn.functional.pad(values, (0, case['top'] - k), value=-INF)
            ids = torch.nn.functional.pad(ids, (0, case['top'] - k), value=-1)
        if rows > 3:  # a row that no teacher saw
            ids[3], values[3] = -1, -INF
        state['top_indices'], state['top_logprobs'] = ids.contiguous(), values.contiguous()
        state['g_loss'] = (0.5 + rand(rows)) / rows
    if case['kind'] != 'score':
        logits = logits.detach().requires_grad_()
    state['logits'] = logits
    return state


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_distill(state) if state['kind'] == 'distill' else _plain_logprobs(state)


def _own(s):
    from oadp_amd.clip.logits import distill_top_logits, token_logprobs
    if s['kind'] == 'distill':
        loss = distill_top_logits(s['logits'], s['top_indices'], s['top_logprobs'], scale=s['scale'], tail=s['tail'])
        grad, = torch.autograd.grad([loss], [s['logits']], [s['g_loss']])
        return dict(loss=loss.detach(), grad=grad)
    a = token_logprobs(s['logits'], s['targets'], top=s['top'], mask=s['mask'], scale=s['scale'])
    out = dict(lse=a.lse.detach(), entropy=a.entropy.detach())
    if s['targets'] is not None:
        out['logprobs'] = a.logprobs.detach()
    if s['top']:
        out['top_logprobs'], out['top_indices'] = a.top_logprobs.detach(), a.top_indices
    if s['kind'] == 'train':
        out['grad'], = torch.autograd.grad([a.logprobs, a.entropy], [s['logits']], [s['g_logprobs'], s['g_entropy']])
    return out


def _plain_logprobs(s):
    """z = scale * logits over the allowed places; d = z - max z; lse = max z + log sum e^d; H = log sum e^d - sum p d."""
    x, scale, top, targets = s['logits'].float(), s['scale'], s['top'], s['targets']
    if s['mask'] is not None:
        x = x.masked_fill(~s['mask'], -INF)
    peak = x.amax(1, keepdim=True)
    empty = peak == -INF
    d = (x - peak.masked_fill(empty, 0)) * scale
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    p = e / total.masked_fill(empty, 1)
    mean = (p * d.masked_fill(e == 0, 0)).sum(1, keepdim=True)
    entropy = (log_total - mean).masked_fill(empty, 0)
    out = dict(lse=(peak * scale + log_total)[:, 0], entropy=entropy[:, 0])
    if targets is not None:
        given = (d.gather(1, targets.clamp_min(0)) - log_total).masked_fill(empty, -INF)
        out['logprobs'] = given.masked_fill(targets < 0, 0)
    if top:
        k = min(top, x.shape[1])
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        best = (d.gather(1, order) - log_total).masked_fill(empty, -INF)
        order = order.masked_fill(best == -INF, -1)
        if top > k:
            order = torch.nn.functional.pad(order, (0, top - k), value=-1)
            best = torch.nn.functional.pad(best, (0, top - k), value=-INF)
        out['top_logprobs'], out['top_indices'] = best, order
    if s['kind'] == 'train':
        # d logp_t / dz_j = [j = t] - p_j;  dH / dz_j = -p_j (log p_j + H)
        g = s['g_logprobs'].masked_fill((targets < 0) | (given == -INF), 0)
        logp = (d - log_total).masked_fill(e == 0, 0)
        grad = -p * (g.sum(1, keepdim=True) + s['g_entropy'][:, None] * (logp + entropy))
        grad = grad.masked_fill(empty, 0).scatter_add_(1, targets.clamp_min(0), g) * scale
        out['grad'] = grad.to(s['logits'].dtype)
    return out


def _plain_distill(s):
    """KL(q || p) per row: q the teacher's list, renormalised or with a bucket for the rest; p the student's softmax."""
    x, scale, tail = s['logits'].float(), s['scale'], s['tail']
    ids, v = s['top_indices'], s['top_logprobs'].double()
    v = v.masked_fill(ids < 0, -INF)
    none = (v == -INF).all(1, keepdim=True)
    at = ids.clamp_min(0)
    z = x * scale
    peak = z.amax(1, keepdim=True)
    d = z - peak
    e = d.exp()
    total = e.sum(1, keepdim=True)
    logp = d.gather(1, at).double() - total.log().double()
    if tail:
        log_q = v
        q = v.exp()
        rest = (1 - q.sum(1, keepdim=True)).clamp_min(0)
    else:
        best = v.amax(1, keepdim=True).masked_fill(none, 0)
        log_q = v - best - (v - best).exp().sum(1, keepdim=True).log()
        q = log_q.exp().masked_fill(none, 0)
    loss = (q * (log_q - logp)).masked_fill(q == 0, 0).sum(1, keepdim=True)
    p = e / total
    grad = p * (q.sum(1, keepdim=True)).float()
    if tail:
        # places that the list does not hold
        outside = torch.zeros_like(x).scatter_add_(1, at, (v > -INF).float()) == 0
        zo = z.masked_fill(~outside, -INF)
        peak_o = zo.amax(1, keepdim=True)
        no_rest = peak_o == -INF
        eo = (zo - peak_o.masked_fill(no_rest, 0)).exp()
        total_o = eo.sum(1, keepdim=True)
        log_rest = ((peak_o - peak).masked_fill(no_rest, 0) + total_o.masked_fill(no_rest, 1).log()
                    - total.log()).double()
        rest = rest.masked_fill(no_rest, 0)
        loss = loss + (rest * (rest.clamp_min(1e-300).log() - log_rest)).masked_fill(rest == 0, 0)
        grad = p * (q.sum(1, keepdim=True) + rest).float() - eo / total_o.masked_fill(no_rest, 1) * rest.float()
    grad = grad.scatter_add_(1, at, -q.float()).masked_fill(none, 0)
    grad = (grad * (s['g_loss'][:, None] * scale)).to(s['logits'].dtype)
    return dict(loss=loss[:, 0].masked_fill(none[:, 0], 0).float(), grad=grad)


def work(case):
    n = case['rows'] * case['vocab']
    b = n * SIZE[case['dtype']] * (1 if case['kind'] == 'score' else 2)
    b += n if case['mask'] == 'rows' else case['vocab'] if case['mask'] == 'labels' else 0
    b += case['rows'] * (8 + case['top'] * 12 + (case['given'] * 12 if case['kind'] != 'distill' else 0))
    # a difference, a product, an exponential, two sums; backward an exponential and two products more
    return dict(bytes=b, flops=n * (6 if case['kind'] == 'score' else 11))


def exact(case, seed):
    """From the definitions, row by row blocks, in 64 bits."""
    s = prepare(case, seed)
    rows = case['rows']
    step = max(1, 2 ** 27 // case['vocab'])
    parts = [_exact_rows(s, slice(a, min(rows, a + step))) for a in range(0, rows, step)]
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    if case['kind'] != 'distill' and case['top']:
        out['top_indices'] = None
    return out


def _exact_rows(s, r):
    z = s['logits'].detach()[r].double() * s['scale']
    n, vocab = z.shape
    if s['mask'] is not None:
        mask = s['mask'] if s['mask'].dim() == 1 else s['mask'][r]
        z = torch.where(mask, z, torch.full_like(z, -INF))
    alive = torch.isfinite(z).any(1)
    lse = torch.logsumexp(z, 1)
    logp = torch.where(alive[:, None], z - lse[:, None], torch.full_like(z, -INF))
    p = logp.exp()
    row = torch.arange(n, device=z.device)[:, None]
    if s['kind'] == 'distill':
        ids, v = s['top_indices'][r], s['top_logprobs'][r].double()
        seen = (ids >= 0) & (v > -INF)
        weight = torch.where(seen, v, torch.full_like(v, -INF)).exp()
        if not s['tail']:
            weight = weight / weight.sum(1, keepdim=True).clamp_min(1e-300)
        q = torch.zeros_like(z)
        q.index_put_((row.expand_as(ids), ids.clamp_min(0)), weight, accumulate=True)
        loss = torch.where(q > 0, q * (q.clamp_min(1e-300).log() - logp), torch.zeros_like(q)).sum(1)
        held = torch.zeros_like(z).index_put_((row.expand_as(ids), ids.clamp_min(0)), seen.double(), accumulate=True) > 0
        grad = p * q.sum(1, keepdim=True) - q
        if s['tail']:
            rest = (1 - weight.sum(1)).clamp_min(0)
            lse_rest = torch.logsumexp(torch.where(held, torch.full_like(z, -INF), z), 1)
            rest = torch.where(torch.isfinite(lse_rest), rest, torch.zeros_like(rest))
            some = rest > 0
            loss = loss + torch.where(some, rest * (rest.clamp_min(1e-300).log() - (lse_rest - lse)), torch.zeros_like(rest))
            inside = torch.where(held | ~some[:, None], torch.zeros_like(z), (z - lse_rest[:, None]).exp())
            grad = grad + rest[:, None] * (p - inside)
        grad = grad * (s['g_loss'][r].double() * s['scale'])[:, None]
        live = seen.any(1)
        return dict(loss=torch.where(live, loss, torch.zeros_like(loss)),
                    grad=torch.where(live[:, None], grad, torch.zeros_like(grad)))
    surprise = torch.where(p > 0, -logp, torch.zeros_like(p))
    entropy = (p * surprise).sum(1)
    out = dict(lse=lse, entropy=entropy)
    if s['targets'] is not None:
        t = s['targets'][r]
        got = torch.where(t < 0, torch.zeros_like(t, dtype=z.dtype), logp[row, t.clamp_min(0)])
        out['logprobs'] = got
    if s['top']:
        best = torch.sort(logp, 1, descending=True).values[:, :s['top']]
        out['top_logprobs'] = torch.cat([best, best.new_full((n, s['top'] - best.shape[1]), -INF)], 1)
    if s['kind'] == 'train':
        g = torch.where((t < 0) | (got == -INF), torch.zeros_like(got), s['g_logprobs'][r].double())
        picked = torch.zeros_like(z).index_put_((row.expand_as(t), t.clamp_min(0)), g, accumulate=True)
        grad = picked - p * g.sum(1, keepdim=True)
        grad = grad + s['g_entropy'][r].double()[:, None] * p * (surprise - entropy[:, None])
        out['grad'] = grad * s['scale']
    return out
