"""The language-model operators: the cases they are measured on, their plain forms, and the calls a user makes of them.

A re-ranking language model reads the words of a sentence (a row of a table a word), carries a state from word to word and
scores the word that follows with the noise-contrastive dot product of the RNN re-ranker.  Three pairs of operators:

  lookup, lookup_grad   y_t = scale * table[id_t];  dtable_v = scale * sum over the tokens t with id_t = v of dy_t.  An id
                        outside the vocabulary is a row of zeros and has no gradient.
  scan, scan_train      a = sigmoid(f), h_t = a_t h_(t-1) + (1 - a_t) x_t, every sentence of a packed batch from a state
                        of its own, and the gradient of all its inputs.
  score, nce_train      s = <h_t, table[c]> - constant for K candidates a token (-inf for none); the loss
                        weight_t (softplus(-z_0) + sum over k > 0 of softplus(z_k)), z = s - log_noise[c], candidate 0 being
                        the word that follows, with the gradients of the states and of the table.  A token without a
                        following word (c_0 outside the vocabulary) has loss and gradient zero.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
NCE_CONSTANT = 9.0   # the logarithm of the normaliser of the re-ranker's models
SCALE = 0.7


def listed():
    return [
        # one word for each of 64 sentences that are scored word by word (hidden size and vocabulary of the benchmark)
        {'name': 'lookup_step', 'op': 'lookup', 'tokens': 64, 'dim': 128, 'vocab': 31200, 'table': 'f32', 'type': 'f32'},
        # the words of a whole batch of 65 536 sentences, from a 32-bit table into 16-bit activations
        {'name': 'lookup_corpus', 'op': 'lookup', 'tokens': 2031616, 'dim': 128, 'vocab': 31200, 'table': 'f32', 'type': 'bf16'},
        # the table's gradient from a few sentences: most of the table has none
        {'name': 'lookup_grad_sentences', 'op': 'lookup_grad', 'tokens': 1003, 'dim': 100, 'vocab': 30000, 'type': 'f32'},
        # ... from a batch of 16 384 sentences: every fifteenth token is the most frequent word
        {'name': 'lookup_grad_corpus', 'op': 'lookup_grad', 'tokens': 507904, 'dim': 256, 'vocab': 65521, 'type': 'bf16'},
        # serving: one word further in each of 64 sentences
        {'name': 'scan_step', 'op': 'scan', 'tokens': 64, 'seqs': 64, 'dim': 128, 'type': 'f32'},
        # one long document
        {'name': 'scan_document', 'op': 'scan', 'tokens': 65536, 'seqs': 1, 'dim': 1024, 'type': 'bf16'},
        # a training step over 16 384 sentences of about 31 words
        {'name': 'scan_train_sentences', 'op': 'scan_train', 'tokens': 507904, 'seqs': 16384, 'dim': 128, 'type': 'f32'},
        # ... over five documents of unlike lengths, odd sizes
        {'name': 'scan_train_documents', 'op': 'scan_train', 'tokens': 40001, 'seqs': 5, 'dim': 1000, 'type': 'f16'},
        # the scores of a global beam of six candidates in each of 64 sentences
        {'name': 'score_beam', 'op': 'score', 'tokens': 64, 'cands': 6, 'dim': 128, 'vocab': 31200, 'type': 'f32'},
        # ... at every word of 16 384 sentences
        {'name': 'score_corpus', 'op': 'score', 'tokens': 507904, 'cands': 6, 'dim': 128, 'vocab': 31200, 'type': 'bf16'},
        # a training step over a few sentences, twenty noise words a token
        {'name': 'nce_train_sentences', 'op': 'nce_train', 'tokens': 1021, 'cands': 21, 'dim': 100, 'vocab': 30000, 'type': 'f32'},
        # ... over some two thousand sentences, a larger vocabulary
        {'name': 'nce_train_corpus', 'op': 'nce_train', 'tokens': 65536, 'cands': 33, 'dim': 256, 'vocab': 65521, 'type': 'bf16'},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(['lookup', 'lookup_grad', 'scan', 'scan_train', 'score', 'nce_train'])
    c = {'op': op, 'type': rng.choice(['f32', 'bf16', 'f16'])}
    c['dim'] = spread(32, 1100) if op in ('scan', 'scan_train') else spread(32, 520)
    if rng.random() < 0.6:
        c['dim'] = max(32, c['dim'] // 8 * 8)
    if op == 'lookup':
        c['tokens'] = spread(1, 500000)
        c['vocab'] = spread(1000, 130000)
        c['table'] = rng.choice([c['type'], 'f32'])
    elif op == 'lookup_grad':
        c['tokens'] = spread(1, 250000)
        c['vocab'] = spread(1000, 65000)
    elif op in ('scan', 'scan_train'):
        c['tokens'] = spread(1, 40000 if op == 'scan' else 30000)
        c['seqs'] = max(1, min(c['tokens'], spread(1, 40000)))
    else:
        c['vocab'] = spread(1000, 65000)
        c['tokens'] = spread(1, 100000 if op == 'score' else 20000)
        c['cands'] = spread(1, 12) if op == 'score' else spread(2, 33)
    return c


def _words(gen, shape, vocab):
    """words by Zipf's law, the most frequent first; one in 64 is none (-1)"""
    u = torch.rand(shape, generator=gen, device='cuda', dtype=torch.float64)
    ids = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).floor().clamp_(0, vocab - 1).to(torch.int32)
    none = torch.rand(shape, generator=gen, device='cuda') < 1.0 / 64
    return torch.where(none, torch.full_like(ids, -1), ids)


def _sentences(gen, tokens, seqs):
    """offsets of the sentences (some of them empty) and the length of the longest"""
    w = torch.rand(seqs, generator=gen, device='cuda', dtype=torch.float64) + 0.25
    ends = (torch.cumsum(w, 0) / w.sum() * tokens).round().to(torch.int32)
    if tokens == seqs:
        ends = torch.arange(1, seqs + 1, device='cuda', dtype=torch.int32)
    elif seqs > 64:
        ends[31:-1:64] = ends[30:-2:64]
    ends[-1] = tokens
    offsets = torch.cat([torch.zeros(1, device='cuda', dtype=torch.int32), ends])
    return offsets, int((offsets[1:] - offsets[:-1]).max())


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(seed)
    dtype = TYPES[case['type']]

    def normal(*shape, mean=0.0, std=1.0, dtype=dtype):
        return torch.randn(shape, generator=gen, device='cuda').mul_(std).add_(mean).to(dtype)

    op, t, d = case['op'], case['tokens'], case['dim']
    s = {'op': op, 'dtype': dtype}
    if op == 'lookup':
        s['table'] = normal(case['vocab'], d, dtype=TYPES[case['table']])
        s['ids'] = _words(gen, (t,), case['vocab'])
    elif op == 'lookup_grad':
        s['vocab'] = case['vocab']
        s['dy'] = normal(t, d)
        s['ids'] = _words(gen, (t,), case['vocab'])
    elif op in ('scan', 'scan_train'):
        s['offsets'], s['max_len'] = _sentences(gen, t, case['seqs'])
        # the gates and the inputs are the halves of one projection of the words
        s['gate'], s['x'] = normal(t, 2 * d).split(d, dim=1)
        s['gate'] += 2.0
        s['state'] = normal(case['seqs'], d, std=0.5, dtype=torch.float32)
        if op == 'scan_train':
            s['dh'] = normal(t, d)
            s['dlast'] = normal(case['seqs'], d, dtype=torch.float32)
    else:
        k, v = case['cands'], case['vocab']
        s['h'] = normal(t, d, std=0.5)
        s['table'] = normal(v, d, std=2.0 / math.sqrt(d))
        s['cands'] = _words(gen, (t, k), v)
        if op == 'nce_train':
            rank = torch.arange(1, v + 1, device='cuda', dtype=torch.float64)
            p = torch.log1p(1.0 / rank) / math.log(v + 1.0)
            s['log_noise'] = (torch.log(p * (k - 1)) - 5.0).float()
            s['weight'] = torch.full((t,), 1.0 / t, device='cuda')
    return s


# ---- the plain forms -------------------------------------------------------------------------------------------------
def _inside(ids, vocab):
    ok = (ids >= 0) & (ids < vocab)
    return ok, torch.where(ok, ids, torch.zeros_like(ids)).long()


def _lookup(table, ids, dtype):
    ok, row = _inside(ids, table.shape[0])
    return (table[row].float() * SCALE * ok[:, None]).to(dtype)


def _lookup_grad(dy, ids, vocab):
    ok, row = _inside(ids, vocab)
    g = torch.zeros(vocab + 1, dy.shape[1], device=dy.device)
    g.index_add_(0, torch.where(ok, row, torch.full_like(row, vocab)), dy.float() * SCALE)
    return g[:vocab]


def _doubling(a, b, longest):
    """y_t = a_t y_(t-1) + b_t along dim 0: after the step of distance d every pair (a, b) stands for the 2 d rows up to its own"""
    d = 1
    while d < longest:
        b = torch.cat([b[:d], a[d:] * b[:-d] + b[d:]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _ends(offsets):
    full = offsets[1:] > offsets[:-1]
    return full, offsets[:-1][full].long(), offsets[1:][full].long() - 1


def _scan(gate, x, offsets, state, longest):
    full, first, last = _ends(offsets)
    a, keep = torch.sigmoid(gate.float()), torch.sigmoid(-gate.float())
    b = keep * x.float()
    b[first] += a[first] * state[full]
    a[first] = 0.0
    h = _doubling(a, b, longest)
    end = state.clone()
    end[full] = h[last]
    return h, end


def _scan_train(gate, x, offsets, state, longest, dh, dlast):
    full, first, last = _ends(offsets)
    h, end = _scan(gate, x, offsets, state, longest)
    a, keep = torch.sigmoid(gate.float()), torch.sigmoid(-gate.float())
    up = dh.float().clone()
    up[last] += dlast[full]
    after = torch.cat([a[1:], torch.zeros_like(a[:1])])
    after[last] = 0.0
    delta = _doubling(after.flip(0), up.flip(0), longest).flip(0)
    before = torch.cat([torch.zeros_like(h[:1]), h[:-1]])
    before[first] = state[full]
    dgate = delta * (before - x.float()) * a * keep
    dstate = dlast.clone()
    dstate[full] = a[first] * delta[first]
    return h.to(x.dtype), end, dgate.to(x.dtype), (delta * keep).to(x.dtype), dstate


def _score(h, table, cands):
    ok, row = _inside(cands, table.shape[0])
    s = (table[row].float() * h.float()[:, None, :]).sum(-1) - NCE_CONSTANT
    return torch.where(ok, s, torch.full_like(s, -math.inf))


def _softplus(z):
    return torch.clamp(z, min=0.0) + torch.log1p(torch.exp(-z.abs()))


def _nce_train(h, table, cands, log_noise, weight):
    ok, row = _inside(cands, table.shape[0])
    ok = ok & ok[:, :1]
    rows, hf = table[row].float(), h.float()
    z = (rows * hf[:, None, :]).sum(-1) - NCE_CONSTANT - log_noise[row]
    sign = torch.ones_like(z)
    sign[:, 0] = -1.0
    loss = (_softplus(sign * z) * ok).sum(1) * weight
    g = sign * torch.sigmoid(sign * z) * ok * weight[:, None]
    dh = (g[:, :, None] * rows).sum(1).to(h.dtype)
    dtable = torch.zeros(table.shape, device=h.device)
    dtable.index_add_(0, row.reshape(-1), (g[:, :, None] * hf[:, None, :]).reshape(-1, h.shape[1]))
    return loss, dh, dtable


def run(state):
    s = state
    op = s['op']
    if own:
        from jumanpp_amd import lm
        if op == 'lookup':
            return lm.embed(s['table'], s['ids'], scale=SCALE, dtype=s['dtype'])
        if op == 'lookup_grad':
            return lm.embed_grad(s['dy'], s['ids'], s['vocab'], scale=SCALE)
        if op == 'scan':
            return lm.scan(s['gate'], s['x'], s['offsets'], s['state'], max_len=s['max_len'])
        if op == 'scan_train':
            h, last, saved = lm.scan(s['gate'], s['x'], s['offsets'], s['state'], max_len=s['max_len'], save=True)
            return (h, last) + lm.scan_grad(s['gate'], s['x'], s['dh'], saved, s['offsets'], s['state'], s['dlast'],
                                            max_len=s['max_len'])
        if op == 'score':
            return lm.nce_score(s['h'], s['table'], s['cands'], NCE_CONSTANT)
        return lm.nce_loss(s['h'], s['table'], s['cands'], s['log_noise'], NCE_CONSTANT, s['weight'])
    if op == 'lookup':
        return _lookup(s['table'], s['ids'], s['dtype'])
    if op == 'lookup_grad':
        return _lookup_grad(s['dy'], s['ids'], s['vocab'])
    if op == 'scan':
        h, end = _scan(s['gate'], s['x'], s['offsets'], s['state'], s['max_len'])
        return h.to(s['dtype']), end
    if op == 'scan_train':
        return _scan_train(s['gate'], s['x'], s['offsets'], s['state'], s['max_len'], s['dh'], s['dlast'])
    if op == 'score':
        return _score(s['h'], s['table'], s['cands'])
    return _nce_train(s['h'], s['table'], s['cands'], s['log_noise'], s['weight'])


def work(case):
    op, t, d, e = case['op'], case['tokens'], case['dim'], BYTES[case['type']]
    if op == 'lookup':
        rows = min(t, case['vocab'])
        return {'bytes': 4 * t + rows * d * BYTES[case['table']] + t * d * e, 'flops': t * d}
    if op == 'lookup_grad':
        return {'bytes': 4 * t + t * d * e + case['vocab'] * d * 4, 'flops': 2 * t * d}
    if op in ('scan', 'scan_train'):
        n = case['seqs']
        ahead = 3 * t * d * e + 2 * n * d * 4 + 4 * (n + 1)   # gate, x -> h; the states in and out
        if op == 'scan':
            return {'bytes': ahead, 'flops': 10 * t * d}
        # the gradient: gate, x, dh -> dgate, dx; the states' gradients
        return {'bytes': ahead + 5 * t * d * e + 3 * n * d * 4 + 4 * (n + 1), 'flops': 32 * t * d}
    k, v = case['cands'], case['vocab']
    rows = min(t * k, v)
    if op == 'score':
        return {'bytes': 8 * t * k + t * d * e + rows * d * e, 'flops': 2 * t * k * d}
    return {'bytes': 4 * t * k + 8 * t + 2 * t * d * e + rows * (d * e + 4) + v * d * 4, 'flops': 6 * t * k * d}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _by_length(offsets):
    """the sentences from the longest to the shortest: start, length, and how many are longer than a position"""
    start = offsets[:-1].long()
    length = offsets[1:].long() - start
    order = torch.argsort(length, descending=True, stable=True)
    lengths = length[order].cpu()
    most = int(lengths[0]) if len(lengths) else 0
    alive = torch.bincount(lengths, minlength=most + 1).flip(0).cumsum(0).flip(0)[1:].tolist()
    return start, length, order, alive


def _exact_scan(s):
    x, z = s['x'].double(), s['gate'].double()
    a = 1.0 / (1.0 + torch.exp(-z))
    start, length, order, alive = _by_length(s['offsets'])
    carried = s['state'].double()[order]
    begin = start[order]
    before, h = torch.empty_like(x), torch.empty_like(x)
    for p, n in enumerate(alive):
        row = begin[:n] + p
        prev = carried[:n]
        now = x[row] + a[row] * (prev - x[row])
        before[row], h[row] = prev, now
        carried[:n] = now
    last = torch.empty_like(carried)
    last[order] = carried
    if s['op'] == 'scan':
        return h, last
    dh, slope = s['dh'].double(), torch.exp(-z) * a * a
    dx, dz = torch.empty_like(x), torch.empty_like(x)
    back = s['dlast'].double()[order]
    end = begin + length[order] - 1
    for p, n in enumerate(alive):
        row = end[:n] - p
        up = dh[row] + back[:n]
        dx[row] = up * (1.0 - a[row])
        dz[row] = up * (before[row] - x[row]) * slope[row]
        back[:n] = up * a[row]
    dstate = torch.empty_like(back)
    dstate[order] = back
    return h, last, dz, dx, dstate


def exact(case, seed):
    s = prepare(case, seed)
    op = s['op']
    if op in ('scan', 'scan_train'):
        return _exact_scan(s)
    if op == 'lookup':
        table = torch.cat([s['table'].double(), torch.zeros(1, case['dim'], device='cuda', dtype=torch.float64)])
        ids = s['ids'].long()
        return SCALE * table[torch.where((ids < 0) | (ids >= case['vocab']), case['vocab'], ids)]
    if op == 'lookup_grad':
        keep = (s['ids'] >= 0) & (s['ids'] < s['vocab'])
        g = torch.zeros(s['vocab'], case['dim'], device='cuda', dtype=torch.float64)
        return g.index_add_(0, s['ids'][keep].long(), s['dy'][keep].double()) * SCALE
    table, v = s['table'].double(), case['vocab']
    outs, dtable = [], torch.zeros(v, case['dim'], device='cuda', dtype=torch.float64)
    for part in torch.arange(case['tokens'], device='cuda').split(4096):
        c, h = s['cands'][part].long(), s['h'][part].double()
        bad = (c < 0) | (c >= v)
        rows = table[c.masked_fill(bad, 0)]
        dot = torch.matmul(rows, h[:, :, None])[:, :, 0] - NCE_CONSTANT
        if op == 'score':
            outs.append((dot.masked_fill(bad, -math.inf),))
            continue
        bad = bad | bad[:, :1]
        z = dot - s['log_noise'].double()[c.masked_fill(bad, 0)]
        z[:, 0] = -z[:, 0]
        w = s['weight'][part].double()
        loss = torch.logaddexp(z, torch.zeros_like(z)).masked_fill(bad, 0.0).sum(1) * w
        g = (1.0 / (1.0 + torch.exp(-z))).masked_fill(bad, 0.0) * w[:, None]
        g[:, 0] = -g[:, 0]
        outs.append((loss, torch.matmul(g[:, None, :], rows)[:, 0, :]))
        dtable.index_add_(0, c.masked_fill(bad, 0).reshape(-1), (g[:, :, None] * h[:, None, :]).reshape(-1, case['dim']))
    if op == 'score':
        return torch.cat([o[0] for o in outs])
    return torch.cat([o[0] for o in outs]), torch.cat([o[1] for o in outs]), dtable
