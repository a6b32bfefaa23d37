"""Checks of the language-model operators against tests/lm_reference.py.  One list for both sides: tests/test_lm_cpu.py runs
it on the emulator build of the kernels, tests/test_lm_gpu.py in one child process on the GPU (torch has to load its HIP
runtime before the library does, which the other GPU tests' process cannot promise):

    python -u tests/lm_checks.py [RESULTS.json]

With a file, every check's result is in it and the status is that of the program; without one, the status says whether all passed.
"""
import json
import os
import sys
import threading
import traceback

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, 'tests')]

import lm_reference as R  # noqa: E402
from jumanpp_amd import lm  # noqa: E402
from jumanpp_amd.native import JppGpuError  # noqa: E402

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
CHECKS = []   # (name, function(E), where): 'both', 'gpu' or 'cpu'


class Env:
    def __init__(self, device, lib_path):
        self.device, self.lib_path, self.gpu = device, lib_path, device != 'cpu'
        self.kw = {} if lib_path is None else {'lib_path': lib_path}

    def to(self, t):
        return None if t is None else t.to(self.device)


def check(where='both', third=False, **grid):
    """the function once for every combination of the named values; third: on the emulator every third one"""
    def add(fn):
        combos = [{}]
        for key, values in grid.items():
            combos = [dict(c, **{key: v}) for c in combos for v in values]
        for c in combos:
            name = fn.__name__ + ''.join('-%s' % str(v).replace('torch.', '').replace(' ', '') for v in c.values())
            CHECKS.append((name, lambda E, fn=fn, c=c: fn(E, **c), 'gpu' if third and len(CHECKS) % 3 else where))
        return fn
    return add


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=F32, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g) * std + mean).to(dtype)


def words(g, vocab, *shape, dtype=torch.int32, none=True):
    """small ids often, some that name no word"""
    u = torch.rand(*shape, generator=g, dtype=torch.float64)
    ids = (torch.exp(u * torch.log(torch.tensor(vocab + 1.0, dtype=torch.float64))) - 1).floor().clamp(0, max(vocab - 1, 0)).to(torch.int64)
    if none:
        pick = torch.rand(*shape, generator=g)
        ids[pick < 0.05] = -1
        ids[(pick >= 0.05) & (pick < 0.08)] = vocab
        if dtype == torch.int64:
            ids[(pick >= 0.08) & (pick < 0.1)] = 2 ** 40
            ids[(pick >= 0.1) & (pick < 0.12)] = -2 ** 40 + 1
        else:
            ids[(pick >= 0.08) & (pick < 0.1)] = 2 ** 31 - 1
            ids[(pick >= 0.1) & (pick < 0.12)] = -2 ** 31
    if vocab == 0:
        ids[:] = 0
    return ids.to(dtype)


def near(what, got, want):
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (what, got.shape, value.shape)
    same = (got == value) | (got.isnan() & value.isnan())
    off = (got - value).abs()
    bad = ~same & ~(off <= bound)
    if bad.any():
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError('%s: %d of %d values outside their bounds; at %d: got %r, want %r +- %r' % (
            what, int(bad.sum()), bad.numel(), i, got.reshape(-1)[i].item(), value.reshape(-1)[i].item(), bound.reshape(-1)[i].item()))


def equal(what, a, b):
    a, b = a.detach().cpu(), b.detach().cpu()
    assert a.dtype == b.dtype and a.shape == b.shape, what
    same = torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
    assert same, '%s: not the same bits' % what


def layout(E, t, kind):
    """the same rows elsewhere: 'plain', 'wide' (rows with a gap), 'half' (columns of a wider matrix, at an odd element)"""
    if kind == 'plain' or t is None:
        return E.to(t)
    n, d = t.shape
    big = torch.full((n + 1, d + 9), float('nan'), dtype=t.dtype)
    at = 0 if kind == 'wide' else 3
    big[:n, at:at + d] = t
    return E.to(big)[:n, at:at + d]


# ---- lookup ------------------------------------------------------------------------------------
@check(third=True, types=[(F32, F32), (BF16, BF16), (F16, F16), (F32, BF16), (F32, F16)], dim=[1, 3, 8, 100, 257])
def embed(E, types, dim):
    g = rng(dim)
    for n, vocab, idt, kind, scale in ((0, 5, torch.int32, 'plain', 1.0), (1, 1, torch.int64, 'plain', 0.5), (70, 40, torch.int64, 'half', -1.7),
                                       (130, 1, torch.int32, 'wide', 3.0), (33, 0, torch.int32, 'plain', 1.0), (301, 900, torch.int32, 'plain', 0.7)):
        table = normal(g, vocab, dim, dtype=types[0])
        ids = words(g, vocab, n, dtype=idt)
        used = torch.zeros(vocab, dtype=torch.bool)
        used[ids[(ids >= 0) & (ids < vocab)].long()] = True
        table[~used] = float('nan')   # nobody reads these
        got = lm.embed(layout(E, table, kind), E.to(ids), scale, dtype=types[1], **E.kw)
        assert got.dtype == types[1]
        near('n=%d vocab=%d' % (n, vocab), got, R.embed(table, ids, scale, types[1]))


def raw_grad(E, dy, ids, vocab, scale, stride=None):
    """embed_grad into a matrix that held NaN, with any stride; the columns behind the rows come back too"""
    lib = lm._lib(E.lib_path)
    n, dim = dy.shape
    grad = torch.full((vocab, stride or dim), float('nan'), device=E.device)
    ws, wp, wn = lm._workspace(lib, 'jppgpu_lm_embed_grad_workspace', (n, vocab, dim), dy)
    if ws is not None:
        ws.fill_(255)
    dev, stream = lm._where(E.lib_path, dy, ids)
    lm._check(lib, lib.jppgpu_lm_embed_grad(lm._rows(dy, 'dy'), lm._ids(ids), n, vocab, dim, scale, lm._rows(grad[:, :dim], 'grad'),
                                            wp, wn, dev, stream))
    return grad


GRAD_CASES = ((0, 7), (1, 1), (2, 300), (64, 5), (65, 70000), (1003, 300), (1100, 2), (5000, 3), (4097, 257), (6500, 1 << 17))


@check(case=GRAD_CASES, dim=[1, 5, 64, 100, 130])
def embed_grad(E, case, dim):
    n, vocab = case
    if not E.gpu and n * dim > 150000:
        dim = dim // 16 + 1
    if vocab * dim > 3000000:
        vocab = 3000000 // dim
    dtype = (F32, BF16, F16)[(n + dim) % 3]
    g = rng(n * 7 + dim)
    dy = normal(g, n, dim, dtype=dtype)
    ids = words(g, vocab, n, dtype=(torch.int32, torch.int64)[dim % 2])
    want = R.embed_grad(dy, ids, vocab, 1.25)
    stride = dim + (dim % 3)
    dyd, idd = layout(E, dy, ('plain', 'wide', 'half')[(n + dim) % 3]), E.to(ids)
    got = raw_grad(E, dyd, idd, vocab, 1.25, stride)
    near('gradient', got[:, :dim], want)
    assert got[:, dim:].isnan().all()
    equal('again', raw_grad(E, dyd, idd, vocab, 1.25, stride)[:, :dim], got[:, :dim])
    equal('lm.embed_grad', lm.embed_grad(dyd, idd, vocab, 1.25, **E.kw), got[:, :dim])


@check(n=[9, 700, 5003], kind=['one', 'none', 'two', 'sorted', 'last'])
def embed_grad_words(E, n, kind):
    """one word for all entries, no word at all, runs that end on tile borders, the last row of the table"""
    vocab, dim = 50, 9
    ids = {'one': torch.full((n,), 7), 'none': torch.full((n,), -1), 'two': torch.arange(n) % 2 * 49,
           'sorted': torch.arange(n) // 8 % vocab, 'last': torch.full((n,), 49)}[kind].to(torch.int32)
    dy = normal(rng(n), n, dim)
    if kind == 'none':
        dy[:] = float('nan')
    near(kind, raw_grad(E, E.to(dy), E.to(ids), vocab, 1.0), R.embed_grad(dy, ids, vocab, 1.0))


def grad_many(E, n, vocab, dim):
    g = rng(n)
    dy, ids = normal(g, n, dim), words(g, vocab, n)
    got = raw_grad(E, E.to(dy), E.to(ids), vocab, 0.75)
    near('gradient', got, R.embed_grad(dy, ids, vocab, 0.75))
    equal('again', raw_grad(E, E.to(dy), E.to(ids), vocab, 0.75), got)


@check(case=[(32768, 1000), (32769, 1000), (70003, 70000)])
def embed_grad_many(E, case):
    """either side of where a thread of the sort takes more entries, and where the tiles' counts get a kernel of their own"""
    grad_many(E, *case, 3 if case[0] % 2 else 5)


@check('gpu', case=[(300007, 200), (1048576, 60), (1048577, 60), (2000003, 1 << 17)])
def embed_grad_very_many(E, case):
    grad_many(E, *case, 6)


@check()
def nce_many(E):
    one_nce(E, 3001, 11, 500, 5, F32)


@check()
def embed_grad_padding_is_not_read_into_sums(E):
    dy = normal(rng(5), 200, 12)
    ids = torch.arange(200, dtype=torch.int32) % 11
    ids[::3] = -1
    dy[::3] = float('nan')
    near('gradient', raw_grad(E, E.to(dy), E.to(ids), 11, 1.0), R.embed_grad(dy, ids, 11, 1.0))


# ---- the recurrence ------------------------------------------------------------------------------
def raw_scan(E, gate, x, offsets, state, max_len, fill):
    """scan into matrices that held `fill`"""
    lib = lm._lib(E.lib_path)
    rows, dim = x.shape
    n = offsets.shape[0] - 1
    h = E.to(fill.to(x.dtype))
    last = torch.full((n, dim), float('nan'), device=E.device)
    saved = torch.full((lib.jppgpu_lm_scan_saved(rows), dim), float('nan'), device=E.device)
    ws, wp, wn = lm._workspace(lib, 'jppgpu_lm_scan_workspace', (rows, n, dim, max_len), x)
    if ws is not None:
        ws.fill_(255)
    dev, stream = lm._where(E.lib_path, x)
    sv = lm._rows(state, 'state') if state is not None else None
    lm._check(lib, lib.jppgpu_lm_scan(lm._rows(gate, 'gate'), lm._rows(x, 'x'), offsets.data_ptr(), n, rows, dim, max_len, sv,
                                      lm._rows(h, 'h'), lm._rows(last, 'last'), saved.data_ptr(), wp, wn, dev, stream))
    return h, last, saved


def raw_scan_grad(E, gate, x, offsets, state, max_len, saved, dh, dlast, fill):
    lib = lm._lib(E.lib_path)
    rows, dim = x.shape
    n = offsets.shape[0] - 1
    dgate, dx = (E.to(fill.to(x.dtype).clone()) for _ in range(2))
    dstate = torch.full((n, dim), float('nan'), device=E.device)
    ws, wp, wn = lm._workspace(lib, 'jppgpu_lm_scan_workspace', (rows, n, dim, max_len), x)
    if ws is not None:
        ws.fill_(255)
    dev, stream = lm._where(E.lib_path, x)
    sv = lm._rows(state, 'state') if state is not None else None
    lv = lm._rows(dlast, 'dlast') if dlast is not None else None
    lm._check(lib, lib.jppgpu_lm_scan_grad(lm._rows(gate, 'gate'), lm._rows(x, 'x'), offsets.data_ptr(), n, rows, dim, max_len, sv,
                                           saved.data_ptr(), lm._rows(dh, 'dh'), lv, lm._rows(dgate, 'dgate'), lm._rows(dx, 'dx'),
                                           lm._rows(dstate, 'dstate'), wp, wn, dev, stream))
    return dgate, dx, dstate


def batch(lengths, front=0, back=0):
    offsets = torch.tensor([front] + lengths, dtype=torch.int64).cumsum(0).to(torch.int32)
    return offsets, int(offsets[-1]) + back


SCAN_CASES = (([1], 0, 0), ([1, 1, 1, 1, 1], 0, 0), ([0, 1, 0], 0, 3), ([8], 5, 0), ([9, 7, 0, 33, 0, 0, 2], 3, 6), ([255, 0, 17], 0, 1),
              ([300], 0, 0), ([0, 0, 257, 1, 40, 0], 2, 40), ([70, 513, 0, 31, 32, 33, 0], 0, 0), ([1000], 37, 70))


def scan_inputs(case, dim, dtype, seed):
    lengths, front, back = case
    offsets, rows = batch(lengths, front, back)
    g = rng(seed)
    n = len(lengths)
    gate, x, dh = normal(g, rows, dim, dtype=dtype, mean=1.5, std=2.0), normal(g, rows, dim, dtype=dtype), normal(g, rows, dim, dtype=dtype)
    # some gates at the ends of their range
    pick = torch.rand(rows, dim, generator=g)
    for i, v in enumerate((float('inf'), -float('inf'), 60.0, -60.0, 120.0, 0.0)):
        gate[(pick > i * 0.01) & (pick <= i * 0.01 + 0.01)] = v
    return offsets, rows, gate, x, dh, normal(g, n, dim), normal(g, n, dim), normal(g, rows, dim)


@check(third=True, dtype=[F32, BF16, F16], case=SCAN_CASES, dim=[1, 64, 100, 201])
def scan(E, case, dim, dtype):
    offsets, rows, gate, x, dh, state, dlast, fill = scan_inputs(case, dim, dtype, dim + len(case[0]))
    odd = (dim + len(case[0])) % 2 == 1
    if odd:
        state = dlast = None
    kinds = ('half', 'wide') if odd else ('plain', 'half')
    gd, xd, dhd = layout(E, gate, kinds[0]), layout(E, x, kinds[1]), layout(E, dh, kinds[0])
    sd, ld, od = E.to(state), E.to(dlast), E.to(offsets)
    fill = fill.to(dtype).float()
    want_h, want_last, _ = R.scan(gate, x, offsets, state, dtype, fill)
    want = R.scan_grad(gate, x, offsets, state, dh, dlast, dtype, fill)
    for max_len in (0, max(case[0])):
        h, last, saved = raw_scan(E, gd, xd, od, sd, max_len, fill)
        near('h, max_len=%d' % max_len, h, want_h)
        near('last', last, want_last)
        got = raw_scan_grad(E, gd, xd, od, sd, max_len, saved, dhd, ld, fill)
        for what, a, b in zip(('dgate', 'dx', 'dstate'), got, want):
            near('%s, max_len=%d' % (what, max_len), a, b)
        h2, last2, saved2 = lm.scan(gd, xd, od, sd, max_len=max_len, save=True, **E.kw)
        b, e = int(offsets[0]), int(offsets[-1])
        equal('h again', h2[b:e], h[b:e])
        equal('last again', last2, last)
        again = lm.scan_grad(gd, xd, dhd, saved2, od, sd, ld, max_len=max_len, **E.kw)
        for what, a, c in zip(('dgate', 'dx'), again, got):
            equal(what + ' again', a[b:e], c[b:e])
        equal('dstate again', again[2], got[2])
        plain = lm.scan(gd, xd, od, sd, max_len=max_len, **E.kw)
        equal('h without saving', plain[0][b:e], h[b:e])


@check(rows=[1, 40, 700])
def scan_one_sentence_without_offsets(E, rows):
    g = rng(rows)
    gate, x = normal(g, rows, 20), normal(g, rows, 20)
    h, last = lm.scan(E.to(gate), E.to(x), **E.kw)
    want_h, want_last, _ = R.scan(gate, x, [0, rows], None, F32, torch.zeros(rows, 20))
    near('h', h, want_h)
    near('last', last, want_last)


@check(long=[False, True], dtype=[F32, F16])
def scan_nan_stays_in_its_sentence(E, long, dtype):
    lengths = [300, 40, 280, 33] if long else [30, 4, 9, 33]
    offsets, rows = batch(lengths)
    g = rng(3)
    gate, x, dh = normal(g, rows, 70, dtype=dtype), normal(g, rows, 70, dtype=dtype), normal(g, rows, 70, dtype=dtype)
    clean = [t.clone() for t in (gate, x, dh)]
    gate[3, 5], x[7, 6], dh[int(offsets[3]) - 1, 7], x[int(offsets[2]) + 1, 8] = (float('nan'),) * 4
    od = E.to(offsets)
    outs = []
    for a, b, c in ((gate, x, dh), clean):
        h, last, saved = lm.scan(E.to(a), E.to(b), od, save=True, **E.kw)
        outs.append((h, last) + lm.scan_grad(E.to(a), E.to(b), E.to(c), saved, od, **E.kw))
    for bad, good, per_row in zip(outs[0], outs[1], (True, False, True, True, False)):
        for i in range(len(lengths)):
            s = slice(int(offsets[i]), int(offsets[i + 1])) if per_row else slice(i, i + 1)
            m = torch.ones(70, dtype=torch.bool)
            m[{0: [5, 6], 1: [], 2: [7, 8], 3: []}[i]] = False
            equal('sentence %d' % i, bad[s].cpu()[:, m], good[s].cpu()[:, m])


@check(long=[False, True])
def scan_step_by_step_is_scan(E, long):
    """serving: the states handed from call to call"""
    n, steps, dim = 5, 12, 33
    g = rng(11)
    gate, x = normal(g, n, steps, dim, dtype=BF16), normal(g, n, steps, dim, dtype=BF16)
    state = normal(g, n, dim)
    off = torch.arange(n + 1, dtype=torch.int32)
    s = E.to(state)
    outs = []
    for t in range(steps):
        h, s = lm.scan(E.to(gate[:, t].contiguous()), E.to(x[:, t].contiguous()), E.to(off), s, max_len=0 if long else 1, **E.kw)
        outs.append(h)
    whole, last = lm.scan(E.to(gate.reshape(n * steps, dim)), E.to(x.reshape(n * steps, dim)), E.to(off * steps), E.to(state), **E.kw)
    equal('h', torch.stack(outs, 1).reshape(n * steps, dim), whole)
    equal('last', s, last)


@check('cpu', offsets=[[0, 30, 10, 40], [5, -3, 60, 41], [40, 0], [0, 1000], [-7, 20], [2 ** 31 - 1, 3, 40], [0, 400, 300, 900, 100]])
def scan_bad_offsets_stay_inside(E, offsets):
    """offsets that fall or leave the batch: any values, but only in the outputs' own rows (the emulator's heap is checked by
    guard rows around every output)"""
    assert not E.gpu, 'host memory: for the emulator alone'
    rows, dim = (700 if max(offsets) > 200 and max(offsets) < 2000 else 41), 10
    g = rng(1)
    gate, x, dh, state = normal(g, rows, dim), normal(g, rows, dim), normal(g, rows, dim), normal(g, len(offsets) - 1, dim)
    off = torch.tensor(offsets, dtype=torch.int32)
    lib = lm._lib(E.lib_path)
    n = len(offsets) - 1
    guard = 12

    def guarded(r):
        big = torch.full((r + 2 * guard, dim), 7.0)
        return big, big[guard:guard + r]

    for max_len in (0, 5):
        (hb, h), (lb, last), (sb, saved), (gb, dgate), (xb, dx), (tb, dstate) = (
            guarded(r) for r in (rows, n, lib.jppgpu_lm_scan_saved(rows), rows, rows, n))
        saved.fill_(0.5)
        ws, wp, wn = lm._workspace(lib, 'jppgpu_lm_scan_workspace', (rows, n, dim, max_len), x)
        M = lambda t: lm._rows(t, 't')  # noqa: E731
        lm._check(lib, lib.jppgpu_lm_scan(M(gate), M(x), off.data_ptr(), n, rows, dim, max_len, M(state), M(h), M(last), saved.data_ptr(),
                                          wp, wn, 0, None))
        lm._check(lib, lib.jppgpu_lm_scan_grad(M(gate), M(x), off.data_ptr(), n, rows, dim, max_len, M(state), saved.data_ptr(), M(dh), None,
                                               M(dgate), M(dx), M(dstate), wp, wn, 0, None))
        for big in (hb, lb, sb, gb, xb, tb):
            assert (big[:guard] == 7.0).all() and (big[-guard:] == 7.0).all()


# ---- noise-contrastive score and loss ------------------------------------------------------------
NCE_CASES = ((0, 3, 9), (1, 1, 1), (5, 2, 3), (33, 6, 40), (9, 21, 300), (7, 70, 65), (3, 129, 11))


def nce_inputs(n, k, vocab, dim, dtype, seed):
    g = rng(seed)
    h, table = normal(g, n, dim, dtype=dtype), normal(g, vocab, dim, dtype=dtype, std=dim ** -0.5)
    ids = words(g, vocab, n, k, dtype=(torch.int32, torch.int64)[seed % 2])
    used = torch.zeros(vocab, dtype=torch.bool)
    used[ids[(ids >= 0) & (ids < vocab)].long().reshape(-1)] = True
    return h, table, ids, used, normal(g, vocab, mean=-9.0, std=2.0), torch.rand(n, generator=g)


@check(third=True, dtype=[F32, BF16, F16], dim=[1, 3, 4, 7, 64, 100, 130, 256, 300, 520])
def nce(E, dim, dtype):
    for n, k, vocab in NCE_CASES:
        one_nce(E, n, k, vocab, dim, dtype)


@check(dim=[1025, 1030, 2048, 2103], dtype=[F32, BF16])
def nce_long_rows(E, dim, dtype):
    one_nce(E, 3, 5, 9, dim, dtype)
    one_nce(E, 2, 70, 9, dim, dtype)


def one_nce(E, n, k, vocab, dim, dtype):
    seed = dim + n * 3 + k
    h, table, ids, used, log_noise, weight = nce_inputs(n, k, vocab, dim, dtype, seed)
    weight = (None, weight)[seed % 2]
    table[~used] = float('nan')
    kinds = ('plain', 'half', 'wide')
    hd, td = layout(E, h, kinds[seed % 3]), layout(E, table, kinds[(seed // 3) % 3])
    what = 'n=%d cands=%d vocab=%d ' % (n, k, vocab)
    near(what + 'score', lm.nce_score(hd, td, E.to(ids), 0.75, **E.kw), R.nce_score(h, table, ids, 0.75)[:2])
    # rows without a following word hold anything
    dead = ~((ids[:, 0] >= 0) & (ids[:, 0] < vocab))
    h[dead] = float('nan')
    hd = layout(E, h, kinds[seed % 3])
    want = R.nce_loss(h, table, ids, log_noise, 0.75, weight, dtype)
    got = lm.nce_loss(hd, td, E.to(ids), E.to(log_noise), 0.75, E.to(weight), **E.kw)
    for name, a, b in zip(('loss', 'dh', 'dtable'), got, want):
        near(what + name, a, b)
    again = lm.nce_loss(hd, td, E.to(ids), E.to(log_noise), 0.75, E.to(weight), **E.kw)
    for name, a, b in zip(('loss', 'dh', 'dtable'), again, got):
        equal(what + name + ' again', a, b)
    equal(what + 'loss alone', lm.nce_loss(hd, td, E.to(ids), E.to(log_noise), 0.75, E.to(weight), grads=False, **E.kw), got[0])


@check()
def nce_one_gradient_at_a_time(E):
    h, table, ids, _, log_noise, weight = nce_inputs(20, 7, 30, 36, F32, 4)
    h, table, ids, log_noise, weight = (E.to(t) for t in (h, table, ids, log_noise, weight))
    loss, dh, dtable = lm.nce_loss(h, table, ids, log_noise, 1.0, weight, **E.kw)
    lib = lm._lib(E.lib_path)
    dev, stream = lm._where(E.lib_path, h)
    for pick in ('dh', 'dtable'):
        a, b, c = torch.empty_like(loss), torch.empty_like(dh), torch.empty_like(dtable)
        ws, wp, wn = lm._workspace(lib, 'jppgpu_lm_nce_loss_workspace', (20, 7, 30, 36), h)
        lm._check(lib, lib.jppgpu_lm_nce_loss(lm._rows(h, 'h'), lm._rows(table, 't'), 30, 36, lm._ids(ids), 20, 7, log_noise.data_ptr(), 1.0,
                                              weight.data_ptr(), a.data_ptr(), lm._rows(b, 'dh') if pick == 'dh' else None,
                                              lm._rows(c, 'dt') if pick == 'dtable' else None, wp, wn, dev, stream))
        equal('loss', a, loss)
        equal(pick, b if pick == 'dh' else c, dh if pick == 'dh' else dtable)


@check(z=[0.0, 1e-3, 5.0, 20.0, 100.0, -30.0, -150.0, 1e30, -1e30])
def nce_far_scores(E, z):
    """softplus and sigmoid over their whole range, each to its own relative precision"""
    h, table = torch.tensor([[z], [z]]), torch.tensor([[1.0], [-1.0]])
    ids = torch.tensor([[0, 1], [1, 0]], dtype=torch.int32)
    ln = torch.zeros(2)
    got = lm.nce_loss(E.to(h), E.to(table), E.to(ids), E.to(ln), 0.0, **E.kw)
    for name, a, b in zip(('loss', 'dh', 'dtable'), got, R.nce_loss(h, table, ids, ln, 0.0, None, F32)):
        near(name, a, b)


@check(dtype=[BF16, F16], dim=[8, 40, 300])
def nce_score_subnormal_rows(E, dim, dtype):
    """the smallest numbers of a 16-bit table count in full: products of theirs with large states"""
    g = rng(dim)
    small = torch.finfo(dtype).smallest_normal
    step = small * torch.finfo(dtype).eps
    table = (torch.randint(-120, 121, (6, dim), generator=g).double() * step).to(dtype)
    assert ((table.double().abs() < small) & (table != 0)).any()
    h = normal(g, 5, dim, dtype=torch.float64, std=100.0 if dtype == F16 else 2.0 ** 110).to(dtype)
    ids = words(g, 6, 5, 7, none=False)
    near('score', lm.nce_score(E.to(h), E.to(table), E.to(ids), 0.0, **E.kw), R.nce_score(h, table, ids, 0.0)[:2])


@check(dtype=[F32, BF16, F16])
def nce_score_not_finite(E, dtype):
    """an infinity or a NaN of a row is in the scores of that row and of no other"""
    inf, nan = float('inf'), float('nan')
    h = torch.ones(2, 32)
    h[1, 5] = 0
    table = torch.ones(5, 32)
    table[1, 5], table[2, 6], table[3, 7], table[3, 8] = inf, -inf, inf, -inf
    table[4, 31] = nan
    ids = torch.tensor([[0, 1, 2, 3, 4, 9], [4, 3, 2, 1, 0, -1]], dtype=torch.int32)
    got = lm.nce_score(E.to(h.to(dtype)), E.to(table.to(dtype)), E.to(ids), 2.0, **E.kw).cpu()
    want = torch.tensor([[30, inf, -inf, nan, nan, -inf], [nan, nan, -inf, nan, 29, -inf]])
    assert torch.equal(got.isnan(), want.isnan()), got
    equal('scores', got[~got.isnan()], want[~want.isnan()])


@check(dtype=[F32, BF16], dim=[4, 1500])
def nce_noise_without_a_logarithm(E, dim, dtype):
    """noise probabilities of zero and infinity are probabilities; a NaN stays with the tokens whose candidate has it"""
    inf, nan = float('inf'), float('nan')
    h = torch.zeros(6, dim, dtype=torch.float64)
    h[:, :4] = torch.tensor([1.0, 0.5, -1.0, 0.25])
    table = torch.zeros(5, dim, dtype=torch.float64)
    table[:, :4] = torch.arange(20).double().reshape(5, 4) / 16 - 0.5
    ln = torch.tensor([-inf, inf, -1.0, nan, 0.5])
    ids = torch.tensor([[0, 1, 4], [1, 2, 4], [2, 0, 4], [3, 2, 4], [2, 3, 2], [2, 4, 4]], dtype=torch.int32)
    got = lm.nce_loss(E.to(h.to(dtype)), E.to(table.to(dtype)), E.to(ids), E.to(ln), 0.5, **E.kw)
    sign = torch.tensor([-1.0, 1.0, 1.0], dtype=torch.float64)
    rows = table[ids.long()]
    z = (rows * h[:, None]).sum(-1) - 0.5 - ln.double()[ids.long()]
    g = sign * torch.sigmoid(sign * z)
    soft = torch.where((sign * z).isnan(), nan, torch.nn.functional.softplus(sign * z, threshold=1e9))
    dtable = torch.zeros_like(table).index_add_(0, ids.long().reshape(-1), (g[:, :, None] * h[:, None]).reshape(-1, dim))
    half = torch.finfo(dtype).eps / 2
    # all terms are at most 4 in magnitude: z within 7 roundings of theirs, a sigmoid or softplus within 10, sums of at most 11
    for what, a, want, out in zip(('loss', 'dh', 'dtable'), got, (soft.sum(1), (g[:, :, None] * rows).sum(1), dtable), (R.U, half, R.U)):
        a = a.cpu().double()
        assert torch.equal(a.isnan(), want.isnan()) and torch.equal(a.isinf(), want.isinf()), (what, a, want)
        fine = want.isfinite()
        assert ((a - want).abs()[fine] <= 4 * 28 * R.U + out * want.abs()[fine]).all(), (what, a, want)


# ---- together --------------------------------------------------------------------------------------
def chain_inputs(lengths, vocab, dim, k, seed, ids=None):
    """a model and a batch of sentences of word ids, as they come out of an analysis"""
    g = rng(seed)
    offsets, rows = batch(lengths)
    if ids is None:
        ids = words(g, vocab, rows, none=False)
    following = torch.cat([ids[1:], ids[:1]]).clone()
    following[offsets[1:][offsets[1:] > offsets[:-1]].long() - 1] = -1   # nothing follows a sentence's last word
    noise = words(g, vocab, rows, k, none=False)
    cands = torch.cat([following[:, None], noise], 1).contiguous()
    return dict(offsets=offsets, ids=ids, cands=cands, table_gate=normal(g, vocab, dim, mean=1.0), table_x=normal(g, vocab, dim),
                table_out=normal(g, vocab, dim, std=dim ** -0.5), log_noise=normal(g, vocab, mean=-8.0), state=normal(g, len(lengths), dim))


def chain_step(E, m, scale=0.9, constant=1.0):
    """one training step of the language model: both lookups, the recurrence, the loss, and all of it backwards"""
    c = {k: E.to(v) for k, v in m.items()}
    vocab = m['table_x'].shape[0]
    gate, x = lm.embed(c['table_gate'], c['ids'], **E.kw), lm.embed(c['table_x'], c['ids'], scale, **E.kw)
    h, last, saved = lm.scan(gate, x, c['offsets'], c['state'], save=True, **E.kw)
    loss, dh, dout = lm.nce_loss(h, c['table_out'], c['cands'], c['log_noise'], constant, **E.kw)
    dgate, dx, dstate = lm.scan_grad(gate, x, dh, saved, c['offsets'], c['state'], **E.kw)
    return loss, lm.embed_grad(dgate, c['ids'], vocab, **E.kw), lm.embed_grad(dx, c['ids'], vocab, scale, **E.kw), dout, dstate, h


def chain_loss64(m, scale=0.9, constant=1.0):
    """the same loss in 64 bits, differentiable"""
    ids = m['ids'].long()
    gate, x = m['table_gate'][ids], m['table_x'][ids] * scale
    a = torch.sigmoid(gate)
    hs = []
    for i in range(len(m['offsets']) - 1):
        v = m['state'][i]
        for t in range(int(m['offsets'][i]), int(m['offsets'][i + 1])):
            v = a[t] * v + (1 - a[t]) * x[t]
            hs.append(v)
    h = torch.stack(hs)
    c = m['cands'].long()
    z = (m['table_out'][c.clamp(min=0)] * h[:, None, :]).sum(-1) - constant - m['log_noise'][c.clamp(min=0)]
    z = torch.cat([-z[:, :1], z[:, 1:]], 1)
    return (torch.nn.functional.softplus(z, threshold=1e9).sum(1) * (c[:, 0] >= 0)).sum()


def check_chain(E, m):
    names = ('table_gate', 'table_x', 'table_out', 'state')
    m64 = {k: v.double() if v.dtype == F32 else v for k, v in m.items()}
    leaves = [m64[k].clone().requires_grad_() for k in names]
    total = chain_loss64(dict(m64, **dict(zip(names, leaves))))
    grads = torch.autograd.grad(total, leaves)
    out = chain_step(E, m)
    # 64-bit autograd of the whole chain; 32-bit roundings of a chain of some fifty operations on values of order 1: 2e-5 of
    # the largest gradient is two hundred of them
    assert abs(out[0].cpu().double().sum() - total.detach()) <= 2e-5 * abs(total.detach())
    for name, a, b in zip(names, out[1:5], grads):
        assert (a.cpu().double() - b).abs().max() <= 2e-5 * b.abs().max(), name
    # and differences of the 64-bit loss along a direction in all four
    g = rng(99)
    way = [torch.randn(v.shape, generator=g, dtype=torch.float64) for v in leaves]
    eps = 1e-5
    up, down = (float(chain_loss64(dict(m64, **{k: v.detach() + s * eps * w for k, v, w in zip(names, leaves, way)}))) for s in (1, -1))
    slope = sum(float((a.cpu().double() * w).sum()) for a, w in zip(out[1:5], way))
    size = sum(float((b.abs() * w.abs()).sum()) for b, w in zip(grads, way))
    assert abs((up - down) / (2 * eps) - slope) <= 2e-5 * size


@check()
def chain_is_the_gradient_of_its_loss(E):
    check_chain(E, chain_inputs([9, 1, 0, 23, 4], 40, 36, 5, 1))


@check()
def chain_of_an_analysis(E):
    """the words of analysed sentences through a language model of one's own: analyse, look up, scan, loss, gradients"""
    import jumanpp_amd as J
    import numpy as np
    gold = os.path.join(ROOT, 'tests', 'golden')
    lines = [l.rstrip('\n') for l in open(os.path.join(gold, 'mini.txt'), encoding='utf-8')]
    ctx = J.Context(os.path.join(gold, 'mini_rnn.img'), lib_path=E.lib_path)
    res = ctx.analyze(lines).fetch(top1=True)
    vocab = 97
    ids, lengths = [], []
    for s in range(len(lines)):
        n = int(res.path_len[s]) if res.status[s] == 0 else 0
        nodes = res.nodes[int(res.node_base[s]):int(res.node_base[s]) + n][::-1]   # text order
        own = [int(e) % vocab for e in nodes['eptr'] if e >= 0]
        ids += own
        lengths.append(len(own))
    assert len(ids) > 100
    check_chain(E, chain_inputs(lengths, vocab, 32, 6, 2, ids=torch.tensor(np.array(ids, dtype=np.int32))))


# ---- refusals --------------------------------------------------------------------------------------
@check()
def refusals(E):
    f = lambda *s, dtype=F32: torch.zeros(*s, dtype=dtype, device=E.device)  # noqa: E731
    i = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device=E.device)  # noqa: E731
    off = torch.tensor([0, 2, 4], dtype=torch.int32, device=E.device)
    saved = f(1, 8)
    calls = [
        (lm.embed, (f(5, 8), i(3, dtype=torch.int16)), {}), (lm.embed, (f(5, 8), i(3, 1)), {}), (lm.embed, (f(5, 8).double(), i(3)), {}),
        (lm.embed, (f(5), i(3)), {}), (lm.embed, (f(5, 8).t(), i(3)), {}), (lm.embed, (f(5, 0), i(3)), {}),
        (lm.embed, (f(5, 8, dtype=BF16), i(3)), {'dtype': F32}), (lm.embed, (f(5, 8, dtype=BF16), i(3)), {'dtype': F16}),
        (lm.embed, (f(5, 8), i(6)[::2]), {}), (lm.embed_grad, (f(4, 8), i(3), 5), {}), (lm.embed_grad, (f(3, 8), i(3), -1), {}),
        (lm.embed_grad, (f(3, 8), i(3), 2 ** 31), {}), (lm.embed_grad, (f(3, 8), i(3, 1), 5), {}),
        (lm.scan, (f(4, 8), f(4, 9), off), {}), (lm.scan, (f(4, 8), f(4, 8, dtype=BF16), off), {}), (lm.scan, (f(4, 8), f(4, 8), off.long()), {}),
        (lm.scan, (f(4, 8), f(4, 8), off, f(3, 8)), {}), (lm.scan, (f(4, 8), f(4, 8), off, f(2, 8, dtype=BF16)), {}),
        (lm.scan, (f(4, 8), f(4, 8), off), {'max_len': -1}), (lm.scan, (f(4, 8), f(4, 8), off[:0]), {}), (lm.scan, (f(4, 0), f(4, 0), off), {}),
        (lm.scan_grad, (f(4, 8), f(4, 8), f(4, 8, dtype=BF16), saved, off), {}), (lm.scan_grad, (f(4, 8), f(4, 8), f(4, 8), f(2, 8), off), {}),
        (lm.scan_grad, (f(4, 8), f(4, 8), f(3, 8), saved, off), {}), (lm.scan_grad, (f(4, 8), f(4, 8), f(4, 8), saved, off, None, f(1, 8)), {}),
        (lm.embed, (f(5, 8), i(4)), {'dtype': torch.int32}), (lm.embed_grad, (f(8), i(8), 5), {}),
        (lm.nce_score, (f(4, 8), f(5, 9), i(4, 2), 0.0), {}), (lm.nce_score, (f(4, 8), f(5, 8), i(3, 2), 0.0), {}),
        (lm.nce_score, (f(4, 8), f(5, 8), i(4, 0), 0.0), {}), (lm.nce_score, (f(4, 8), f(5, 8, dtype=F16), i(4, 2), 0.0), {}),
        (lm.nce_loss, (f(4, 8), f(5, 8), i(4, 2), f(4), 0.0), {}), (lm.nce_loss, (f(4, 8), f(5, 8), i(4, 2), f(5, dtype=F16), 0.0), {}),
        (lm.nce_loss, (f(4, 8), f(5, 8), i(4, 2), f(5), 0.0, f(5)), {}), (lm.nce_loss, (f(4, 8), f(5, 8), i(4, 2), f(5, 1), 0.0), {}),
    ]
    for n, (fn, args, kw) in enumerate(calls):
        try:
            fn(*args, **kw, **E.kw)
        except JppGpuError:
            continue
        raise AssertionError('call %d of %s was not refused' % (n, fn.__name__))


@check()
def refusals_of_the_c_abi(E):
    """what the wrapper cannot get wrong: aliases, workspaces, strides, types, devices"""
    import struct
    lib = lm._lib(E.lib_path)
    a, b, c, out = (torch.zeros(6, 8, device=E.device) for _ in range(4))
    ids = torch.zeros(6, dtype=torch.int32, device=E.device)
    off = torch.tensor([0, 6], dtype=torch.int32, device=E.device)
    st, last = torch.zeros(1, 8, device=E.device), torch.zeros(1, 8, device=E.device)
    saved = torch.zeros(1, 8, device=E.device)
    ws = torch.zeros(1 << 16, dtype=torch.uint8, device=E.device)
    vec = torch.zeros(64, device=E.device)
    M = lambda t, stride=8, type=0, pad=0, shift=0: struct.pack('=QqiI', t.data_ptr() + shift, stride, type, pad)  # noqa: E731
    N = struct.pack('=QqiI', 0, 8, 0, 0)
    I = lambda t, n=4, pad=0, shift=0: struct.pack('=QiI', t.data_ptr() + shift, n, pad)  # noqa: E731
    dev, stream = lm._where(E.lib_path, a)
    w, wn = ws.data_ptr(), ws.numel()
    emb = lambda t=M(a), v=6, d=8, i=I(ids), n=6, o=M(out), device=dev: lib.jppgpu_lm_embed(t, v, d, i, n, 1.0, o, device, stream)  # noqa: E731
    eg = lambda dy=M(a), i=I(ids), n=6, v=6, d=8, o=M(out), wp=w, wb=wn: lib.jppgpu_lm_embed_grad(dy, i, n, v, d, 1.0, o, wp, wb, dev, stream)  # noqa: E731
    sc = lambda g=M(a), x=M(b), o=off.data_ptr(), n=1, r=6, d=8, ml=0, s=M(st), h=M(out), l=M(last), sv=saved.data_ptr(), wp=w, wb=wn: \
        lib.jppgpu_lm_scan(g, x, o, n, r, d, ml, s, h, l, sv, wp, wb, dev, stream)  # noqa: E731
    c2, out2, ds = torch.zeros(6, 8, device=E.device), torch.zeros(6, 8, device=E.device), torch.zeros(1, 8, device=E.device)
    sg = lambda dh=M(c), sv=saved.data_ptr(), dg=M(out), dx=M(out2), dl=M(last), s=M(ds): \
        lib.jppgpu_lm_scan_grad(M(a), M(b), off.data_ptr(), 1, 6, 8, 0, M(st), sv, dh, dl, dg, dx, s, w, wn, dev, stream)  # noqa: E731
    nl = lambda h=M(a), t=M(b), k=1, ln=vec.data_ptr(), lo=vec.data_ptr() + 64, dh=M(out), dt=M(out2), wp=w, wb=wn: \
        lib.jppgpu_lm_nce_loss(h, t, 6, 8, I(ids), 6, k, ln, 1.0, None, lo, dh, dt, wp, wb, dev, stream)  # noqa: E731
    for good in (emb, eg, sc, sg, nl):
        assert good() == 0, lib.jppgpu_last_error()
    bad = [lambda: emb(t=None), lambda: emb(t=N), lambda: emb(t=M(a, 7)), lambda: emb(t=M(a, 2 ** 41)), lambda: emb(t=M(a, 8, 3)), lambda: emb(t=M(a, pad=1)),
           lambda: emb(t=M(a, shift=2)), lambda: emb(v=-1), lambda: emb(d=0), lambda: emb(d=-8), lambda: emb(n=-1), lambda: emb(o=M(a)), lambda: emb(i=I(ids, 2)),
           lambda: emb(i=I(ids, 4, 1)), lambda: emb(i=I(ids, 8, 0, 4)), lambda: emb(i=None), lambda: emb(device=99), lambda: emb(device=-1),
           lambda: eg(o=M(out, 8, 1)), lambda: eg(wb=16), lambda: eg(wp=None), lambda: eg(wp=w + 4, wb=wn - 4), lambda: eg(n=2 ** 31), lambda: eg(o=M(a)), lambda: eg(dy=N),
           lambda: sc(o=None), lambda: sc(n=-1), lambda: sc(r=-1), lambda: sc(r=2 ** 31), lambda: sc(h=M(a)), lambda: sc(h=M(b)), lambda: sc(l=M(st)), lambda: sc(h=N),
           lambda: sc(l=M(last, 8, 1)), lambda: sc(s=M(st, 8, 2)), lambda: sc(h=M(out, 8, 1)), lambda: sc(o=off.data_ptr() + 2), lambda: sc(sv=saved.data_ptr() + 1),
           lambda: sc(r=600, ml=600, wb=0), lambda: sc(ml=-1),
           lambda: sg(sv=None), lambda: sg(dg=M(c)), lambda: sg(dx=M(out)), lambda: sg(s=M(last)), lambda: sg(dg=N), lambda: sg(dx=M(out2, 8, 1)), lambda: sg(dl=M(last, 8, 1)),
           lambda: nl(k=0), lambda: nl(ln=None), lambda: nl(lo=None), lambda: nl(dh=M(out, 8, 1)), lambda: nl(dt=M(out2, 8, 2)), lambda: nl(wb=0), lambda: nl(dh=M(a)),
           lambda: nl(dt=M(b)), lambda: nl(dt=M(out)), lambda: nl(k=2 ** 31 - 1), lambda: nl(t=M(b, 8, 1)), lambda: nl(ln=vec.data_ptr() + 2)]
    for n, call in enumerate(bad):
        if E.gpu is False and n in (16, 17):
            assert call() == 1
            continue
        assert call() == 1, n
        assert lib.jppgpu_last_error()


# ---- on the GPU alone --------------------------------------------------------------------------------
@check('gpu')
def cpu_tensors_are_refused(E):
    for call in (lambda: lm.embed(torch.zeros(3, 4), torch.zeros(2, dtype=torch.int32)),
                 lambda: lm.scan(torch.zeros(3, 4), torch.zeros(3, 4)),
                 lambda: lm.embed(torch.zeros(3, 4, device='cuda'), torch.zeros(2, dtype=torch.int32))):
        try:
            call()
        except JppGpuError:
            continue
        raise AssertionError('not refused')


@check('gpu', big=[False, True])
def streams(E, big):
    """on a stream of the caller's, behind work that is still running there; two streams at once"""
    m = [chain_inputs([9, 1, 0, 23, 4] if not big else [900, 40, 3000], 40, 36, 5, s) for s in (1, 2)]
    want = [chain_step(E, x) for x in m]
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in m]
    got = []
    for s, x in zip(side, m):
        with torch.cuda.stream(s):
            a = torch.randn(3000, 3000, device='cuda')
            for _ in range(20):
                a = (a @ a).clamp_(-1, 1)
            x = dict(x, table_x=(x['table_x'].to('cuda') + a[:x['table_x'].shape[0], :36] * 0.0))
            got.append(chain_step(E, x))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            equal('on a stream', a, b)


@check('gpu')
def threads(E):
    """threads at once, each on a stream of its own; one that is refused has its own message"""
    m = [chain_inputs([9, 1, 0, 23, 4] if s % 2 else [900, 40, 700], 40, 36, 5, s) for s in range(4)]
    want = [chain_step(E, x) for x in m]
    torch.cuda.synchronize()
    trouble = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = chain_step(E, m[i])
                    torch.cuda.current_stream().synchronize()
                    for a, b in zip(got, want[i]):
                        equal('in thread %d' % i, a, b)
        except Exception:
            trouble.append(traceback.format_exc())

    def refused():
        try:
            for _ in range(50):
                try:
                    lm.embed(torch.zeros(3, 4, device='cuda', dtype=BF16), torch.zeros(2, dtype=torch.int32, device='cuda'), dtype=F32)
                except JppGpuError as e:
                    assert 'of the table' in str(e), e
                    continue
                raise AssertionError('not refused')
        except Exception:
            trouble.append(traceback.format_exc())

    running = [threading.Thread(target=work, args=(i,)) for i in range(len(m))] + [threading.Thread(target=refused)]
    for t in running:
        t.start()
    for t in running:
        t.join()
    assert not trouble, trouble[0]


@check('gpu', big=[False, True])
def graph(E, big):
    """captured once, replayed with other inputs in the same buffers, eager work of the same operators in between"""
    m = chain_inputs([9, 1, 0, 23, 4] if not big else [900, 40, 3000], 40, 36, 5, 1)
    c = {k: v.to('cuda') for k, v in m.items()}
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        chain_step(E, c)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = chain_step(E, c)
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):   # a second graph of the same calls, with workspaces of its own
        out2 = chain_step(E, c)
    for seed in range(1, 5):
        new = chain_inputs([9, 1, 0, 23, 4] if not big else [900, 40, 3000], 40, 36, 5, seed)
        for k in c:
            c[k].copy_(new[k])
        g.replay()
        g2.replay()
        eager = chain_step(E, new)
        torch.cuda.synchronize()
        for a, b, d in zip(out, eager, out2):
            equal('replay %d' % seed, a, b)
            equal('replay %d of the second graph' % seed, d, b)


@check('gpu')
def offsets_beyond_32_bits(E):
    """more than 2^32 elements: rows far into the matrices"""
    table = torch.randn(1000, 256, device='cuda', dtype=BF16)
    n = 2 ** 24 + 77
    ids = torch.arange(n, device='cuda', dtype=torch.int32) * 31 % 1000
    out = lm.embed(table, ids)
    for a, b in ((0, 5000), (2 ** 23 - 7, 2 ** 23 + 5000), (n - 5000, n)):
        equal('rows', out[a:b], table[ids[a:b].long()])
    grad = lm.embed_grad(out, ids, 1000)
    count = torch.bincount(ids, minlength=1000).double()
    want = table.double() * count[:, None]
    # every word's rows are equal: a 32-bit sum of n of them is within n U of n times one
    assert ((grad.double() - want).abs() <= count[:, None] * R.U * want.abs() + 1e-30).all()
    del grad
    gate = out
    half = 2 ** 23
    offsets = torch.tensor([0, half, n - 300, n], dtype=torch.int32, device='cuda')
    for max_len in (0, 100):
        h, last, saved = lm.scan(gate, out, offsets, max_len=max_len, save=True)
        h1, last1, saved1 = lm.scan(gate[-300:], out[-300:], max_len=1)[:2] + (None,)
        # the last sentence alone, walked by one wavefront in both: other splits round elsewhere
        want_h, want_last, _ = R.scan(gate[-300:].cpu(), out[-300:].cpu(), [0, 300], None, BF16, torch.zeros(300, 256))
        near('h', h[-300:], want_h)
        near('last', last[2:], want_last)
        near('alone', h1, want_h)
        if max_len == 0:
            dgate, dx, dstate = lm.scan_grad(gate, out, h, saved, offsets, max_len=max_len)
            hc = h[-300:].cpu()
            want = R.scan_grad(gate[-300:].cpu(), out[-300:].cpu(), [0, 300], None, hc, None, BF16, torch.zeros(300, 256))
            near('dgate', dgate[-300:], want[0])
            near('dx', dx[-300:], want[1])
            near('dstate', dstate[2:], want[2])
            del dgate, dx, dstate
        del h, last, saved


@check('gpu', dtype=[F32, BF16])
def large(E, dtype):
    """the sizes of a whole batch: against 64 bits on the GPU, by the norms of the differences"""
    g = torch.Generator(device='cuda')
    g.manual_seed(5)
    n, vocab, dim, k = 200003, 30011, 100, 9
    ids = (torch.rand(n, k, generator=g, device='cuda') ** 4 * vocab).int()
    h = torch.randn(n, dim, generator=g, device='cuda').to(dtype)
    table = (torch.randn(vocab, dim, generator=g, device='cuda') * 0.1).to(dtype)
    ln = torch.full((vocab,), -9.0, device='cuda')
    loss, dh, dtable = lm.nce_loss(h, table, ids, ln, 1.0)
    z = torch.matmul(table.double()[ids.long()], h.double()[:, :, None])[:, :, 0] + 8.0
    z[:, 0] *= -1
    want = torch.nn.functional.softplus(z, threshold=1e9).sum(1)
    gz = torch.sigmoid(z)
    gz[:, 0] *= -1
    wdh = torch.matmul(gz[:, None, :], table.double()[ids.long()])[:, 0]
    wdt = torch.zeros(vocab, dim, dtype=torch.float64, device='cuda')
    wdt.index_add_(0, ids.reshape(-1).long(), (gz[:, :, None] * h.double()[:, None, :]).reshape(-1, dim))
    rel = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    # norms of roundings: independent ones of U (32 bits) or half a unit of the type, a sum's at most the root of its length times
    assert rel(loss, want) <= 16 * R.U and rel(dh, wdh) <= torch.finfo(dtype).eps / 2 + 16 * R.U and rel(dtable, wdt) <= 300 * R.U


# ---- long memories, infinities, padded batches -----------------------------------------------------------
@check(dtype=[F32, BF16, F16], max_len=[0, 1])
def scan_open_gates_do_not_drift(E, dtype, max_len):
    """gates near one over a long sentence: the state is a mean over 1 / (1 - a) rows, so weights of state and input that do not
    sum to one would show that many times over.  What 32-bit states cannot do without is the rounding of every row's result.
    Those of N rows within the state's memory, N <= 1 / (2 (1 - a)), are off by at most U of it and independent (the rows
    differ), so their sum has a standard deviation of at most U sqrt(N / 3) of the largest state; four roundings a row (the
    result's, the map's of a chunk, the sum's and the step's of the gradient) double that, and six deviations are 7 U sqrt(N).
    The weights' own roundings act on differences from the mean, without the factor: 20 U."""
    rows = 20000
    g = rng(17)
    columns = [7.25, 8.0, 9.0, 10.0, 11.0, 3.0, 0.0, -9.0]
    gate = torch.tensor(columns + [9.0, 9.0]).repeat(rows, 1)
    gate[:, -2:] += torch.randn(rows, 2, generator=g)
    gate = gate.to(dtype)
    x, dh = (normal(g, rows, len(columns) + 2, dtype=dtype, mean=1.0, std=0.3) for _ in range(2))
    state, dlast = torch.full((1, x.shape[1]), 0.25), torch.full((1, x.shape[1]), -3.0)
    off = torch.tensor([0, rows], dtype=torch.int32)
    # 64 bits
    z, xd, dhd = gate.double(), x.double(), dh.double()
    a, b = torch.sigmoid(z), torch.sigmoid(-z)
    before, h, delta = torch.empty_like(xd), torch.empty_like(xd), torch.empty_like(xd)
    v = state[0].double()
    for t in range(rows):
        before[t] = v
        v = v + b[t] * (xd[t] - v)
        h[t] = v
    back = dlast[0].double()
    for t in reversed(range(rows)):
        delta[t] = dhd[t] + back
        back = delta[t] * a[t]
    memory = (0.5 / b.mean(0)).clamp(1, rows)
    tol = (7 * memory.sqrt() + 20) * R.U
    most, most_d = before.abs().amax(0).maximum(xd.abs().amax(0)), delta.abs().amax(0)
    e_h, e_d = tol * most, tol * most_d
    diff = (before - xd).abs()
    want = [R.out_round(h, e_h.expand_as(h), dtype), R.out_round(v[None], e_h[None], F32),
            R.out_round(delta * a * b * (before - xd), a * b * (e_d * diff + delta.abs() * e_h + 20 * R.U * delta.abs() * most), dtype),
            R.out_round(delta * b, b * (e_d + 20 * R.U * delta.abs()), dtype), R.out_round(back[None], e_d[None], F32)]
    od = E.to(off)
    hg, last, saved = lm.scan(E.to(gate), E.to(x), od, E.to(state), max_len=max_len, save=True, **E.kw)
    got = (hg, last) + lm.scan_grad(E.to(gate), E.to(x), E.to(dh), saved, od, E.to(state), E.to(dlast), max_len=max_len, **E.kw)
    for what, p, q in zip(('h', 'last', 'dgate', 'dx', 'dstate'), got, want):
        near(what, p, q)


@check(dtype=[F32, BF16], max_len=[0, 1])
def scan_infinite_inputs(E, dtype, max_len):
    """an infinity is what the formula makes of it, in the columns that have it and in no other: infinite states behind an infinite
    input, NaN where opposite ones meet; and differences beyond the largest number are no infinities"""
    inf = float('inf')
    rows, dim = 300, 70
    g = rng(23)
    gate, x, dh = normal(g, rows, dim, mean=1.0, dtype=dtype), normal(g, rows, dim, dtype=dtype), normal(g, rows, dim, dtype=dtype)
    state, dlast = normal(g, 1, dim), normal(g, 1, dim)
    od = torch.tensor([0, rows], dtype=torch.int32)

    def run(gate, x, dh, state, dlast):
        h, last, saved = lm.scan(E.to(gate), E.to(x), E.to(od), E.to(state), max_len=max_len, save=True, **E.kw)
        return [t.cpu() for t in (h, last) + lm.scan_grad(E.to(gate), E.to(x), E.to(dh), saved, E.to(od), E.to(state), E.to(dlast), max_len=max_len, **E.kw)]

    plain = run(gate, x, dh, state, dlast)
    x[40, 3], x[41, 4], x[203, 4], state[0, 69], dh[250, 5], dlast[0, 6], dh[17, 8], dh[16, 8] = inf, inf, -inf, -inf, inf, -inf, inf, -inf
    big = 3e38
    x[60, 7], x[61, 7], gate[60, 7], gate[61, 7] = big, -big, 0, 0
    gate[:, 9], state[0, 9], dlast[0, 9] = -9, inf, inf   # (their product over a chunk is below the smallest number)
    dirty = [3, 4, 5, 6, 7, 8, 9, 69]
    got = run(gate, x, dh, state, dlast)
    clean = torch.ones(dim, dtype=torch.bool)
    clean[dirty] = False
    for what, a, b in zip(('h', 'last', 'dgate', 'dx', 'dstate'), got, plain):
        equal(what + ' of the other columns', a[:, clean], b[:, clean])
    h, last, dgate, dx, dstate = got
    assert h[:40, 3].isfinite().all() and (h[40:, 3] == inf).all() and last[0, 3] == inf
    assert (h[41:203, 4] == inf).all() and h[203:, 4].isnan().all() and last[0, 4].isnan()
    assert (h[:, 69] == -inf).all() and last[0, 69] == -inf
    assert (h[:, 9] == inf).all() and last[0, 9] == inf and (dx[:, 9] == inf).all() and dstate[0, 9] == inf
    assert (dx[:251, 5] == inf).all() and dx[251:, 5].isfinite().all() and dstate[0, 5] == inf
    assert (dx[:, 6] == -inf).all() and dstate[0, 6] == -inf
    assert dx[18:, 8].isfinite().all() and dx[17, 8] == inf and dx[:17, 8].isnan().all() and dstate[0, 8].isnan()
    # half of 3e38 and a half of the state, then a quarter of it and half of -3e38: rounded values of that size
    want = torch.stack([x[60, 7].double() / 2, x[60, 7].double() / 4 + x[61, 7].double() / 2])
    assert ((h[60:62, 7].double() - want).abs() <= torch.finfo(dtype).eps * 3e38).all()
    assert h[:, 7].isfinite().all() and dx[:, 7].isfinite().all()


@check(dtype=[F32, BF16, F16])
def scan_states_are_32_bit_states(E, dtype):
    """what comes back in 32 bits is right to 32 bits, whatever the rows are: one step whose result is a gate's weight itself, whose
    relative rounding is that of two instructions of 2 U each and two sums (6 U), and the step's (2 U)"""
    z = torch.linspace(0.25, 80, 320).to(dtype).float()
    n, dim = 4, len(z)
    gate = torch.stack([-z, z, -z, z]).to(dtype)
    x = torch.tensor([0.0, 1.0, 0.0, 1.0])[:, None].expand(n, dim).contiguous().to(dtype)
    state = torch.tensor([1.0, 0.0, -3.0, 0.0])[:, None].expand(n, dim).contiguous()
    dlast = torch.tensor([1.0, 0.0, 5.0, 0.0])[:, None].expand(n, dim).contiguous()
    off = E.to(torch.arange(n + 1, dtype=torch.int32))
    h, last, saved = lm.scan(E.to(gate), E.to(x), off, E.to(state), max_len=1, save=True, **E.kw)
    _, _, dstate = lm.scan_grad(E.to(gate), E.to(x), torch.zeros_like(h), saved, off, E.to(state), E.to(dlast), max_len=1, **E.kw)
    s = torch.sigmoid(-z.double())
    scale = torch.tensor([1.0, 1.0, 3.0, 1.0], dtype=torch.float64)[:, None]
    near('last', last, (torch.tensor([1.0, 1.0, -3.0, 1.0], dtype=torch.float64)[:, None] * s, R.SLACK * 8 * R.U * scale * s + R.TINY))
    want = torch.stack([s, 0 * s, 5 * s, 0 * s])
    near('dstate', dstate, (want, R.SLACK * 8 * R.U * want + R.TINY))


@check(dtype=[F32, BF16, F16], dim=[8, 128, 600])
def nce_dh_is_summed_in_32_bits(E, dtype, dim):
    """far scores whose parts of dh nearly cancel: what is left shows the precision of each part, which is rounded to the type only
    in the end.  A part's gradient is within 7 U (sigmoid 6 U, weight), the sum of three parts within 5 U of their magnitudes."""
    pairs = [(-20.0, -19.5), (-40.0, -39.0), (-60.0, -58.5), (-12.0, -11.75), (8.0, -7.5), (30.0, 25.0), (-3.0, -2.5), (-80.0, -78.0)]
    n, cands = len(pairs), 3
    h = torch.zeros(n, dim)
    h[:, 0] = 1
    table = torch.zeros(2 * n + 1, dim, dtype=torch.float64)
    table[2 * n, 0] = 1.0
    g = rng(31)
    for i, (z1, z2) in enumerate(pairs):
        table[2 * i, 0], table[2 * i + 1, 0] = z1, z2
        w = (torch.rand(dim - 1, generator=g) + 1).to(dtype).double()
        ratio = torch.sigmoid(torch.tensor(z1, dtype=torch.float64)) / torch.sigmoid(torch.tensor(z2, dtype=torch.float64))
        table[2 * i, 1:], table[2 * i + 1, 1:] = w, -(w * ratio)
    table = table.to(dtype)
    ids = torch.stack([torch.full((n,), 2 * n), torch.arange(n) * 2, torch.arange(n) * 2 + 1], 1).to(torch.int32)
    _, dh, _ = lm.nce_loss(E.to(h.to(dtype)), E.to(table), E.to(ids), E.to(torch.zeros(2 * n + 1)), 0.0, **E.kw)
    rows = table.double()[ids.long()]
    z = rows[:, :, 0]   # (exact: products with one and zero)
    gz = torch.sigmoid(z)
    gz[:, 0] = -torch.sigmoid(-z[:, 0])
    parts = gz[:, :, None] * rows
    want = parts.sum(1)
    assert (want.abs()[:, 1:] < 0.01 * parts.abs().sum(1)[:, 1:]).any()
    near('dh', dh, R.out_round(want, 12 * R.U * parts.abs().sum(1), dtype))


# lengths, rows in front, rows behind: empty sentences at the ends and between, many more than rows
EMPTY_CASES = (([1000] + [0] * 4000, 0, 984), ([0] * 3000 + [400, 0, 0, 300] + [0] * 3000 + [5, 270] + [0] * 70, 33, 700), ([0] * 2000, 0, 600),
               ([0] * 2000, 600, 0), ([300] + [0, 1] * 200 + [0] * 64 + [290], 7, 9))


@check(case=range(len(EMPTY_CASES)), dtype=[F32, F16])
def scan_many_empty_sentences(E, case, dtype):
    """a batch of a fixed number of sentences and rows, most of them unused: the rows and states of the others, and the states of
    the empty ones"""
    dim = 9
    lengths, front, back = EMPTY_CASES[case]
    offsets, rows, gate, x, dh, state, dlast, fill = scan_inputs((lengths, front, back), dim, dtype, case)
    fill = fill.to(dtype).float()
    want_h, want_last, _ = R.scan(gate, x, offsets, state, dtype, fill)
    want = R.scan_grad(gate, x, offsets, state, dh, dlast, dtype, fill)
    gd, xd, dhd, sd, ld, od = (E.to(t) for t in (gate, x, dh, state, dlast, offsets))
    for max_len in (0, 1000, 1):
        h, last, saved = raw_scan(E, gd, xd, od, sd, max_len, fill)
        near('h', h, want_h)
        near('last', last, want_last)
        for what, a, b in zip(('dgate', 'dx', 'dstate'), raw_scan_grad(E, gd, xd, od, sd, max_len, saved, dhd, ld, fill), want):
            near(what, a, b)


@check(where_from=['behind', 'between'])
def scan_empty_sentences_are_not_walked(E, where_from):
    """what a batch's sentences without a row cost does not depend on whose way they lie in: as many in front of all rows, where no
    chunk meets them, take as long.  (Walked one by one, those behind took ten times as long on the emulator.)"""
    import time
    n, rows, dim = 40000, 1984, 4
    g = rng(1)
    gate, x, dh = (E.to(normal(g, rows, dim)) for _ in range(3))

    def took(lengths):
        offsets = E.to(batch(lengths)[0])
        best = 1e9
        for _ in range(3):
            t = time.perf_counter()
            h, last, saved = lm.scan(gate, x, offsets, max_len=1000, save=True, **E.kw)
            lm.scan_grad(gate, x, h, saved, offsets, max_len=1000, **E.kw)
            if E.gpu:
                torch.cuda.synchronize()
            best = min(best, time.perf_counter() - t)
        return best

    none = [0] * n
    plain = took(none + [700, 300])
    assert took([700] + none + [300] if where_from == 'between' else [700, 300] + none) < 3 * plain


@check(case=[([5, 0, 7], 3, 9), ([300], 40, 70), ([0, 0], 0, 40), ([0], 30, 0), ([], 6, 7), ([9, 2], 0, 5000), ([2, 270, 1], 1000, 3000)], dtype=[F32, F16],
       dim=[36, 130])
def scan_rows_of_no_sentence_are_zero(E, case, dtype, dim):
    """a padded batch: nothing is left in the results' other rows that a product with the whole matrix would take up"""
    lengths, front, back = case
    offsets, rows, gate, x, dh, state, dlast, _ = scan_inputs(case, dim, dtype, len(lengths))
    gate[:front], x[:front], dh[:front] = (float('nan'),) * 3
    gate[rows - back:], x[rows - back:], dh[rows - back:] = (float('nan'),) * 3
    gd, xd, dhd, sd, ld, od = (E.to(t) for t in (gate, x, dh, state, dlast, offsets))
    rest = torch.ones(rows, dtype=torch.bool)
    rest[front:rows - back] = False
    for max_len in (0, max(lengths + [1])):
        fill = torch.full((rows, dim), float('nan'))
        for _ in range(3):   # (memory that held something else)
            soil = [E.to(torch.full((rows, dim), float('nan'), dtype=dtype)) for _ in range(4)]
            del soil
            h, last, saved = lm.scan(gd, xd, od, sd, max_len=max_len, save=True, **E.kw)
            dgate, dx, dstate = lm.scan_grad(gd, xd, dhd, saved, od, sd, ld, max_len=max_len, **E.kw)
            for what, t in zip(('h', 'dgate', 'dx'), (h, dgate, dx)):
                assert (t.cpu()[rest] == 0).all(), what
        # the caller's own matrices keep what they hold, unless they are to be cleared
        left = raw_scan(E, gd, xd, od, sd, max_len, fill)
        assert left[0].cpu()[rest].isnan().all()
        equal('h', left[0].cpu()[~rest], h.cpu()[~rest])
        equal('last', left[1], last)


@check()
def clearing_is_for_results_of_a_batch(E):
    """the flag of a packed batch's results is no type of anything else"""
    import struct
    lib = lm._lib(E.lib_path)
    a, b, c, out, out2, out3 = (torch.zeros(6, 8, device=E.device) for _ in range(6))
    off = torch.tensor([0, 6], dtype=torch.int32, device=E.device)
    st, last, saved, ids = torch.zeros(1, 8, device=E.device), torch.zeros(1, 8, device=E.device), torch.zeros(1, 8, device=E.device), off.new_zeros(6)
    M = lambda t, clear=0: struct.pack('=QqiI', t.data_ptr(), 8, clear, 0)  # noqa: E731
    dev, stream = lm._where(E.lib_path, a)
    sc = lambda g=0, s=0, h=0, l=0: lib.jppgpu_lm_scan(M(a, g), M(b), off.data_ptr(), 1, 6, 8, 0, M(st, s), M(out, h), M(last, l),  # noqa: E731
                                                       saved.data_ptr(), None, 0, dev, stream)
    sg = lambda dh=0, dg=0, dx=0, ds=0: lib.jppgpu_lm_scan_grad(M(a), M(b), off.data_ptr(), 1, 6, 8, 0, M(st), saved.data_ptr(), M(c, dh), None,  # noqa: E731
                                                                M(out2, dg), M(out3, dx), M(last, ds), None, 0, dev, stream)
    em = lambda o=0: lib.jppgpu_lm_embed(M(a), 6, 8, struct.pack('=QiI', ids.data_ptr(), 4, 0), 6, 1.0, M(out, o), dev, stream)  # noqa: E731
    assert sc() == sc(h=0x100) == sg() == sg(dg=0x100) == sg(dx=0x100) == sg(dg=0x100, dx=0x100) == em() == 0
    assert 0 not in (sc(g=0x100), sc(s=0x100), sc(l=0x100), sc(h=0x200), sc(h=0x101), sg(dh=0x100), sg(ds=0x100), sg(dx=0x102), em(o=0x100))


@check()
def recorded_gradients_are_refused(E):
    """no call is part of torch's graph of a loss: an input whose gradient is being recorded would lose it without a word"""
    g = rng(41)
    n, dim, vocab = 6, 12, 9
    gate, x, table = E.to(normal(g, n, dim)), E.to(normal(g, n, dim)), E.to(normal(g, vocab, dim))
    ids, cands = E.to(words(g, vocab, n)), E.to(words(g, vocab, n, 3))
    off, state, ln, weight = E.to(torch.tensor([0, 2, n], dtype=torch.int32)), E.to(normal(g, 2, dim)), E.to(normal(g, vocab)), E.to(torch.rand(n, generator=g))
    saved = lm.scan(gate, x, off, state, save=True, **E.kw)[2]
    calls = [(lm.embed, [table, ids]), (lm.embed_grad, [x, ids, vocab]), (lm.scan, [gate, x, off, state]),
             (lm.scan_grad, [gate, x, gate, saved, off, state, state]), (lm.nce_score, [x, table, cands, 0.5]),
             (lm.nce_loss, [x, table, cands, ln, 0.5, weight])]
    for fn, args in calls:
        want = fn(*args, **E.kw)
        for i, a in enumerate(args):
            if not torch.is_tensor(a) or not a.is_floating_point():
                continue
            leaf = [a.detach().clone().requires_grad_() if j == i else b for j, b in enumerate(args)]
            for these in (leaf, [b * 1 if torch.is_tensor(b) and b.requires_grad else b for b in leaf]):
                try:
                    fn(*these, **E.kw)
                except JppGpuError as e:
                    assert 'no_grad' in str(e), e
                else:
                    raise AssertionError('%s, argument %d: not refused' % (fn.__name__, i))
                for off_ in (torch.no_grad, torch.inference_mode):
                    with off_():
                        got = fn(*these, **E.kw)
                    for p, q in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                        equal(fn.__name__, p, q)


@check(dim=[36, 300, 1500], dtype=[F32, BF16])
def nce_dh_alone_leaves_the_workspace(E, dim, dtype):
    """the gradients of the scores are written for the table's gradient alone (and for dh of rows that are walked in blocks)"""
    n, k, vocab = 20, 7, 30
    h, table, ids, used, log_noise, weight = nce_inputs(n, k, vocab, dim, dtype, 4)
    h, table, ids, log_noise, weight = (E.to(t) for t in (h, table, ids, log_noise, weight))
    _, want, _ = lm.nce_loss(h, table, ids, log_noise, 1.0, weight, **E.kw)
    lib = lm._lib(E.lib_path)
    dev, stream = lm._where(E.lib_path, h)
    loss, dh = torch.empty(n, device=E.device), torch.empty_like(h)
    ws, wp, wn = lm._workspace(lib, 'jppgpu_lm_nce_loss_workspace', (n, k, vocab, dim), h)
    ws.fill_(255)
    lm._check(lib, lib.jppgpu_lm_nce_loss(lm._rows(h, 'h'), lm._rows(table, 't'), vocab, dim, lm._ids(ids), n, k, log_noise.data_ptr(), 1.0,
                                          weight.data_ptr(), loss.data_ptr(), lm._rows(dh, 'dh'), None, wp, wn, dev, stream))
    equal('dh', dh, want)
    in_blocks = dim * dh.element_size() // 16 > 256
    assert in_blocks or bool((ws == 255).all())


@check('gpu', types=[(F32, BF16), (F32, F16), (F32, F32), (BF16, BF16), (F16, F16)], dim=[100, 257], size=['small', 'many', 'streamed'])
def embed_many(E, types, dim, size):
    """either side of where a thread takes four packs and of where results leave with the hint, at widths that no pack divides"""
    per = 16 // torch.tensor([], dtype=types[1]).element_size()
    packs = -(-dim // per)
    four = 4 * 256 * 2048
    n = {'small': (four - 1) // packs, 'many': -(-four // packs), 'streamed': (64 << 20) // (dim * torch.tensor([], dtype=types[1]).element_size()) + 1}[size]
    vocab = 5003
    table = torch.randn(vocab, dim, device='cuda').to(types[0])
    ids = torch.randint(-3, vocab + 3, (n,), device='cuda', dtype=torch.int32)
    got = lm.embed(table, ids, 0.7, dtype=types[1])
    ok = (ids >= 0) & (ids < vocab)
    scale = float(torch.tensor(0.7))
    for part in torch.arange(n, device='cuda').split(50000):
        exact = torch.where(ok[part][:, None], table[torch.where(ok, ids, 0)[part].long()].double() * scale, 0.0)
        # the product rounded to 32 bits (U) and then to the type, or to the type at once: halves have an instruction for both
        value, bound = R.out_round(exact, R.U * exact.abs(), types[1])
        assert bool(((got[part].double() - value).abs() <= bound).all())


@check('gpu', dtype=[F32, BF16, F16], dim=[130, 201, 300], long=[False, True])
def scan_streamed(E, dtype, dim, long):
    """results beyond where they leave with the hint, at widths whose last pack is moved back: a walk of short sentences, and chunks"""
    rows = (64 << 20) // (dim * torch.tensor([], dtype=dtype).element_size()) + 77
    g = rng(dim)
    cut = torch.randint(0, rows + 1, (40 if long else rows // 20,), generator=g).sort().values
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), cut, torch.tensor([rows])]).to(torch.int32)
    n = len(offsets) - 1
    longest = int((offsets[1:] - offsets[:-1]).max())
    d = torch.Generator(device='cuda')
    d.manual_seed(dim)
    gate, x, dh = (torch.randn(rows, dim, generator=d, device='cuda').mul_(2).add_(m).to(dtype) for m in (1.5, 0.0, 0.0))
    state, dlast = (torch.randn(n, dim, generator=d, device='cuda') for _ in range(2))
    od = offsets.cuda()
    assert long or longest <= 256
    h, last, saved = lm.scan(gate, x, od, state, max_len=longest, save=True)
    out = lm.scan_grad(gate, x, dh, saved, od, state, dlast, max_len=longest)
    for i in [0, 1, n // 3, n // 2, n - 2, n - 1] + torch.randint(0, n, (20 if not long else 2,), generator=g).tolist():
        a, b = int(offsets[i]), int(offsets[i + 1])
        if b - a > 12000:
            continue
        rows_of = [t[a:b].cpu() for t in (gate, x, dh)]
        states = [t[i:i + 1].cpu() for t in (state, dlast)]
        fill = torch.zeros(b - a, dim)
        want_h, want_last, _ = R.scan(rows_of[0], rows_of[1], [0, b - a], states[0], dtype, fill)
        near('h of sentence %d' % i, h[a:b], want_h)
        near('last of sentence %d' % i, last[i:i + 1], want_last)
        want = R.scan_grad(rows_of[0], rows_of[1], [0, b - a], states[0], rows_of[2], states[1], dtype, fill)
        for what, p, q in zip(('dgate', 'dx', 'dstate'), (out[0][a:b], out[1][a:b], out[2][i:i + 1]), want):
            near('%s of sentence %d' % (what, i), p, q)


@check()
def scores_reach_the_lattice(E):
    """a language model of one's own as a host scorer: at every boundary the states of the global beam's left words (looked up and put
    through one step of the recurrence) score all words that may follow, and the scores, which are those of the same model in 64
    bits, go into the analysis's cells and change its paths"""
    import jumanpp_amd as J
    import numpy as np
    gold = os.path.join(ROOT, 'tests', 'golden')
    lines = [l.rstrip('\n') for l in open(os.path.join(gold, 'mini.txt'), encoding='utf-8')]
    vocab, dim, constant, unknown = 97, 32, 2.0, -4.0
    g = rng(7)
    gates, inputs, out = normal(g, vocab, dim), normal(g, vocab, dim, std=4.0), normal(g, vocab, dim)
    dev = [E.to(t) for t in (gates, inputs, out)]

    def word(node):
        return int(node['eptr']) % vocab if node['eptr'] >= 0 else -1

    def boundaries(lat):
        """(first cell row, left words of the global beam, right words) of every scored boundary"""
        for s in range(lat['n']):
            if lat['status'][s] != 0 or int(lat['ncp'][s]) == 0:
                continue
            nb, bb = int(lat['node_base'][s]), int(lat['bnd_base'][s])
            for b in range(bb + 2, bb + int(lat['ncp'][s]) + 3):
                right = nb + int(lat['bnd_first'][b])
                n = int(lat['bnd_count'][b])
                if n == 0:
                    continue   # (nothing starts here: no global beam)
                ends = nb + int(lat['end_first'][b])
                left = [nb + int(lat['end_nodes'][ends + int(lat['gbeam_entries'][b][i]['left'])]) for i in range(int(lat['gbeam_count'][b]))]
                if left:
                    yield right, [word(lat['nodes'][i]) for i in left], [word(lat['nodes'][right + r]) for r in range(n)]

    def own(lat, idx, cells):
        todo = list(boundaries(lat))
        most = max(len(r) for _, _, r in todo)
        ids = torch.tensor([w for _, left, _ in todo for w in left], dtype=torch.int32)
        cands = torch.tensor([right + [-1] * (most - len(right)) for _, left, right in todo for _ in left], dtype=torch.int32)
        idd, off = E.to(ids), E.to(torch.arange(len(ids) + 1, dtype=torch.int32))
        h, _ = lm.scan(lm.embed(dev[0], idd, **E.kw), lm.embed(dev[1], idd, **E.kw), off, max_len=1, **E.kw)
        scores = lm.nce_score(h, dev[2], E.to(cands), constant, **E.kw).cpu().numpy()
        scores = np.where(np.isfinite(scores), scores, np.float32(unknown))
        row = 0
        for first, left, right in todo:
            cells[first:first + len(right), :len(left), idx] = scores[row:row + len(left), :len(right)].T
            row += len(left)

    def in64(lat, idx, cells):
        a, b, c = (t.double().numpy() for t in (gates, inputs, out))
        for first, left, right in boundaries(lat):
            for i, l in enumerate(left):
                h = b[l] / (1 + np.exp(a[l])) if l >= 0 else np.zeros(dim)
                for r, w in enumerate(right):
                    cells[first + r, i, idx] = c[w] @ h - constant if w >= 0 else unknown

    def paths(scorer, weight):
        kept = []

        def keeping(lat, idx, cells):
            scorer(lat, idx, cells)
            kept.append(cells[:, :, idx].copy())
        ctx = J.Context(os.path.join(gold, 'mini.img'), lib_path=E.lib_path, host_scorer_weights=[weight])
        res = ctx.analyze_scored(lines, [keeping]).fetch(top1=True)
        got = []
        for s in range(len(lines)):
            n = int(res.path_len[s]) if res.status[s] == 0 else 0
            nodes = res.nodes[int(res.node_base[s]):int(res.node_base[s]) + n]
            got.append([(int(x['eptr']), int(x['start']), int(x['end'])) for x in nodes])
        return got, kept[0]

    def replay(lat, idx, into):
        into[:, :, idx] = cells

    mine, cells = paths(own, 0.5)
    _, cells64 = paths(in64, 0.5)
    # 32-bit roundings of a state (10 U) and of a product of 32 terms (34 U) of magnitudes that sum to less than 100
    assert np.abs(cells.astype(np.float64) - cells64).max() <= 50 * R.U * 100 and (cells64 != 0).sum() > 1000
    # (two words unknown to the model score alike, so roundings may choose between paths: the paths are those of these scores)
    assert mine == paths(replay, 0.5)[0]
    without = paths(lambda lat, idx, cells: None, 0.5)[0]
    assert sum(a != b for a, b in zip(mine, without)) >= 3, 'the scorer has to matter'


@check(dtype=[F32, F16], dim=[130, 203, 262], max_len=[0, 1])
def scan_not_finite_stays_in_its_column(E, dtype, dim, max_len):
    """infinities and NaN next to every kind of column: of the same pack, of the pack that is moved back to the row's end, which two
    lanes have; the other columns keep their bits"""
    inf, nan = float('inf'), float('nan')
    offsets, rows, gate, x, dh, state, dlast, _ = scan_inputs(([290, 0, 41], 3, 5), dim, dtype, dim)
    od = E.to(offsets)

    def run(gate, x, dh, state, dlast):
        h, last, saved = lm.scan(E.to(gate), E.to(x), od, E.to(state), max_len=max_len, save=True, **E.kw)
        return [t.cpu() for t in (h, last) + lm.scan_grad(E.to(gate), E.to(x), E.to(dh), saved, od, E.to(state), E.to(dlast), max_len=max_len, **E.kw)]

    plain = run(gate, x, dh, state, dlast)
    dirty = [1, 6, 127, 129, dim - 1, dim - 3, dim - 5]
    x[20, 1], dh[100, 6], gate[200, 127], state[0, 129], dlast[0, dim - 1], x[300, dim - 3], gate[5, dim - 5] = inf, -inf, nan, inf, nan, -inf, nan
    got = run(gate, x, dh, state, dlast)
    again = run(gate, x, dh, state, dlast)
    clean = torch.ones(dim, dtype=torch.bool)
    clean[dirty] = False
    for what, a, b, c in zip(('h', 'last', 'dgate', 'dx', 'dstate'), got, plain, again):
        equal(what + ' of the other columns', a[:, clean], b[:, clean])
        equal(what + ' again', a, c)
        assert not a.isfinite().all(), what


def run_all(device, lib_path, path=None):
    E = Env(device, lib_path)
    results = {}
    for name, fn, where in CHECKS:
        if where == 'cpu':
            continue
        print('check', name, flush=True)
        try:
            fn(E)
            torch.cuda.synchronize()
            results[name] = 'ok'
        except Exception:
            results[name] = traceback.format_exc()
            print(results[name], flush=True)
        if path is not None:
            with open(path, 'w') as f:
                json.dump(results, f)
        if 'HIP error' in results[name] or 'hipError' in results[name]:
            break   # (nothing more runs on a GPU that has failed)
    return results


def main(args, device='cuda'):
    done = run_all(device, None, args[0] if args else None)
    bad = [k for k, v in done.items() if v != 'ok']
    due = sum(where != 'cpu' for _, _, where in CHECKS)
    print('%s checks, %d failed' % (len(done) if len(done) == due else '%d of %d' % (len(done), due), len(bad)), flush=True)
    return 1 if not args and (bad or len(done) < due) else 0


if __name__ == '__main__':
    torch.zeros(1, device='cuda')   # torch's HIP runtime first
    sys.exit(main(sys.argv[1:]))
