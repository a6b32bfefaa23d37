"""The operators of a re-ranking language model on torch tensors (C ABI: include/jppgpu_lm.h).

The analysis path scores with the recurrent language model of a model file.  These calls are that chain's operators on the
caller's own tensors, with their gradients, to train a model of one's own and to ask it for scores from a host scorer:

    y = embed(table, ids, scale)                      dtable = embed_grad(dy, ids, vocab, scale)
    h, last = scan(gate, x, offsets, state)           dgate, dx, dstate = scan_grad(gate, x, dh, saved, offsets, state, dlast)
    scores = nce_score(h, table, ids, constant)       loss, dh, dtable = nce_loss(h, table, ids, log_noise, constant, weight)

Tensors live on one GPU; the work is enqueued on torch's current stream of that GPU, nothing waits, and every call may be
captured into a graph.  They are no part of torch's record of a loss: gradients are the calls on the right, and a tensor that
requires one is refused unless torch.no_grad() is on.  Rows may have any stride, columns are contiguous; float32, bfloat16 and
float16 (sums and states are 32-bit).  An id outside the vocabulary names no word: a row of zeros, no gradient, a score of
-inf.  A packed batch is rows and n + 1 int32 offsets, as jppgpu_analyze_batch takes its sentences.

There is no CPU implementation behind this module.  (tests/ pass `lib_path` of the emulator build; test infrastructure.)
"""
import ctypes as C
import functools
import struct

import torch

from .native import JppGpuError, load_library

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}
_pack_matrix = struct.Struct('=QqiI').pack
_pack_ids = struct.Struct('=QiI').pack
_libs = {}


def _lib(path=None):
    lib = _libs.get(path)
    if lib is None:
        lib = load_library(path)
        p, i64, i32, f32, u64 = C.c_void_p, C.c_int64, C.c_int32, C.c_float, C.c_uint64
        mat = C.c_char_p   # a packed jppgpu_lm_matrix / jppgpu_lm_ids, or None
        lib.jppgpu_lm_embed.argtypes = [mat, i64, i64, mat, i64, f32, mat, i32, p]
        lib.jppgpu_lm_embed_grad_workspace.argtypes = [i64, i64, i64, p]
        lib.jppgpu_lm_embed_grad.argtypes = [mat, mat, i64, i64, i64, f32, mat, p, u64, i32, p]
        lib.jppgpu_lm_scan_saved.argtypes = [i64]
        lib.jppgpu_lm_scan_saved.restype = i64
        lib.jppgpu_lm_scan_workspace.argtypes = [i64, i64, i64, i64, p]
        lib.jppgpu_lm_scan.argtypes = [mat, mat, p, i64, i64, i64, i64, mat, mat, mat, p, p, u64, i32, p]
        lib.jppgpu_lm_scan_grad.argtypes = [mat, mat, p, i64, i64, i64, i64, mat, p, mat, mat, mat, mat, mat, p, u64, i32, p]
        lib.jppgpu_lm_nce_score.argtypes = [mat, mat, i64, i64, mat, i64, i64, f32, p, i32, p]
        lib.jppgpu_lm_nce_loss_workspace.argtypes = [i64, i64, i64, i64, p]
        lib.jppgpu_lm_nce_loss.argtypes = [mat, mat, i64, i64, mat, i64, i64, p, f32, p, p, mat, mat, p, u64, i32, p]
        _libs[path] = lib
    return lib


def _raw_stream(index):
    """the current stream's handle (torch.cuda.current_stream builds a Stream object around it first: a microsecond)"""
    get = getattr(torch._C, '_cuda_getCurrentRawStream', None)
    return get(index) if get is not None else torch.cuda.current_stream(index).cuda_stream


def _check(lib, rc):
    if rc:
        raise JppGpuError(lib.jppgpu_last_error().decode())


def _refuse(why):
    raise JppGpuError('jumanpp_amd.lm: ' + why)


def _where(lib_path, first, *others):
    """(device ordinal, stream) of the call; every tensor on the device of the first, none that torch records gradients for"""
    index = first.get_device()
    recorded = torch.is_grad_enabled()
    lost = recorded and first.requires_grad
    for t in others:
        if t is None:
            continue
        if t.get_device() != index:
            _refuse('the tensors are on different devices (%s, %s)' % (first.device, t.device))
        lost = lost or recorded and t.requires_grad
    if lost:
        _refuse('a tensor requires a gradient, which these calls do not record: they have their own (embed_grad, scan_grad, '
                'nce_loss); call them under torch.no_grad()')
    if index < 0:
        if lib_path is None or first.device.type != 'cpu':
            _refuse('the tensors are on %s, not on a GPU' % first.device)
        return 0, None   # (device memory of the emulator build is host memory)
    return index, _raw_stream(index)


def _rows(t, what, n=None, dim=None):
    """the packed jppgpu_lm_matrix of a 2-d tensor (of n x dim, where given)"""
    try:
        rows, cols = t.shape
        stride, step = t.stride()
        code = _TYPES[t.dtype]
    except ValueError:
        _refuse('%s has %d dimensions, not 2' % (what, t.dim()))
    except KeyError:
        _refuse('%s is %s; float32, bfloat16 and float16 are supported' % (what, t.dtype))
    if n is not None and (rows != n or cols != dim):
        _refuse('%s is %s, not (%d, %d)' % (what, tuple(t.shape), n, dim))
    if step != 1 and cols > 1:
        _refuse('the columns of %s are not contiguous' % what)
    # (torch gives a tensor of at most one row any stride)
    return _pack_matrix(t.data_ptr(), stride if rows > 1 else cols, code, 0)


_CLEAR_REST = 0x100   # JPPGPU_LM_CLEAR_REST


def _out(t, dim, flags=0):
    """... of one of our own results"""
    return _pack_matrix(t.data_ptr(), dim, _TYPES[t.dtype] | flags, 0)


def _ids(t, what='ids'):
    size = _ID_BYTES.get(t.dtype)
    if size is None:
        _refuse('%s are %s, not int32 or int64' % (what, t.dtype))
    if not t.is_contiguous():
        _refuse('%s are not contiguous' % what)
    return _pack_ids(t.data_ptr(), size, 0)


def _vector(t, what, n, dtype):
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        _refuse('%s is not a contiguous vector of %d %s' % (what, n, dtype))
    return t.data_ptr()


@functools.lru_cache(maxsize=256)
def _workspace_bytes(lib, name, *sizes):
    need = C.c_uint64()
    _check(lib, getattr(lib, name)(*sizes, C.addressof(need)))
    return need.value


def _workspace(lib, name, sizes, like):
    """(tensor or None, pointer, bytes) of a workspace; torch's allocator keeps it for the stream, or for the graph"""
    need = _workspace_bytes(lib, name, *sizes)
    if need == 0:
        return None, 0, 0
    ws = like.new_empty(need, dtype=torch.uint8)
    return ws, ws.data_ptr(), need


def embed(table, ids, scale=1.0, dtype=None, lib_path=None):
    """scale * table[ids] [n, dim], zeros where an id names no word.  dtype: of the result; the table's, or a 16-bit type from
    a 32-bit table."""
    lib = _lib(lib_path)
    dev, stream = _where(lib_path, table, ids)
    if ids.dim() != 1:
        _refuse('ids have %d dimensions, not 1' % ids.dim())
    rows, idv = _rows(table, 'table'), _ids(ids)
    n, (vocab, dim) = ids.shape[0], table.shape
    if dtype is not None and dtype not in _TYPES:
        _refuse('rows of %s; float32, bfloat16 and float16 are supported' % dtype)
    out = table.new_empty((n, dim), dtype=dtype)
    _check(lib, lib.jppgpu_lm_embed(rows, vocab, dim, idv, n, scale, _out(out, dim), dev, stream))
    return out


def embed_grad(dy, ids, vocab, scale=1.0, lib_path=None):
    """The gradient of embed's table, float32 [vocab, dim], from that of its result: rows summed by word in a fixed order."""
    lib = _lib(lib_path)
    dev, stream = _where(lib_path, dy, ids)
    rows, idv = _rows(dy, 'dy'), _ids(ids)
    n, dim = dy.shape
    if ids.dim() != 1 or ids.shape[0] != n:
        _refuse('ids are %s, dy has %d rows' % (tuple(ids.shape), n))
    ws, wp, wn = _workspace(lib, 'jppgpu_lm_embed_grad_workspace', (n, vocab, dim), dy)
    grad = dy.new_empty((vocab, dim), dtype=torch.float32)
    _check(lib, lib.jppgpu_lm_embed_grad(rows, idv, n, vocab, dim, scale, _out(grad, dim), wp, wn, dev, stream))
    return grad


def _batch(offsets, rows, device):
    """(offsets, their pointer, sentences); without offsets all rows are one sentence"""
    if offsets is None:
        offsets = torch.arange(0, 2, dtype=torch.int32, device=device).mul_(rows)
    if offsets.dtype != torch.int32 or offsets.dim() != 1 or offsets.shape[0] < 1 or not offsets.is_contiguous():
        _refuse('offsets are not a contiguous vector of n + 1 int32')
    return offsets, offsets.data_ptr(), offsets.shape[0] - 1


def scan(gate, x, offsets=None, state=None, max_len=None, save=False, lib_path=None):
    """The gated linear recurrence h_t = a_t h_(t-1) + (1 - a_t) x_t, a = sigmoid(gate), over every sentence of a packed batch
    (offsets None: one sentence), from its row of `state` (float32 [n, dim]; None: zero).  Returns (h, last): h as x, last
    float32 [n, dim] the states behind the sentences; rows of h that belong to no sentence are zero.  One row a
    sentence is the serving step.  max_len: the longest sentence, where the host knows it; it decides how the work is split.
    save=True: (h, last, saved) with what scan_grad needs of the forward pass."""
    lib = _lib(lib_path)
    dev, stream = _where(lib_path, x, gate, offsets, state)
    xv = _rows(x, 'x')
    rows, dim = x.shape
    gv = _rows(gate, 'gate', rows, dim)
    offsets, op, n = _batch(offsets, rows, x.device)
    sv = _rows(state, 'state', n, dim) if state is not None else None
    max_len = max_len or 0
    h = x.new_empty((rows, dim))
    last = x.new_empty((n, dim), dtype=torch.float32)
    saved = x.new_empty((lib.jppgpu_lm_scan_saved(rows), dim), dtype=torch.float32) if save else None
    ws, wp, wn = _workspace(lib, 'jppgpu_lm_scan_workspace', (rows, n, dim, max_len), x)
    _check(lib, lib.jppgpu_lm_scan(gv, xv, op, n, rows, dim, max_len, sv, _out(h, dim, _CLEAR_REST), _out(last, dim),
                                   saved.data_ptr() if save else None, wp, wn, dev, stream))
    return (h, last, saved) if save else (h, last)


def scan_grad(gate, x, dh, saved, offsets=None, state=None, dlast=None, max_len=None, lib_path=None):
    """The gradients (dgate, dx, dstate) of scan's inputs from those of its results, dh and dlast (float32; None: zero).
    gate, x, offsets, state as in the scan(..., save=True) that returned `saved`.  Rows of dgate and dx that belong to no
    sentence are zero."""
    lib = _lib(lib_path)
    dev, stream = _where(lib_path, x, gate, dh, saved, offsets, state, dlast)
    xv = _rows(x, 'x')
    rows, dim = x.shape
    gv, dv = _rows(gate, 'gate', rows, dim), _rows(dh, 'dh', rows, dim)
    offsets, op, n = _batch(offsets, rows, x.device)
    sv = _rows(state, 'state', n, dim) if state is not None else None
    lv = _rows(dlast, 'dlast', n, dim) if dlast is not None else None
    if saved.dtype != torch.float32 or tuple(saved.shape) != (lib.jppgpu_lm_scan_saved(rows), dim) or not saved.is_contiguous():
        _refuse('saved is not what scan(..., save=True) returned for these rows')
    max_len = max_len or 0
    dgate, dx = x.new_empty((rows, dim)), x.new_empty((rows, dim))
    dstate = x.new_empty((n, dim), dtype=torch.float32)
    ws, wp, wn = _workspace(lib, 'jppgpu_lm_scan_workspace', (rows, n, dim, max_len), x)
    _check(lib, lib.jppgpu_lm_scan_grad(gv, xv, op, n, rows, dim, max_len, sv, saved.data_ptr(), dv, lv, _out(dgate, dim, _CLEAR_REST),
                                        _out(dx, dim, _CLEAR_REST), _out(dstate, dim), wp, wn, dev, stream))
    return dgate, dx, dstate


def _candidates(h, table, ids):
    if ids.dim() != 2 or ids.shape[0] != h.shape[0] or ids.shape[1] < 1:
        _refuse('ids are %s, h has %d rows' % (tuple(ids.shape), h.shape[0]))
    if h.shape[1] != table.shape[1]:
        _refuse('h has %d columns, the table %d' % (h.shape[1], table.shape[1]))


def nce_score(h, table, ids, constant, lib_path=None):
    """<h_t, table[ids[t, k]]> - constant, float32 [n, cands]; -inf where the id names no word."""
    lib = _lib(lib_path)
    dev, stream = _where(lib_path, h, table, ids)
    hv, tv, idv = _rows(h, 'h'), _rows(table, 'table'), _ids(ids)
    _candidates(h, table, ids)
    scores = h.new_empty(ids.shape, dtype=torch.float32)
    _check(lib, lib.jppgpu_lm_nce_score(hv, tv, table.shape[0], table.shape[1], idv, ids.shape[0], ids.shape[1], constant,
                                        scores.data_ptr(), dev, stream))
    return scores


def nce_loss(h, table, ids, log_noise, constant, weight=None, grads=True, lib_path=None):
    """The noise-contrastive loss of every token and the gradients of its sum: (loss float32 [n], dh as h, dtable float32
    [vocab, dim]), or the loss alone with grads=False.  ids [n, cands]: the word that follows the token, then the words drawn
    from the noise; log_noise[v] = ln((cands - 1) p(v)), float32 [vocab]; weight: float32 [n] (None: 1).  A token without a
    following word counts nothing, a noise id that names no word is left out."""
    lib = _lib(lib_path)
    dev, stream = _where(lib_path, h, table, ids, log_noise, weight)
    hv, tv, idv = _rows(h, 'h'), _rows(table, 'table'), _ids(ids)
    _candidates(h, table, ids)
    n, cands = ids.shape
    vocab, dim = table.shape
    ln = _vector(log_noise, 'log_noise', vocab, torch.float32)
    wt = _vector(weight, 'weight', n, torch.float32) if weight is not None else None
    loss = h.new_empty(n, dtype=torch.float32)
    if not grads:
        _check(lib, lib.jppgpu_lm_nce_loss(hv, tv, vocab, dim, idv, n, cands, ln, constant, wt, loss.data_ptr(), None, None,
                                           None, 0, dev, stream))
        return loss
    ws, wp, wn = _workspace(lib, 'jppgpu_lm_nce_loss_workspace', (n, cands, vocab, dim), h)
    dh = h.new_empty((n, dim))
    dtable = h.new_empty((vocab, dim), dtype=torch.float32)
    _check(lib, lib.jppgpu_lm_nce_loss(hv, tv, vocab, dim, idv, n, cands, ln, constant, wt, loss.data_ptr(), _out(dh, dim),
                                       _out(dtable, dim), wp, wn, dev, stream))
    return loss, dh, dtable
