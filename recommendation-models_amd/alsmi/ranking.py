"""Ranking a catalogue: item tables in 4 bits, scores changed before the selection, and the
selection itself, on device tensors.

The reference ends at ``predict_all`` (src/als.py:347-364), one user's score for every item.  A
recommender goes on from there: it keeps the item table small (``mx4_quantize``), scores a block of
users against it (``mx4_scores``), takes out what a user has already seen or may not get and
shifts the rest (``adjust_scores``) and keeps the best few (``topk_rows``).  ``ALS.recommend``
runs that chain; the functions here are the same steps for scores from any model.

Every function enqueues on the current stream of its tensors' device and returns without waiting.
Tensors are 2-D with unit stride inside a row (rows may be strided); results carry no gradient.
Arguments that do not fit raise ValueError before anything is launched.
"""
import ctypes
import math

import numpy as np
import torch

from . import _lib

_CODES = {torch.float32: _lib.F32, torch.float64: _lib.F64, torch.float16: _lib.F16,
          torch.bfloat16: _lib.BF16}
_FLOATS = tuple(_CODES)
# A small call is mostly its host time, so what every call does is kept short: the current device and
# the current stream's handle without the objects around them, entry points looked up once.
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device
_entry = {}
_NARROW = (torch.float32, torch.float16, torch.bfloat16)
BLOCK = 32
MAX_K = 1024
MAX_WIDTH = 1 << 20


def _matrix(name, t, dtypes):
    """Row stride of a 2-D tensor of one of `dtypes` with unit stride inside a row."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError('%s must be a 2-D tensor' % name)
    if t.dtype not in dtypes:
        raise ValueError('%s must be one of %s, got %s'
                         % (name, ', '.join(str(d) for d in dtypes), t.dtype))
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError('%s requires a gradient, which this operator does not give; detach it'
                         % name)
    n, m = t.shape
    row, step = t.stride()
    if m > 1 and step != 1:
        raise ValueError('%s must have unit stride inside a row' % name)
    if n > 1:
        if row < m:
            raise ValueError('%s must not have overlapping rows' % name)
        return row
    return m


def _vector(name, t, dtype, size=None):
    if not isinstance(t, torch.Tensor) or t.dim() != 1 or t.dtype != dtype or \
            not t.is_contiguous():
        raise ValueError('%s must be a contiguous 1-D %s tensor' % (name, dtype))
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError('%s requires a gradient, which this operator does not give; detach it'
                         % name)
    if size is not None and t.numel() != size:
        raise ValueError('%s must have %d entries, got %d' % (name, size, t.numel()))


def _device(t, *others):
    """The HIP device that `t` and the other tensors (or None) are on."""
    if not t.is_cuda:
        raise ValueError('tensors must be on a HIP device; there is no CPU fallback')
    device = t.device
    for o in others:
        if o is not None and o.device != device:
            raise ValueError('tensors on %s and on %s in one call' % (device, o.device))
    return device


def _p(t):
    return t.data_ptr() if t is not None else None


def _call(device, name, *args):
    """Enqueue an entry point on the current stream of `device`."""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(_lib.load(), name)
    index = device.index
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = fn(*args, _raw_stream(index))
    if status != 0:
        _lib.check(status, name)


def _span(t):
    """First and last byte address of a tensor with no negative strides."""
    size = sum((n - 1) * step for n, step in zip(t.shape, t.stride())) + 1
    return t.data_ptr(), t.data_ptr() + size * t.element_size()


def _overlap(a, b):
    """Whether two tensors (vectors, or rows of unit stride) share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = _span(a), _span(b)
    if a0 >= b1 or b0 >= a1:
        return False
    # rows the same distance apart may lie beside each other, such as column ranges of one matrix
    apart = {t.stride(0) * t.element_size() for t in (a, b) if t.dim() == 2 and t.shape[0] > 1}
    if len(apart) != 1:
        return True
    apart, off = apart.pop(), b0 - a0
    a_row, b_row = (t.shape[-1] * t.element_size() for t in (a, b))
    return off % apart < a_row or off % apart + b_row > apart


def _result(name, out, shape, dtype, like, *sources):
    """`out` checked, or a new tensor on the device of `like`, and its row stride."""
    if out is None:
        return like.new_empty(shape, dtype=dtype), shape[1]
    ld = _matrix(name, out, (dtype,))
    if tuple(out.shape) != tuple(shape):
        raise ValueError('%s must have shape %s, got %s' % (name, tuple(shape), tuple(out.shape)))
    if any(s is not None and _overlap(out, s) for s in sources):
        raise ValueError('%s must not overlap the operands' % name)
    return out, ld


class Mx4Table(object):
    """Rows held in 4-bit microscaled floating point: `codes` uint8 [n, 16 * nb], two four-bit
    codes a byte, and `scales` uint8 [n, nb], one power of two per block of 32 elements,
    nb = ceil(width / 32); 17 bytes for 32 elements.  ``mx4_quantize`` makes one; the constructor
    takes codes and scales kept elsewhere."""

    def __init__(self, codes, scales, width):
        width = int(width)
        if not 1 <= width <= MAX_WIDTH:
            raise ValueError('width must be between 1 and %d, got %d' % (MAX_WIDTH, width))
        blocks = (width + BLOCK - 1) // BLOCK
        for name, t, cols in (('codes', codes, blocks * 16), ('scales', scales, blocks)):
            if not torch.is_tensor(t) or t.dtype != torch.uint8 or t.dim() != 2 or \
                    t.shape[1] != cols or not t.is_contiguous():
                raise ValueError('%s must be a contiguous uint8 tensor [n, %d]' % (name, cols))
        if codes.shape[0] != scales.shape[0]:
            raise ValueError('codes and scales must have the same number of rows')
        if codes.data_ptr() % 4:
            raise ValueError('codes must be aligned to 4 bytes')
        self.codes, self.scales, self.width = codes, scales, width

    @classmethod
    def _of(cls, codes, scales, width):
        """A table of parts known to fit each other."""
        self = cls.__new__(cls)
        self.codes, self.scales, self.width = codes, scales, width
        return self

    @property
    def shape(self):
        return (self.codes.shape[0], self.width)

    @property
    def device(self):
        return self.codes.device

    @property
    def nbytes(self):
        return self.codes.numel() + self.scales.numel()

    def __len__(self):
        return self.codes.shape[0]


def mx4_quantize(x):
    """The rows of `x` (float32, float64, float16 or bfloat16) as an ``Mx4Table``.

    Each block of 32 elements of a row is scaled by 2^(floor(log2 max|x|) - 2), its elements
    rounded to the nearest of 0, 1/2, 1, 3/2, 2, 3, 4, 6 with a sign (ties to the even code,
    larger ones to 6).  A block with an infinity or a NaN reads back as NaN."""
    ld = _matrix('x', x, _FLOATS)
    n, width = x.shape
    if not 1 <= width <= MAX_WIDTH:
        raise ValueError('x must have between 1 and %d columns, got %d' % (MAX_WIDTH, width))
    device = _device(x)
    blocks = (width + BLOCK - 1) // BLOCK
    codes = x.new_empty((n, blocks * 16), dtype=torch.uint8)
    scales = x.new_empty((n, blocks), dtype=torch.uint8)
    _call(device, 'alsmi_mx4_quantize', _CODES[x.dtype], n, width, _p(x), ld, _p(codes),
          _p(scales))
    return Mx4Table._of(codes, scales, width)


def mx4_dequantize(table, dtype=torch.float32, rows=None, out=None):
    """The values `table` stands for, [n, width] of `dtype`; with `rows` (int32) those rows in
    that order, NaN for a row the table does not have.  Exact but for float16, and for elements of
    2^128 or more, which are infinities in float32 and bfloat16."""
    if not isinstance(table, Mx4Table):
        raise ValueError('table must be an Mx4Table')
    if dtype not in _CODES:
        raise ValueError('dtype must be one of %s' % ', '.join(str(d) for d in _FLOATS))
    if rows is not None:
        _vector('rows', rows, torch.int32)
    n = len(table) if rows is None else rows.numel()
    out, ld = _result('out', out, (n, table.width), dtype, table.codes, table.codes, table.scales,
                      rows)
    device = _device(table.codes, table.scales, rows, out)
    _call(device, 'alsmi_mx4_dequantize', _CODES[dtype], n, _p(rows), len(table), table.width,
          _p(table.codes), _p(table.scales), _p(out), ld)
    return out


def mx4_scores(a, table, rows=None, out_dtype=None, out=None):
    """``a @ table.T``, [m, n] with n = len(table): the scores of the rows of `a` against every row
    of `table`.

    `a` is a float32, float16 or bfloat16 tensor [m, width] or another ``Mx4Table`` of the same
    width.  Products are exact and sums float32, except that of a float32 activation bits below
    2^-133 are cut off and that beside float activations a table element of 2^128 or more (scale
    bytes 253 and 254, from float64 rows) counts as an infinity.  With `rows` (int32) the rows of `a` with those
    ids, NaN for one it does not have.  The result has `out_dtype` (float32, float16 or
    bfloat16), by default that of `a`, float32 for a table."""
    if not isinstance(table, Mx4Table):
        raise ValueError('table must be an Mx4Table')
    held = isinstance(a, Mx4Table)
    if held:
        ld, code, data, a_scales = a.width, _lib.MX4, a.codes, a.scales
    else:
        ld, data, a_scales = _matrix('a', a, _NARROW), a, None
        code = _CODES[a.dtype]
    codes, scales, width = table.codes, table.scales, table.width
    n, (n_rows, a_width) = codes.shape[0], a.shape
    if a_width != width:
        raise ValueError('a has %d columns, the table %d' % (a_width, width))
    if rows is not None:
        _vector('rows', rows, torch.int32)
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else (torch.float32 if held else a.dtype)
    if out_dtype not in _NARROW:
        raise ValueError('out_dtype must be one of %s' % ', '.join(str(d) for d in _NARROW))
    m = n_rows if rows is None else rows.numel()
    if m and n_rows == 0:
        raise ValueError('rows of an empty a')
    out, ldo = _result('out', out, (m, n), out_dtype, codes, data, a_scales, rows, codes, scales)
    device = _device(codes, scales, data, a_scales, rows, out)
    size = _lib.load().alsmi_mx4_scores_workspace_bytes(code, m, n, width)
    ws = codes.new_empty(size) if size else None
    _call(device, 'alsmi_mx4_scores', code, m, _p(rows), n_rows, data.data_ptr(), ld, _p(a_scales), n,
          width, codes.data_ptr(), scales.data_ptr(), _CODES[out_dtype], out.data_ptr(), ldo, _p(ws))
    return out


def pack_mask(allowed):
    """Host array of truth values [items] or [masks, items] -> the bit words ``adjust_scores``
    takes, int32 [masks, ceil(items / 32)]: item i is bit i % 32 of word i // 32."""
    allowed = np.atleast_2d(np.asarray(allowed, dtype=bool))
    if allowed.ndim != 2:
        raise ValueError('allowed must have one or two dimensions')
    n, m = allowed.shape
    words = (m + 31) // 32
    data = np.zeros((n, words * 4), dtype=np.uint8)
    packed = np.packbits(allowed, axis=1, bitorder='little')
    data[:, :packed.shape[1]] = packed
    return data.view('<u4').astype(np.uint32).view(np.int32)


def _lists(name, lists, n_values):
    """(ptr, ids[, values]) of ragged lists, checked; the number of lists."""
    if not isinstance(lists, (tuple, list)) or len(lists) != 2 + n_values:
        raise ValueError('%s must be a tuple of %d tensors' % (name, 2 + n_values))
    _vector('%s pointers' % name, lists[0], torch.int64)
    _vector('%s ids' % name, lists[1], torch.int32)
    if n_values:
        _vector('%s values' % name, lists[2], torch.float32, lists[1].numel())
    if lists[0].numel() < 1:
        raise ValueError('%s pointers must have one entry more than there are lists' % name)
    return lists[0].numel() - 1


def _penalty(name, value, n_rows, args, kept):
    """A penalty in the argument block, as a per-row array or one number."""
    if isinstance(value, torch.Tensor):
        _vector(name, value, torch.float32, n_rows)
        kept.append(value)
        setattr(args, name, value.data_ptr())
        return
    value = float(value)
    if math.isnan(value) or (name == 'repetition' and not (0 < value < math.inf)):
        raise ValueError('%s must be %s, got %r' % (
            name, 'a positive number' if name == 'repetition' else 'a number', value))
    setattr(args, name + '_value', value)


def adjust_scores(scores, history=None, history_rows=None, repetition=None, frequency=None,
                  presence=None, exclude=False, item_bias=None, row_bias=None, mask=None,
                  mask_rows=None, out=None):
    """Change score rows [n, items] (float32, float64, float16, bfloat16) before a selection.

    For row r and item i, with c the number of times i occurs in the row's history:

        c > 0:  x = s / repetition if s > 0 else s * repetition, then
                x -= frequency * c + presence
        x += item_bias[i];  x += the last value given for i in the row's `row_bias`
        x = -inf where the row's mask has no bit i, or where c > 0 with `exclude`

    worked in float32 (float64 for float64 scores) and rounded once.

    history       (ptr int64 [lists + 1], ids int32): list l is ids[ptr[l]:ptr[l + 1]], in any
                  order, ids may repeat; ids outside the items are skipped (padding).  Row r has
                  list r, or list history_rows[r] (int32 [n]; none where that does not exist).
    repetition, frequency, presence
                  numbers or float32 tensors [n]; repetition > 0.  Defaults 1, 0, 0.
    item_bias     float32 [items]; float64 too for float64 scores.
    row_bias      (ptr int64 [n + 1], ids int32, values float32), lists as in `history`.
    mask          int32 [masks, ceil(items / 32)], see ``pack_mask``; row r has mask r (a single mask
                  serves every row), or mask mask_rows[r] (int32 [n]): a negative id is no mask, one
                  past the last leaves the row nothing.
    out           a tensor like `scores`, or `scores` itself (or a view of just its elements); new
                  by default."""
    ld = _matrix('scores', scores, _FLOATS)
    n, m = scores.shape
    args = _lib.Adjust()
    args.n_rows, args.n_items, args.ld_scores = n, m, ld
    args.repetition_value = 1.0
    kept = []  # every tensor the call reads beside the scores
    if history is not None:
        lists = _lists('history', history, 0)
        kept += history
        args.history_ptr, args.history_ids = history[0].data_ptr(), history[1].data_ptr()
        args.n_history, args.n_history_rows = history[1].numel(), lists
        if history_rows is not None:
            _vector('history_rows', history_rows, torch.int32, n)
            kept.append(history_rows)
            args.history_rows = history_rows.data_ptr()
        elif lists != n:
            raise ValueError('history has %d lists for %d rows' % (lists, n))
        if exclude:
            args.exclude = 1
    elif history_rows is not None or exclude:
        raise ValueError('history_rows and exclude need a history')
    for name, value in (('repetition', repetition), ('frequency', frequency),
                        ('presence', presence)):
        if value is not None:
            if history is None or exclude:
                raise ValueError('%s needs a history that is not excluded' % name)
            _penalty(name, value, n, args, kept)
    if item_bias is not None:
        wide = torch.float32
        if scores.dtype is torch.float64 and getattr(item_bias, 'dtype', None) is torch.float64:
            wide, args.item_bias_dtype = torch.float64, _lib.F64
        _vector('item_bias', item_bias, wide, m)
        kept.append(item_bias)
        args.item_bias = item_bias.data_ptr()
    if row_bias is not None:
        if _lists('row_bias', row_bias, 1) != n:
            raise ValueError('row_bias must have one list for each of the %d rows' % n)
        kept += row_bias
        args.bias_ptr, args.bias_ids = row_bias[0].data_ptr(), row_bias[1].data_ptr()
        args.bias_values, args.n_bias = row_bias[2].data_ptr(), row_bias[1].numel()
    if mask is not None:
        if not isinstance(mask, torch.Tensor) or mask.dtype != torch.int32 or mask.dim() != 2 or \
                mask.shape[1] != (m + 31) // 32 or not mask.is_contiguous():
            raise ValueError('mask must be a contiguous int32 tensor [masks, %d]'
                             % ((m + 31) // 32))
        if mask.shape[0] == 0:
            raise ValueError('mask has no rows')
        kept.append(mask)
        args.mask, args.n_masks = mask.data_ptr(), mask.shape[0]
        if mask_rows is not None:
            _vector('mask_rows', mask_rows, torch.int32, n)
            kept.append(mask_rows)
            args.mask_rows = mask_rows.data_ptr()
        elif mask.shape[0] not in (1, n):
            raise ValueError('mask must have one row or one for each of the %d rows' % n)
    elif mask_rows is not None:
        raise ValueError('mask_rows needs a mask')
    if out is None:
        out, args.ld_out = scores.new_empty((n, m)), m
    elif out is not scores:
        same = isinstance(out, torch.Tensor) and out.data_ptr() == scores.data_ptr() and \
            out.shape == scores.shape and out.stride() == scores.stride()
        out, args.ld_out = _result('out', out, (n, m), scores.dtype, scores,
                                   *(kept if same else [scores] + kept))
    else:
        args.ld_out = ld
        if any(_overlap(out, t) for t in kept):
            raise ValueError('out must not overlap the operands')
    device = _device(scores, out, *kept)
    _call(device, 'alsmi_adjust_scores', _CODES[scores.dtype], ctypes.byref(args),
          scores.data_ptr(), out.data_ptr())
    return out


def topk_rows(scores, k, max_workspace_bytes=1 << 30):
    """The k largest scores of every row of `scores` (float32, float64, float16, bfloat16):
    (items int32 [n, k], scores [n, k]), best first, equal scores by the smaller item id.
    1 <= k <= min(1024, items).  NaN and -0.0 rank as in ``alsmi_topk_items``."""
    ld = _matrix('scores', scores, _FLOATS)
    n, m = scores.shape
    k = int(k)
    if not 1 <= k <= min(MAX_K, m):
        raise ValueError('k must be between 1 and min(%d, number of items), got %r' % (MAX_K, k))
    device = _device(scores)
    code = _CODES[scores.dtype]
    items = scores.new_empty((n, k), dtype=torch.int32)
    best = scores.new_empty((n, k))
    if n == 0:
        return items, best
    need = _lib.load().alsmi_topk_rows_workspace_bytes
    batch = n
    size = need(code, n, m, k)
    if size > max_workspace_bytes and n > 1:
        batch = max(1, min(n, max_workspace_bytes // need(code, 1, m, k)))
        size = need(code, batch, m, k)
    ws = scores.new_empty(size, dtype=torch.uint8)
    for lo in range(0, n, batch):
        hi = min(n, lo + batch)
        part = scores if batch == n else scores[lo:hi]
        _call(device, 'alsmi_topk_rows', code, hi - lo, m, _p(part), ld, k,
              _p(items if batch == n else items[lo:hi]), _p(best if batch == n else best[lo:hi]),
              _p(ws))
    return items, best
