"""The ranking operators' refusals and host-side parts (no GPU): the functions of alsmi.ranking reject
what does not fit before anything is launched, and so do the entry points of the C ABI."""
import ctypes

import numpy as np
import pytest
import torch

from alsmi import _lib, ranking as rk
from oracle import ranking_oracle as ro


def table(n=4, width=40):
    codes, scales = ro.mx4_quantize(np.random.default_rng(0).standard_normal((n, width)))
    return rk.Mx4Table(torch.from_numpy(codes), torch.from_numpy(scales), width)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


def i64(*v):
    return torch.tensor(v, dtype=torch.int64)


def f32(*v):
    return torch.tensor(v, dtype=torch.float32)


X = torch.zeros(3, 8)
HIST = (i64(0, 1, 1, 2), i32(0, 1))

REFUSED = {
    'quantize: 1-D': (lambda: rk.mx4_quantize(torch.zeros(8)), '2-D'),
    'quantize: integers': (lambda: rk.mx4_quantize(torch.zeros(2, 8, dtype=torch.int32)), 'one of'),
    'quantize: no columns': (lambda: rk.mx4_quantize(torch.zeros(2, 0)), 'columns'),
    'quantize: columns': (lambda: rk.mx4_quantize(torch.zeros(8, 2).t()), 'unit stride'),
    'quantize: expanded': (lambda: rk.mx4_quantize(torch.zeros(1, 8).expand(3, 8)), 'overlapping'),
    'quantize: gradient': (lambda: rk.mx4_quantize(torch.zeros(2, 8, requires_grad=True)), 'gradient'),
    'quantize: host': (lambda: rk.mx4_quantize(X), 'HIP device'),
    'table: codes': (lambda: rk.Mx4Table(torch.zeros(2, 16, dtype=torch.uint8),
                                         torch.zeros(2, 2, dtype=torch.uint8), 40), 'codes'),
    'table: scales': (lambda: rk.Mx4Table(torch.zeros(2, 32, dtype=torch.uint8),
                                          torch.zeros(2, 1, dtype=torch.uint8), 40), 'scales'),
    'table: rows': (lambda: rk.Mx4Table(torch.zeros(2, 32, dtype=torch.uint8),
                                        torch.zeros(3, 2, dtype=torch.uint8), 40), 'number of rows'),
    'table: width': (lambda: rk.Mx4Table(torch.zeros(2, 0, dtype=torch.uint8),
                                         torch.zeros(2, 0, dtype=torch.uint8), 0), 'width'),
    'table: alignment': (lambda: rk.Mx4Table(torch.zeros(33, dtype=torch.uint8)[1:].view(2, 16),
                                             torch.zeros(2, 1, dtype=torch.uint8), 32), 'aligned'),
    'dequantize: no table': (lambda: rk.mx4_dequantize(X), 'Mx4Table'),
    'dequantize: type': (lambda: rk.mx4_dequantize(table(), torch.int32), 'dtype'),
    'dequantize: rows': (lambda: rk.mx4_dequantize(table(), rows=i64(0)), 'rows'),
    'dequantize: out': (lambda: rk.mx4_dequantize(table(), out=torch.zeros(4, 41)), 'shape'),
    'dequantize: host': (lambda: rk.mx4_dequantize(table()), 'HIP device'),
    'scores: width': (lambda: rk.mx4_scores(torch.zeros(2, 39), table()), 'columns'),
    'scores: fp64': (lambda: rk.mx4_scores(torch.zeros(2, 40, dtype=torch.float64), table()), 'one of'),
    'scores: out type': (lambda: rk.mx4_scores(torch.zeros(2, 40), table(),
                                               out_dtype=torch.float64), 'out_dtype'),
    'scores: out shape': (lambda: rk.mx4_scores(torch.zeros(2, 40), table(),
                                                out=torch.zeros(2, 5)), 'shape'),
    'scores: rows of nothing': (lambda: rk.mx4_scores(torch.zeros(0, 40), table(), rows=i32(0)), 'empty'),
    'scores: rows type': (lambda: rk.mx4_scores(torch.zeros(2, 40), table(), rows=i64(0)), 'rows'),
    'scores: no table': (lambda: rk.mx4_scores(torch.zeros(2, 40), torch.zeros(4, 40)), 'Mx4Table'),
    'scores: host': (lambda: rk.mx4_scores(torch.zeros(2, 40), table()), 'HIP device'),
    'adjust: type': (lambda: rk.adjust_scores(X.to(torch.int32)), 'one of'),
    'adjust: history type': (lambda: rk.adjust_scores(X, history=(i32(0, 0, 0, 0), i32(0))), 'pointers'),
    'adjust: history ids': (lambda: rk.adjust_scores(X, history=(i64(0, 0, 0, 0), i64(0))), 'ids'),
    'adjust: history shape': (lambda: rk.adjust_scores(X, history=HIST[0]), 'tuple'),
    'adjust: lists': (lambda: rk.adjust_scores(X, history=(i64(0, 1), i32(0))), 'lists'),
    'adjust: no pointers': (lambda: rk.adjust_scores(X, history=(i64(), i32()),
                                                     history_rows=i32(0, 0, 0)), 'pointers'),
    'adjust: history rows': (lambda: rk.adjust_scores(X, history=HIST, history_rows=i32(0)), 'history_rows'),
    'adjust: rows without lists': (lambda: rk.adjust_scores(X, history_rows=i32(0, 0, 0)), 'need a history'),
    'adjust: exclude nothing': (lambda: rk.adjust_scores(X, exclude=True), 'need a history'),
    'adjust: penalty': (lambda: rk.adjust_scores(X, presence=1.0), 'needs a history'),
    'adjust: excluded penalty': (lambda: rk.adjust_scores(X, history=HIST, exclude=True,
                                                          frequency=1.0), 'needs a history'),
    'adjust: repetition': (lambda: rk.adjust_scores(X, history=HIST, repetition=0.0), 'positive'),
    'adjust: NaN': (lambda: rk.adjust_scores(X, history=HIST, presence=float('nan')), 'a number'),
    'adjust: penalty size': (lambda: rk.adjust_scores(X, history=HIST, frequency=f32(1.0)), 'entries'),
    'adjust: bias size': (lambda: rk.adjust_scores(X, item_bias=f32(1.0)), 'entries'),
    'adjust: row bias lists': (lambda: rk.adjust_scores(X, row_bias=(i64(0, 1), i32(0), f32(1))), 'row_bias'),
    'adjust: row bias values': (lambda: rk.adjust_scores(X, row_bias=(i64(0, 1, 1, 1), i32(0), f32(1, 2))),
                                'entries'),
    'adjust: mask words': (lambda: rk.adjust_scores(X, mask=torch.zeros(3, 2, dtype=torch.int32)), 'mask'),
    'adjust: mask rows': (lambda: rk.adjust_scores(X, mask=torch.zeros(2, 1, dtype=torch.int32)), 'one row'),
    'adjust: no masks': (lambda: rk.adjust_scores(X, mask=torch.zeros(0, 1, dtype=torch.int32),
                                                  mask_rows=i32(0, 0, 0)), 'no rows'),
    'adjust: rows without mask': (lambda: rk.adjust_scores(X, mask_rows=i32(0, 0, 0)), 'needs a mask'),
    'adjust: out type': (lambda: rk.adjust_scores(X, out=X.to(torch.float16)), 'out'),
    'adjust: out overlaps': (lambda: rk.adjust_scores(torch.zeros(40)[:24].view(3, 8),
                                                      out=X), 'HIP device'),
    'adjust: host': (lambda: rk.adjust_scores(X), 'HIP device'),
    'topk: k = 0': (lambda: rk.topk_rows(X, 0), 'k must'),
    'topk: k': (lambda: rk.topk_rows(X, 9), 'k must'),
    'topk: k > 1024': (lambda: rk.topk_rows(torch.zeros(1, 2000), 1025), 'k must'),
    'topk: type': (lambda: rk.topk_rows(X.to(torch.int64), 1), 'one of'),
    'topk: host': (lambda: rk.topk_rows(X, 1), 'HIP device'),
}


@pytest.mark.parametrize('name', sorted(REFUSED))
def test_refused(name):
    call, match = REFUSED[name]
    with pytest.raises(ValueError, match=match):
        call()


def test_overlapping_output_is_refused():
    base = torch.zeros(64)
    with pytest.raises(ValueError, match='overlap'):
        rk.adjust_scores(base[:24].view(3, 8), out=base[8:32].view(3, 8))
    t = table()
    with pytest.raises(ValueError, match='overlap'):
        a = base[:40].view(1, 40)
        rk.mx4_scores(a, t, out=base[:4].view(1, 4))


def test_pack_mask():
    rng = np.random.default_rng(1)
    for n, m in ((1, 1), (3, 31), (2, 32), (4, 33), (2, 100)):
        allowed = rng.random((n, m)) < 0.5
        words = rk.pack_mask(allowed)
        assert words.dtype == np.int32 and words.shape == (n, (m + 31) // 32)
        bit = np.arange(m)
        assert (((words[:, bit // 32] >> (bit % 32)) & 1).astype(bool) == allowed).all()
        # nothing set behind the last item
        last = words[:, -1].view(np.uint32) >> np.uint32((m - 1) % 32)
        assert (last <= 1).all()


def test_c_entry_points_refuse():
    """Status -1 and a message naming the call, for every argument that the kernels rely on."""
    lib = _lib.load()
    buf = (ctypes.c_double * 64)()
    p = ctypes.cast(buf, ctypes.c_void_p)
    odd = ctypes.c_void_p(p.value + 1)

    def refused(name, *args):
        assert getattr(lib, name)(*args) == -1
        assert name.encode() in lib.alsmi_last_error()

    q = 'alsmi_mx4_quantize'
    refused(q, 4, 1, 8, p, 8, p, p, None)
    refused(q, 0, -1, 8, p, 8, p, p, None)
    refused(q, 0, 1, 0, p, 8, p, p, None)
    refused(q, 0, 1, (1 << 20) + 1, p, 8, p, p, None)
    refused(q, 0, 2, 8, p, 7, p, p, None)
    refused(q, 0, 1, 8, None, 8, p, p, None)
    refused(q, 0, 1, 8, p, 8, odd, p, None)
    assert lib.alsmi_mx4_quantize(0, 0, 8, None, 8, None, None, None) == 0
    d = 'alsmi_mx4_dequantize'
    refused(d, 4, 1, None, 1, 8, p, p, p, 8, None)
    refused(d, 0, 2, None, 1, 8, p, p, p, 8, None)
    refused(d, 0, 2, None, 2, 8, p, p, p, 7, None)
    refused(d, 0, 1, None, 1, 0, p, p, p, 8, None)
    refused(d, 0, 1, None, 1, 8, odd, p, p, 8, None)
    refused(d, 0, 1, None, 1, 8, p, p, None, 8, None)
    s = 'alsmi_mx4_scores'
    refused(s, 1, 1, None, 1, p, 8, None, 1, 8, p, p, 0, p, 1, None, None)
    refused(s, 0, 1, None, 1, p, 8, None, 1, 8, p, p, 1, p, 1, None, None)
    refused(s, 0, 2, None, 1, p, 8, None, 1, 8, p, p, 0, p, 1, None, None)
    refused(s, 0, 1, p, 0, p, 8, None, 1, 8, p, p, 0, p, 1, None, None)
    refused(s, 0, 2, None, 2, p, 7, None, 1, 8, p, p, 0, p, 1, None, None)
    refused(s, 0, 2, None, 2, p, 8, None, 2, 8, p, p, 0, p, 1, None, None)
    refused(s, 4, 1, None, 1, p, 8, None, 1, 8, p, p, 0, p, 1, None, None)
    refused(s, 4, 1, None, 1, odd, 8, p, 1, 8, p, p, 0, p, 1, None, None)
    refused(s, 0, 1, None, 1, p, 8, None, 1, 8, odd, p, 0, p, 1, None, None)
    assert lib.alsmi_mx4_scores_workspace_bytes(0, 16, 1000, 64) == 0
    need = lib.alsmi_mx4_scores_workspace_bytes(0, 128, 16384, 640)
    assert need == 128 * 640 * 2 * 3
    refused(s, 0, 128, None, 128, p, 640, None, 16384, 640, p, p, 0, p, 16384, None, None)
    assert lib.alsmi_mx4_scores(0, 0, None, 0, None, 8, None, 5, 8, None, None, 0, None, 5, None, None) == 0

    def adjust(dtype=0, scores=p, out=p, **fields):
        a = _lib.Adjust(n_rows=2, n_items=8, ld_scores=8, ld_out=8, repetition_value=1.0)
        for name, value in fields.items():
            setattr(a, name, value)
        return lib.alsmi_adjust_scores(dtype, ctypes.byref(a), scores, out, None)

    for bad in (dict(dtype=4), dict(scores=None), dict(out=None), dict(n_rows=-1), dict(ld_out=7),
                dict(ld_scores=7), dict(history_ptr=p, n_history=1, n_history_rows=2),
                dict(history_ptr=p, n_history=1, history_ids=p, n_history_rows=1),
                dict(history_ptr=p, n_history=-1, history_ids=p, n_history_rows=2),
                dict(bias_ptr=p, n_bias=1, bias_ids=p), dict(bias_ptr=p, n_bias=1, bias_values=p),
                dict(mask=p, n_masks=0)):
        assert adjust(**bad) == -1, bad
        assert b'alsmi_adjust_scores' in lib.alsmi_last_error()
    assert lib.alsmi_adjust_scores(0, None, p, p, None) == -1
    assert adjust(n_rows=0) == 0
    t = 'alsmi_topk_rows'
    refused(t, 4, 1, 8, p, 8, 1, p, p, p, None)
    refused(t, 0, 1, 8, p, 8, 0, p, p, p, None)
    refused(t, 0, 1, 8, p, 8, 9, p, p, p, None)
    refused(t, 0, 2, 8, p, 7, 1, p, p, p, None)
    refused(t, 0, 1, 8, None, 8, 1, p, p, p, None)
    refused(t, 0, 1, 8, p, 8, 1, p, p, ctypes.c_void_p(p.value + 8 if p.value % 16 == 0 else p.value),
            None)
    assert lib.alsmi_topk_rows_workspace_bytes(9, 1, 8, 1) == 0
    assert lib.alsmi_topk_rows_workspace_bytes(0, 1, 8, 1) > 0
    refused('alsmi_score_items', 2, 4, 1, p, p, p, 1, p, p, None)
    refused('alsmi_score_items', 0, 129, 1, p, p, p, 1, p, p, None)
    refused('alsmi_score_items', 0, 4, 1, None, p, p, 1, p, p, None)


def test_recommend_refuses():
    from alsmi import ALS
    als = ALS(rank=3)
    als.user_feats, als.item_feats = np.ones((3, 4)), np.ones((3, 5))
    for kw, error in ((dict(catalogue='mx3'), ValueError), (dict(item_bias=np.zeros(4)), ValueError),
                      (dict(allowed=np.ones(4)), ValueError), (dict(exclude_seen=True), ValueError),
                      (dict(allowed=np.ones((3, 5))), ValueError)):
        with pytest.raises(error):
            als.recommend([0, 1], k=2, **kw)
    with pytest.raises(IndexError):
        als.recommend([4], k=2, exclude_seen=True)


def test_output_over_any_operand_is_refused():
    flat = torch.zeros(4096, dtype=torch.uint8)
    ids = flat[:8].view(torch.int32)
    t = rk.Mx4Table(torch.zeros(2, 32, dtype=torch.uint8), flat[64:68].view(2, 2), 40)
    over = lambda n: flat[:16 * n * 4].view(torch.float32)
    with pytest.raises(ValueError, match='overlap'):
        rk.mx4_dequantize(t, rows=ids, out=over(5).view(2, 40))
    with pytest.raises(ValueError, match='overlap'):
        rk.mx4_scores(torch.zeros(2, 40), t, out=flat[64:80].view(torch.float32).view(2, 2))
    with pytest.raises(ValueError, match='overlap'):
        rk.mx4_scores(torch.zeros(2, 40), t, rows=ids, out=flat[:16].view(torch.float32).view(2, 2))
    with pytest.raises(ValueError, match='overlap'):
        rk.adjust_scores(torch.zeros(1, 4), item_bias=flat[:16].view(torch.float32),
                         out=flat[8:24].view(torch.float32).view(1, 4))


def test_score_items_refuses():
    from alsmi import device as dev
    U, V = torch.zeros(5, 16), torch.zeros(7, 16)
    users = torch.zeros(4, dtype=torch.int32)
    for bad in ((users.long(), U, V), (users[::2], U, V), (users, U, V.double())):
        with pytest.raises(ValueError):
            dev.score_items(3, *bad)
    with pytest.raises(ValueError):
        dev.score_items(3, users, U, V, out=torch.zeros(4, 8))


def test_workspaces_serve_smaller_calls():
    """A caller sizes a workspace for its largest call."""
    from alsmi import _lib
    lib = _lib.load()
    rng = np.random.default_rng(5)
    log = lambda top: int(np.exp(rng.random() * np.log(top)))
    for _ in range(3000):
        n, m, k = log(5000000), 1 + log(3000000), 1 + log(1023)
        code = int(rng.integers(0, 4))
        most = lib.alsmi_topk_rows_workspace_bytes(code, n, m, k)
        assert most <= 2 * 1024 * 1024 * 16 + 16
        assert lib.alsmi_topk_rows_workspace_bytes(code, log(n), m, k) <= most
        assert lib.alsmi_topk_rows_workspace_bytes(code, n, log(m), k) <= most
        assert lib.alsmi_topk_rows_workspace_bytes(code, n, m, log(k)) <= most
        rows, width = log(20000), 1 + log(100000)
        code = int(rng.choice([_lib.F32, _lib.F16, _lib.BF16, _lib.MX4]))
        most = lib.alsmi_mx4_scores_workspace_bytes(code, rows, m, width)
        assert most <= 1 << 28
        for other in ((log(rows), m, width), (rows, log(m), width), (rows, m, log(width))):
            assert lib.alsmi_mx4_scores_workspace_bytes(code, *other) <= most


BAD_TABLES = {
    'bf16': (lambda u, U, V: (u, U.bfloat16(), V.bfloat16()), 'float32 or float64'),
    'fp16': (lambda u, U, V: (u, U.half(), V.half()), 'float32 or float64'),
    'integers': (lambda u, U, V: (u, U.int(), V.int()), 'float32 or float64'),
    'two types': (lambda u, U, V: (u, U, V.double()), 'share a dtype'),
    'the rank alone': (lambda u, U, V: (u, U[:, :3], V), 'contiguous'),
    'items: the rank alone': (lambda u, U, V: (u, U, V[:, :3].contiguous()), 'contiguous'),
    'another rank': (lambda u, U, V: (u, torch.zeros(5, 32), torch.zeros(7, 32)), 'contiguous'),
    'every other row': (lambda u, U, V: (u, U[::2], V), 'contiguous'),
    'columns': (lambda u, U, V: (u, U, torch.zeros(16, 7).t()), 'contiguous'),
    '1-D': (lambda u, U, V: (u, U.view(-1), V), 'contiguous'),
    'user type': (lambda u, U, V: (u.long(), U, V), 'users'),
    'every other user': (lambda u, U, V: (u[::2], U, V), 'users'),
    'host': (lambda u, U, V: (u, U, V), 'HIP device'),
}


@pytest.mark.parametrize('name', sorted(BAD_TABLES))
def test_tables_that_the_kernels_would_misread_are_refused(name):
    """The kernels take whole padded rows of fp32 or fp64, one behind the other: 16-bit tables would be
    read (and scores written) past their ends, narrower ones at wrong offsets."""
    from alsmi import device as dev
    make, match = BAD_TABLES[name]
    users, U, V = make(torch.zeros(4, dtype=torch.int32), torch.zeros(5, 16), torch.zeros(7, 16))
    with pytest.raises(ValueError, match=match):
        dev.score_items(3, users, U, V)
    with pytest.raises(ValueError, match=match):
        dev.topk_items(3, users, U, V, 2)


def test_score_rows_refuses():
    lib = _lib.load()
    p = ctypes.cast((ctypes.c_double * 64)(), ctypes.c_void_p)
    for bad in ((2, 4, 1, p, 1, p, p, 1, p, p), (0, 129, 1, p, 1, p, p, 1, p, p),
                (0, 4, 1, None, 1, p, p, 1, p, p), (0, 4, 1, p, 0, p, p, 1, p, p),
                (0, 4, 1, p, 1, p, p, -1, p, p), (0, 4, 1, p, 1, p, p, 1, p, None)):
        assert lib.alsmi_score_rows(*bad, None) == -1
        assert b'alsmi_score_rows' in lib.alsmi_last_error()
    assert lib.alsmi_score_rows(0, 4, 0, None, 0, None, None, 5, None, None, None) == 0


def test_item_bias_type_follows_the_scores():
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        with pytest.raises(ValueError, match='item_bias must be'):
            rk.adjust_scores(X.to(dtype), item_bias=torch.zeros(8, dtype=torch.float64))
    with pytest.raises(ValueError, match='entries'):
        rk.adjust_scores(X.double(), item_bias=torch.zeros(7, dtype=torch.float64))
    with pytest.raises(ValueError, match='HIP device'):
        rk.adjust_scores(X.double(), item_bias=torch.zeros(8, dtype=torch.float64))
    lib = _lib.load()
    p = ctypes.cast((ctypes.c_double * 64)(), ctypes.c_void_p)
    for dtype, bias in ((_lib.F32, _lib.F64), (_lib.BF16, _lib.F64), (_lib.F64, _lib.F16), (_lib.F64, -1)):
        a = _lib.Adjust(n_rows=2, n_items=8, ld_scores=8, ld_out=8, repetition_value=1.0, item_bias=p,
                        item_bias_dtype=bias)
        assert lib.alsmi_adjust_scores(dtype, ctypes.byref(a), p, p, None) == -1
        assert b'item bias' in lib.alsmi_last_error()


def test_outputs_beside_and_upon_the_operands():
    """Column ranges of one matrix share its span and no element; a view of the scores is the scores.
    Against the sets of addresses."""
    def cells(t):
        rows = t if t.dim() == 2 else t[None]
        size = t.element_size()
        return {rows[i, j].data_ptr() + b for i in range(rows.shape[0]) for j in range(rows.shape[1])
                for b in range(size)}
    rng = np.random.default_rng(2)
    base = torch.zeros(4000, dtype=torch.uint8)
    seen = set()
    for _ in range(3000):
        ts = []
        for _ in range(2):
            dtype = [torch.float32, torch.float16, torch.uint8][rng.integers(3)]
            flat = base.view(dtype)
            n, m, extra = (int(rng.integers(1, 6)) for _ in range(3))
            ld = int(rng.choice([16, 20, m + extra])) // (4 if rng.random() < 0.3 else 1)
            ld = max(ld, m)
            at = int(rng.integers(0, 40))
            ts.append(flat[at:at + n * ld].view(n, ld)[:, :m] if rng.random() < 0.8
                      else flat[at:at + m])
        meet = bool(cells(ts[0]) & cells(ts[1]))
        apart = {t.stride(0) * t.element_size() for t in ts if t.dim() == 2 and t.shape[0] > 1}
        assert rk._overlap(*ts) or not meet
        if len(apart) == 1:  # exact; strides that differ may be refused where they only interleave
            assert rk._overlap(*ts) == meet
            seen.add(meet)
    assert seen == {True, False}
    both = torch.zeros(3, 32)
    for scores, out in ((both[:, :16], both[:, 16:]), (both[:, 16:], both[:, :16]), (both, both[:]),
                        (both[:, 4:9], both.view(3, 32)[:, 4:9]), (both[:1, :8], both[:1, 8:16])):
        with pytest.raises(ValueError, match='HIP device'):
            rk.adjust_scores(scores, out=out)
    for scores, out in ((both[:, :16], both[:, 15:31]), (both[:, :16], both[:, 1:17]),
                        (both[:2], both[1:])):
        with pytest.raises(ValueError, match='overlap'):
            rk.adjust_scores(scores, out=out)
    with pytest.raises(ValueError, match='overlap'):
        rk.adjust_scores(both, item_bias=both[0], out=both[:])
    with pytest.raises(ValueError, match='one of'):
        rk.adjust_scores(both, out=both.view(torch.int32))
