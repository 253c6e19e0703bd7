"""What the norm, the cache's calls and the attention over it refuse, at the C entry and in the Python front end; no GPU, nothing
is ever run."""
import ctypes as C

import pytest
import torch

from nnops_b200 import capi, ops

BASE = 0x7000_0000_1000    # never dereferenced: validation comes first


def _norm(**over):
    a = capi.RmsNormI8Args(x=BASE, weight=BASE + 0x10000, out=BASE + 0x20000, scale=BASE + 0x30000, rows=2, cols=64, x_stride=64, out_stride=64,
                           eps=1e-6, float_type=1, weight_type=1)
    for k, v in over.items():
        setattr(a, k, v)
    return a


def _cache(cls, **over):
    a = cls(k=BASE, v=BASE + 0x10000, k_scale=BASE + 0x20000, v_scale=BASE + 0x21000, pages=4, page_stride=2 * 16 * 64, scale_page_stride=2, heads=2,
            page_tokens=16, dim=64, page_table=BASE + 0x30000, table_stride=4, table_pages=4, lens=BASE + 0x31000, cu=BASE + 0x32000, seqs=2, rows=6)
    if cls is capi.CacheRowsArgs:
        a.rows_k, a.rows_v = BASE + 0x40000, BASE + 0x50000
        a.k_stride_row = a.v_stride_row = 128
        a.k_stride_head = a.v_stride_head = 64
    else:
        a.q, a.out, a.q_heads, a.causal, a.scale = BASE + 0x40000, BASE + 0x50000, 4, 1, 0.125
        a.q_stride_row = a.out_stride_row = 256
        a.q_stride_head = a.out_stride_head = 64
    a.float_type = 1
    for k, v in over.items():
        setattr(a, k, v)
    return a


def test_norm_arguments(nnb200_lib):
    before = nnb200_lib.nnb200_launch_count()
    for over in (dict(rows=-1), dict(cols=-1), dict(rows=1 << 31), dict(float_type=3), dict(float_type=-1), dict(weight_type=2), dict(x=None),
                 dict(weight=None), dict(out=None), dict(scale=None), dict(x=BASE + 1), dict(weight=BASE + 1), dict(scale=BASE + 2),
                 dict(residual=BASE + 1), dict(residual_out=BASE + 1), dict(out_stride=63), dict(residual_out=BASE, residual_out_stride=1)):
        assert nnb200_lib.nnb200_rms_norm_i8(C.byref(_norm(**over)), None) == capi.INVALID_ARGUMENT, over
    assert nnb200_lib.nnb200_rms_norm_i8(None, None) == capi.INVALID_ARGUMENT
    assert nnb200_lib.nnb200_rms_norm_i8(C.byref(_norm(rows=0, x=None)), None) == capi.OK
    assert nnb200_lib.nnb200_launch_count() == before


WRONG_CACHE = [dict(rows=-1), dict(rows=1 << 31), dict(seqs=-1), dict(seqs=0), dict(heads=0), dict(dim=0), dict(pages=-1), dict(pages=1 << 31),
               dict(table_pages=-1), dict(table_pages=1 << 30), dict(table_stride=3), dict(table_stride=-4), dict(k=None), dict(v=None),
               dict(k_scale=None), dict(v_scale=None), dict(lens=None), dict(page_table=None), dict(k=BASE + 8), dict(v=BASE + 4),
               dict(k_scale=BASE + 2), dict(v_scale=BASE + 1), dict(lens=BASE + 2), dict(cu=BASE + 1), dict(page_table=BASE + 3), dict(page_stride=2047),
               dict(page_stride=2032), dict(page_stride=2056), dict(scale_page_stride=1), dict(cu=None, rows=7), dict(float_type=3)]
UNKNOWN_CACHE = [dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=256), dict(dim=24), dict(dim=272)]


@pytest.mark.parametrize("entry", ["nnb200_cache_write_i8", "nnb200_cache_read_i8", "nnb200_attention_i8"])
def test_cache_arguments(nnb200_lib, entry):
    cls = capi.AttentionI8Args if "attention" in entry else capi.CacheRowsArgs
    call = getattr(nnb200_lib, entry)
    before = nnb200_lib.nnb200_launch_count()
    for over in WRONG_CACHE:
        assert call(C.byref(_cache(cls, **over)), None) == capi.INVALID_ARGUMENT, over
    for over in UNKNOWN_CACHE:
        assert call(C.byref(_cache(cls, **over)), None) == capi.UNSUPPORTED, over
    pointers = ("q", "out") if cls is capi.AttentionI8Args else ("rows_k", "rows_v")
    for name in pointers:
        for value in (None, BASE + 1):
            assert call(C.byref(_cache(cls, **{name: value})), None) == capi.INVALID_ARGUMENT, name
    assert call(None, None) == capi.INVALID_ARGUMENT
    assert call(C.byref(_cache(cls, rows=0, k=None, lens=None)), None) == capi.OK    # nothing to do
    assert nnb200_lib.nnb200_launch_count() == before


def test_attention_arguments(nnb200_lib):
    call = nnb200_lib.nnb200_attention_i8
    for over in (dict(q_heads=0), dict(q_heads=3), dict(window=-1), dict(sinks=-1), dict(window=4, causal=0), dict(force_engine=9),
                 dict(workspace=BASE + 8, workspace_bytes=1 << 40)):
        assert call(C.byref(_cache(capi.AttentionI8Args, **over)), None) == capi.INVALID_ARGUMENT, over
    for dim in (16, 80, 112, 160):
        assert call(C.byref(_cache(capi.AttentionI8Args, dim=dim, page_stride=1 << 20)), None) == capi.UNSUPPORTED, dim
    assert call(C.byref(_cache(capi.AttentionI8Args, rows=0x7FFFFFFE, q_heads=64)), None) == capi.UNSUPPORTED
    assert nnb200_lib.nnb200_attention_i8_workspace_bytes(C.byref(_cache(capi.AttentionI8Args, rows=0))) == 0
    assert nnb200_lib.nnb200_attention_i8_workspace_bytes(None) == 0


def test_outputs_whose_rows_overlap(nnb200_lib):
    """rows = 6 of 2 heads (read) or 4 (attention) of 64 values."""
    read, attention = nnb200_lib.nnb200_cache_read_i8, nnb200_lib.nnb200_attention_i8
    for row, head in ((0, 64), (64, 64), (127, 64), (128, 0), (128, 63), (64, 383), (-128, 64)):
        for name in "kv":
            over = {f"{name}_stride_row": row, f"{name}_stride_head": head}
            assert read(C.byref(_cache(capi.CacheRowsArgs, **over)), None) == capi.INVALID_ARGUMENT, over
    for row, head in ((0, 64), (64, 64), (255, 64), (256, 63), (64, 383), (1, 1)):
        over = dict(out_stride_row=row, out_stride_head=head)
        assert attention(C.byref(_cache(capi.AttentionI8Args, **over)), None) == capi.INVALID_ARGUMENT, over
    assert attention(C.byref(_cache(capi.AttentionI8Args, rows=1, seqs=1, cu=None, out_stride_row=0, out_stride_head=63)), None) == capi.INVALID_ARGUMENT


def test_blocks_agree_with_the_header():
    assert C.sizeof(capi.CacheRowsArgs) == 17 * 8 + 6 * 8 + 8
    assert C.sizeof(capi.AttentionI8Args) == 17 * 8 + 9 * 8 + 16 + 16
    assert C.sizeof(capi.RmsNormI8Args) == 12 * 8 + 16


def test_caches_that_are_none():
    codes, scale = torch.zeros((4, 2, 16, 64), dtype=torch.int8), torch.zeros((4, 2))
    for bad in [(codes.short(), codes, scale, scale), (codes, codes[:3], scale, scale), (codes, codes, scale[:3], scale[:3]), (codes, codes, scale.half(), scale),
                (codes.transpose(1, 2), codes.transpose(1, 2), torch.zeros((4, 16)), torch.zeros((4, 16))), (codes[0], codes[0], scale, scale),
                (codes[..., ::2], codes[..., ::2], scale, scale), (codes, codes, torch.zeros((2, 4)).t(), torch.zeros((2, 4)).t())]:
        with pytest.raises(ValueError):
            ops.CacheI8(*bad)
    ops.CacheI8(codes, codes, scale, scale)


def test_the_front_end_has_no_cpu_path(nnb200_lib):
    cache = ops.CacheI8.empty(4, 2, 16, 64, "cpu")
    x, ints = torch.zeros((2, 2, 64)), torch.zeros((2, 2), dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.rms_norm_i8(torch.zeros((2, 64)), torch.zeros(64))
    for call in (lambda: ops.cache_write_i8(cache, x, x, ints, ints[0]), lambda: ops.cache_read_i8(cache, ints, ints[0], rows=2),
                 lambda: ops.attention_i8_cache(x, cache, ints, ints[0])):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_what_the_front_end_refuses(nnb200_lib, monkeypatch):
    """The checks come before anything is looked at on a device: a cache that says it is on one."""
    cache = ops.CacheI8.empty(4, 2, 16, 64, "cpu")
    monkeypatch.setattr(ops, "_native", ops._NoFront())
    x, table, lens = torch.zeros((4, 2, 64)), torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros((4, 4, 64))
    with pytest.raises(ValueError):
        ops.cache_write_i8(cache, x.int(), x.int(), table, lens)
    with pytest.raises(ValueError):
        ops.cache_write_i8(cache, x, x.half(), table, lens)
    with pytest.raises(ValueError):
        ops.cache_write_i8(cache, x, x[:3], table, lens)
    with pytest.raises(ValueError):
        ops.cache_write_i8(cache, x[..., :32], x[..., :32], table, lens)
    with pytest.raises(ValueError):
        ops.cache_read_i8(cache, table, lens)
    with pytest.raises(ValueError):
        ops.cache_read_i8(cache, table, lens, rows=4, out_dtype=torch.int8)
    for kw in (dict(window=-1), dict(sinks=-1), dict(window=3, causal=False), dict(out=q.half()), dict(out=q[:3])):
        with pytest.raises(ValueError):
            ops.attention_i8_cache(q, cache, table, lens, **kw)
    with pytest.raises(ValueError):
        ops.attention_i8_cache(q[:, :3], cache, table, lens)
    with pytest.raises(ValueError):
        ops.attention_i8_cache(q.double(), cache, table, lens)

    class There:
        type = "cuda"

        def __eq__(self, other):
            return other == torch.device("cpu")

        __hash__ = None

    cache.device = There()
    for bad in [(table.long(), lens, None), (table, lens.long(), None), (table[:1], lens, None), (table, lens, lens), (table, lens[None], None),
                (table.t().contiguous().t(), lens, None), (torch.zeros((3, 3), dtype=torch.int32), torch.zeros(3, dtype=torch.int32), None)]:
        with pytest.raises(ValueError):
            ops._sequences(cache, *bad, 4)
    assert ops._sequences(cache, table, lens, None, 4)[-2:] == (2, 4)


def test_a_cache_whose_tensors_are_replaced(nnb200_lib, monkeypatch):
    """A call takes the tensors that the cache has then, wherever they lie, and not those it was made with."""
    cache = ops.CacheI8.empty(4, 2, 16, 64, "cpu")
    table, lens = torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)

    class There:
        type = "cuda"

        def __eq__(self, other):
            return other == torch.device("cpu")

        __hash__ = None

    cache.device = There()

    def taken():
        fields = ops._sequences(cache, table, lens, None, 4)
        assert fields[:4] == tuple(t.data_ptr() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale))
        assert fields[4:10] == (cache.k.shape[0], cache.k.stride(0), cache.k_scale.stride(0), *cache.k.shape[1:])
        assert (cache.pages, cache.heads, cache.page_tokens, cache.dim) == tuple(cache.k.shape)

    taken()
    old = cache.k, cache.v, cache.k_scale, cache.v_scale
    cache.k, cache.v = (torch.cat([t, t]) for t in old[:2])    # grown
    with pytest.raises(ValueError):
        ops._sequences(cache, table, lens, None, 4)    # its scales are not
    cache.k_scale, cache.v_scale = (torch.cat([t, t]) for t in old[2:])
    taken()
    cache.k.data = torch.zeros_like(cache.k)    # another storage in the same tensor
    taken()
    for t in (cache.k, cache.v):
        t.resize_(9, 2, 16, 64)
    for t in (cache.k_scale, cache.v_scale):
        t.resize_(9, 2)
    taken()
    cache.v = cache.v.transpose(1, 2)
    with pytest.raises(ValueError):
        ops._sequences(cache, table, lens, None, 4)
    cache.v = old[1].short()
    with pytest.raises(ValueError):
        ops._sequences(cache, table, lens, None, 4)

    # The compiled half is handed the same ones.
    class Front:
        def __getattr__(self, name):
            return lambda *args: args

    monkeypatch.setattr(ops, "_native", Front())
    cache.k, cache.v, cache.k_scale, cache.v_scale = old
    q = torch.zeros((4, 4, 64))
    for args in (ops.attention_i8_cache(q, cache, table, lens)[1:], ops.cache_read_i8(cache, table, lens, rows=4)):
        assert all(a is b for a, b in zip(args[:4], old))


def test_a_norm_that_would_write_over_rows_not_yet_read(nnb200_lib):
    """residual_out upon x or residual: row for row, or nowhere.  (Rows of 64 f16 values, 128 bytes.)"""
    call = nnb200_lib.nnb200_rms_norm_i8
    before = nnb200_lib.nnb200_launch_count()
    other = BASE + 0x40000
    for name, at in (("x", BASE), ("residual", other)):
        base = dict(rows=4, x_stride=128, residual=other, residual_stride=128, residual_out_stride=128)
        for over in (dict(residual_out=at, residual_out_stride=64), dict(residual_out=at, residual_out_stride=136), dict(residual_out=at + 2),
                     dict(residual_out=at + 126), dict(residual_out=at - 2), dict(residual_out=at + 256 * 3 + 126), dict(residual_out=at + 256 - 126),
                     dict(residual_out=at + 128, residual_out_stride=64), {"residual_out": at, f"{name}_stride": 0},
                     {"residual_out": at - 256 * 3, f"{name}_stride": -128}, dict(residual_out=BASE - 0x1000, residual_out_stride=1 << 61),
                     {"residual_out": BASE + 0x90000, f"{name}_stride": 1 << 62}, {"residual_out": BASE + 0x90000, f"{name}_stride": (1 << 63) - 1}):
            assert call(C.byref(_norm(**(base | over))), None) == capi.INVALID_ARGUMENT, (name, over)
        assert call(C.byref(_norm(**(base | dict(rows=1, residual_out=at + 64)))), None) == capi.INVALID_ARGUMENT
        # Row upon row, between the rows, before and behind them: no mistake, but there is no device here.
        if not torch.cuda.is_available():
            for over in (dict(residual_out=at), dict(residual_out=at + 128), dict(residual_out=at - 128), dict(residual_out=at - 256 * 3 - 128),
                         dict(residual_out=at + 256 * 3 + 128, residual_out_stride=64), dict(rows=1, residual_out=at, residual_out_stride=5000)):
                assert call(C.byref(_norm(**(base | over))), None) == capi.INTERNAL, (name, over)
    assert nnb200_lib.nnb200_launch_count() == before


def test_a_norm_of_no_columns_is_a_call(nnb200_lib):
    """Its rows have scales to be written: nothing but those is needed, and it is not answered with nothing done."""
    call = nnb200_lib.nnb200_rms_norm_i8
    assert call(C.byref(_norm(cols=0, scale=None)), None) == capi.INVALID_ARGUMENT
    if not torch.cuda.is_available():
        # Rows of nothing lie nowhere.
        assert call(C.byref(_norm(cols=0, rows=4, residual=BASE + 64, residual_out=BASE + 2, residual_out_stride=1, x_stride=3)), None) == capi.INTERNAL
        assert call(C.byref(_norm(cols=0, x=None, weight=None, out=None)), None) == capi.INTERNAL
    assert call(C.byref(_norm(rows=0, cols=0, scale=None)), None) == capi.OK


def test_keys_and_values_read_into_one_place(nnb200_lib):
    """Which of the two it would hold depended on timing.  To be written they may be the same."""
    same = _cache(capi.CacheRowsArgs, rows_k=BASE + 0x40000, rows_v=BASE + 0x40000)
    assert nnb200_lib.nnb200_cache_read_i8(C.byref(same), None) == capi.INVALID_ARGUMENT
    if not torch.cuda.is_available():
        assert nnb200_lib.nnb200_cache_write_i8(C.byref(same), None) == capi.INTERNAL
        apart = _cache(capi.CacheRowsArgs, k_stride_row=256, v_stride_row=256, rows_v=BASE + 0x40000 + 256)    # in rows of both
        assert nnb200_lib.nnb200_cache_read_i8(C.byref(apart), None) == capi.INTERNAL
