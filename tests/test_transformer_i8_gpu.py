"""RMS norm into 8 bits, the 8-bit key/value cache and the attention over it, against plain implementations: codes, scales and
values read back bit for bit, sums against 64 bits."""
import ctypes as C
import math

import pytest
import torch

from nnops_b200 import capi, ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
TYPES = [torch.float16, torch.bfloat16, torch.float32]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(shape, generator=g)


# ---- RMS norm ---------------------------------------------------------------------------------

def _norm_reference(x, w, residual, eps):
    """Codes by the f32 formula (each step rounded once, as documented), scale and sum in 64 bits."""
    h = x.float() if residual is None else x.float() + residual.float()
    t = h * w.float()
    top = t.abs().amax(1).clamp(min=2.0 ** -100)
    codes = torch.round(t * (torch.tensor(127.0) / top)[:, None]).to(torch.int8)
    scale = top.double() / (127 * torch.sqrt(h.double().square().mean(1) + eps))
    return codes, scale, h.to(x.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 8), (7, 136), (9, 256), (2, 264), (130, 512), (4, 520), (3, 1000), (2, 4096),
                                       (3, 8192), (2, 8200), (2, 16384), (1, 32768), (1, 40008), (2, 16389)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(cuda_device, nnb200_lib, dtype, rows, cols, residual):
    g = _gen(rows * 100003 + cols)
    x, w = _randn(g, rows, cols).to(dtype), (1 + 0.2 * _randn(g, cols)).to(dtype)
    r = (3 * _randn(g, rows, cols)).to(dtype) if residual else None
    codes, scale, h = _norm_reference(x, w, r, 1e-5)
    got = ops.rms_norm_i8(x.cuda(), w.cuda(), residual=r.cuda() if residual else None, eps=1e-5)
    assert torch.equal(got[0].cpu(), codes)
    # One rounding to f32 of a scale whose sum is in 64 bits, and eps as an f32: 2^-24 each, doubled by the rounding of the test's own.
    assert ((got[1].cpu().double() - scale).abs() <= 2.0 ** -22 * scale).all()
    if residual:
        assert torch.equal(got[2].cpu(), h)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("cols", [512, 1001])
def test_norm_in_place_strided_with_an_f32_weight(cuda_device, nnb200_lib, dtype, cols):
    g = _gen(cols)
    x, r, w = _randn(g, 6, cols).to(dtype), _randn(g, 6, cols).to(dtype), 1 + _randn(g, cols)
    codes, scale, h = _norm_reference(x, w, r, 1e-6)
    pad = cols + 24
    xs, rs = torch.zeros((6, pad), dtype=dtype, device="cuda"), torch.zeros((6, pad), dtype=dtype, device="cuda")
    xs[:, 8:8 + cols], rs[:, 16:16 + cols] = x.cuda(), r.cuda()
    out = torch.full((6, pad), 99, dtype=torch.int8, device="cuda")
    for into in (xs[:, 8:8 + cols], rs[:, 16:16 + cols]):
        xs[:, 8:8 + cols], rs[:, 16:16 + cols] = x.cuda(), r.cuda()
        got = ops.rms_norm_i8(xs[:, 8:8 + cols], w.cuda(), residual=rs[:, 16:16 + cols], residual_out=into, out=out[:, 8:8 + cols])
        assert got[2].data_ptr() == into.data_ptr()
        assert torch.equal(got[0].cpu(), codes) and torch.equal(into.cpu(), h)
        assert (got[1].cpu().double() - scale).abs().max() <= 2.0 ** -22 * scale.max()
        assert (out[:, :8] == 99).all() and (out[:, 8 + cols:] == 99).all()


def test_norm_rows_that_are_no_numbers_or_nothing(cuda_device, nnb200_lib):
    for cols in (64, 1025):
        x = torch.ones((6, cols), device="cuda")
        x[0, 3], x[1, 5], x[2, 7] = math.nan, math.inf, -math.inf
        x[3] = 0
        x[4] = 1e-38
        x[5] = 1e30    # its squares pass f32
        codes, scale = ops.rms_norm_i8(x, torch.ones(cols, device="cuda"), eps=1e-6)
        assert scale[:3].isnan().all() and (codes[:4] == 0).all()
        assert 0 < scale[3] < 1e-20 and 0 < scale[4] < 1e-20    # 2^-100 / (127 sqrt(eps)), and nothing is divided by zero
        assert (codes[5] == 127).all() and abs(scale[5].item() * 127 - 1) < 1e-6
    empty = ops.rms_norm_i8(torch.ones((0, 8), device="cuda"), torch.ones(8, device="cuda"))
    assert empty[0].shape == (0, 8)


# ---- cache --------------------------------------------------------------------------------------

class _Plain:
    """A cache on the CPU, and what a write does to it."""

    def __init__(self, pages, heads, tokens, dim):
        self.codes = [torch.zeros((pages, heads, tokens, dim), dtype=torch.int8) for _ in range(2)]
        self.scale = [torch.zeros((pages, heads)) for _ in range(2)]
        self.tokens = tokens

    def write(self, k, v, table, lens, cu):
        for codes, scales, x in zip(self.codes, self.scale, (k.float(), v.float())):
            for b, length in enumerate(lens):
                n = cu[b + 1] - cu[b]
                first = max(0, length - n)
                for slot in range(first // self.tokens, -(-length // self.tokens) if n else 0):
                    page, start = table[b][slot], slot * self.tokens
                    low, high = max(first, start), min(length, start + self.tokens)
                    rows = x[cu[b] + low - (length - n): cu[b] + high - (length - n)]    # [tokens, heads, dim]
                    need = (rows.abs().amax((0, 2)) / torch.tensor(127.0)).clamp(min=2.0 ** -60)
                    if low == start and start >= first:
                        after = need
                    else:
                        after = torch.maximum(scales[page], need)
                        ratio = scales[page] / after
                        codes[page] = torch.round(codes[page].float() * ratio[:, None, None]).to(torch.int8)
                    codes[page, :, low - start: high - start] = torch.round(rows * (torch.tensor(1.0) / after)[None, :, None]).to(torch.int8).transpose(0, 1)
                    scales[page] = after

    def values(self, which, table, length):
        """[length, heads, dim] of one sequence, f32."""
        ids = torch.tensor(table[: -(-length // self.tokens)], dtype=torch.long)
        x = self.codes[which][ids].float() * self.scale[which][ids][..., None, None]
        return x.transpose(1, 2).flatten(0, 1)[:length]


def _tables(g, lens, tokens, spare=3):
    need = [-(-n // tokens) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    wide = max(1, *need) if need else 1
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (wide - n))
        at += n
    return table, sum(need) + spare


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _cu(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def _same(cache, plain):
    return (torch.equal(cache.k.cpu(), plain.codes[0]) and torch.equal(cache.v.cpu(), plain.codes[1]) and
            torch.equal(cache.k_scale.cpu(), plain.scale[0]) and torch.equal(cache.v_scale.cpu(), plain.scale[1]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,dim,tokens", [(1, 16, 16), (3, 96, 32), (2, 128, 64), (2, 256, 128), (1, 80, 128), (5, 64, 16)])
@pytest.mark.parametrize("strided", [False, True])
def test_a_cache_that_grows(cuda_device, nnb200_lib, dtype, heads, dim, tokens, strided):
    """Prompts, single tokens, runs that end inside a page, nothing at all: after every call codes and scales are the
    plain cache's, and what is read back is what they stand for."""
    g = _gen(heads * dim + tokens)
    finally_ = [3 * tokens + 5, 1, 2 * tokens, 0, tokens + 1, 17]
    table, pages = _tables(g, finally_, tokens)
    cache, plain = ops.CacheI8.empty(pages, heads, tokens, dim, "cuda"), _Plain(pages, heads, tokens, dim)
    lens = [0] * len(finally_)
    steps = [[2 * tokens + 3, 1, 1, 0, tokens - 1, 5], [1, 0, tokens, 0, 1, 1], [1, 0, tokens - 1, 0, 1, 11], [tokens + 1, 0, 0, 0, 0, 0]]
    for i, new in enumerate(steps):
        lens = [a + b for a, b in zip(lens, new)]
        rows = sum(new)
        k, v = (((1 + 2 * i) * _randn(g, rows, heads, dim)).to(dtype) for _ in range(2))
        if strided:    # three tensors in one, off the 16-byte rule by their heads' distance
            both = torch.zeros((rows, heads, 3 * dim + 5), dtype=dtype, device="cuda")
            both[..., 3:3 + dim], both[..., 7 + dim:7 + 2 * dim] = k.cuda(), v.cuda()
            dk, dv = both[..., 3:3 + dim], both[..., 7 + dim:7 + 2 * dim]
        else:
            dk, dv = k.cuda(), v.cuda()
        ops.cache_write_i8(cache, dk, dv, _i32(table), _i32(lens), cu=_i32(_cu(new)))
        plain.write(k, v, table, lens, _cu(new))
        assert _same(cache, plain), i
        got = ops.cache_read_i8(cache, _i32(table), _i32(lens), rows=sum(lens), cu=_i32(_cu(lens)), out_dtype=dtype)
        for which in range(2):
            want = torch.cat([plain.values(which, t, n) for t, n in zip(table, lens)])
            assert torch.equal(got[which].cpu(), want.to(dtype)), i


def test_uniform_rows_need_no_cu(cuda_device, nnb200_lib):
    g = _gen(5)
    lens, tokens, heads, dim = [40, 33, 64, 0, 16, 2], 16, 2, 64
    table, pages = _tables(g, lens, tokens)
    for n in (1, 3, 20):
        cache, plain = ops.CacheI8.empty(pages, heads, tokens, dim, "cuda"), _Plain(pages, heads, tokens, dim)
        k, v = (_randn(g, n * len(lens), heads, dim) for _ in range(2))
        ops.cache_write_i8(cache, k.cuda(), v.cuda(), _i32(table), _i32(lens))
        plain.write(k, v, table, lens, [n * i for i in range(len(lens) + 1)])
        assert _same(cache, plain)
        out = tuple(torch.full((n * len(lens), heads, dim + 8), 7.0, device="cuda")[..., :dim] for _ in range(2))
        got = ops.cache_read_i8(cache, _i32(table), _i32(lens), out=out)
        for which in range(2):
            for b, length in enumerate(lens):
                want = plain.values(which, table[b], length)
                want = torch.cat([torch.zeros(max(0, n - length), heads, dim), want[max(0, length - n):]])
                assert torch.equal(got[which][b * n:(b + 1) * n].cpu(), want)


def test_rows_behind_the_last_sequence_stay_as_they_are(cuda_device, nnb200_lib):
    lens, new = [20, 5], [4, 2]
    table, pages = _tables(_gen(1), lens, 16)
    cache = ops.CacheI8.empty(pages, 1, 16, 64, "cuda")
    k = torch.ones((10, 1, 64), device="cuda")
    k[:2] = k[8:] = math.nan    # rows before the first sequence's and behind the last one's
    cu = _i32([2, 6, 8])
    ops.cache_write_i8(cache, k, k, _i32(table), _i32(lens), cu=cu)
    assert cache.k_scale.isfinite().all() and (cache.k != 0).sum() == 6 * 64
    out = tuple(torch.full((10, 1, 64), 5.0, device="cuda") for _ in range(2))
    ops.cache_read_i8(cache, _i32(table), _i32(lens), cu=cu, out=out)
    q = torch.full((10, 2, 64), 5.0, device="cuda")
    ops.attention_i8_cache(q.clone(), cache, _i32(table), _i32(lens), cu=cu, out=q)
    for t in (*out, q):
        assert (t[:2] == 5).all() and (t[8:] == 5).all() and (t[2:8] != 5).all()


def test_a_page_that_is_no_number_until_it_begins_anew(cuda_device, nnb200_lib):
    cache = ops.CacheI8.empty(2, 2, 16, 64, "cuda")
    table = _i32([[1]])

    def write(length, rows):
        ops.cache_write_i8(cache, rows, rows, table, _i32([length]))
        return ops.cache_read_i8(cache, table, _i32([length]), rows=length, out_dtype=torch.float32)[0]

    for bad in (math.nan, math.inf, -math.inf):
        x = torch.ones((1, 2, 64), device="cuda")
        assert write(1, x).isfinite().all()
        x[0, 1, 9] = bad
        got = write(2, x)
        assert got[:, 0].isfinite().all() and got[:, 1].isnan().all()
        got = write(3, torch.ones((1, 2, 64), device="cuda"))
        assert got[:, 0].isfinite().all() and got[:, 1].isnan().all()
        assert (write(1, torch.zeros((1, 2, 64), device="cuda")) == 0).all()    # begins anew, with nothing in it
        assert (cache.k_scale[1] == 2.0 ** -60).all()


# ---- attention ------------------------------------------------------------------------------------

def _attention_reference(q, cache, table, lens, cu, group, causal, window, sinks, scale):
    """In 64 bits, and for each output what it may be off by: see the terms."""
    codes, scales = (cache.k.cpu(), cache.v.cpu()), (cache.k_scale.cpu(), cache.v_scale.cpu())
    tokens, dim = codes[0].shape[2:]
    out, tol = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
    split = q.dtype is torch.float32
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0 or length == 0:
            continue
        ids = torch.tensor(table[b][: -(-length // tokens)], dtype=torch.long)
        k, v = ((codes[i][ids].double() * scales[i][ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:length] for i in range(2))
        pos = length - n + torch.arange(n)
        j = torch.arange(length)
        seen = (j[None] <= pos[:, None]) if causal else torch.ones((n, length), dtype=torch.bool)
        if window:
            seen &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
        x = q[cu[b]:cu[b + 1]].double()
        for a in range(q.shape[1]):
            kh, vh = k[:, a // group], v[:, a // group]
            z = torch.where(seen, x[:, a] @ kh.T * scale, -math.inf)
            p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
            o, spread = p @ vh, p @ vh.abs()
            # A weight's exponent: a dot product of dim terms in f32 (and q's own roundings: 2^-22 of its largest, or f16's least step,
            # 2^-25 of it), then three roundings of an exponent below 2^7, and ex2's.
            products = (x[:, a].abs().amax(1) * kh.abs().sum(1).max() * scale)[:, None]
            exponent = (dim + 8) * 2.0 ** -24 * (x[:, a].abs() @ kh.abs().T * scale).amax(1, keepdim=True) + products * 2.0 ** -22 + 2.0 ** -16
            # The weight as an f16 (f32 rows: as two), against a largest one of 1; sums of `length` terms in f32.
            weight = (2.0 ** -22 if split else 2.0 ** -11) + length * 2.0 ** -24
            least = length * 2.0 ** -25 * 127 * scales[1][ids, a // group].double().max()
            off = spread * (2 * exponent + weight) + least * seen.any(1, keepdim=True)
            out[cu[b]:cu[b + 1], a] = o
            tol[cu[b]:cu[b + 1], a] = off + (o.abs() + off) * HALF_STEP[q.dtype]
    return out, tol


def _filled(g, pages, heads, tokens, dim):
    """A cache of random codes, and scales that differ from page to page by a factor of up to a thousand (values)."""
    made = [torch.randint(-127, 128, (pages, heads, tokens, dim), generator=g, dtype=torch.int32).to(torch.int8).cuda() for _ in range(2)]
    ks = torch.exp(0.3 * _randn(g, pages, heads)) / 80
    vs = torch.exp(1.2 * _randn(g, pages, heads)) / 80
    return ops.CacheI8(*made, ks.cuda(), vs.cuda())


def _check_attention(g, dtype, heads, group, dim, tokens, lens, new, *, causal=True, window=0, sinks=0, scale=None, uniform=False, engine="auto"):
    table, pages = _tables(g, lens, tokens)
    cache = _filled(g, pages, heads, tokens, dim)
    cu = _cu(new)
    q = _randn(g, cu[-1], heads * group, dim).to(dtype)
    got = ops.attention_i8_cache(q.cuda(), cache, _i32(table), _i32(lens), cu=None if uniform else _i32(cu), causal=causal, window=window,
                                 sinks=sinks, scale=scale, engine=engine)
    want, tol = _attention_reference(q, cache, table, lens, cu, group, causal, window, sinks, 1 / math.sqrt(dim) if scale is None else scale)
    assert got.dtype is dtype
    off = (got.cpu().double() - want).abs()
    assert (off <= tol).all(), (off / tol.clamp(min=1e-300)).max().item()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,tokens", [(1, 1, 16), (2, 4, 64), (3, 7, 32), (2, 8, 128), (1, 16, 16)])
def test_single_tokens(cuda_device, nnb200_lib, dtype, dim, heads, group, tokens):
    lens = [1, 0, 15, 16, 17, 129, 700, 1000]
    _check_attention(_gen(dim + group), dtype, heads, group, dim, tokens, lens, [1] * len(lens), uniform=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,group,tokens", [(64, 2, 3, 16), (128, 1, 8, 128), (96, 2, 5, 64), (256, 1, 4, 32), (128, 3, 1, 32)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 3), (40, 20), (100, 1), (64, 500)])
def test_several_tokens_masks_and_ragged_rows(cuda_device, nnb200_lib, dtype, dim, heads, group, tokens, window, sinks):
    """Rows before the sequence see nothing, a sequence has no row or no token, windows end inside pages."""
    lens = [5, 333, 0, 64, 200, 31, 90]
    new = [5, 37, 2, 0, 1, 40, 17]
    _check_attention(_gen(dim + window), dtype, heads, group, dim, tokens, lens, new, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
def test_without_causality_and_with_a_scale(cuda_device, nnb200_lib, dtype, dim):
    _check_attention(_gen(dim), dtype, 2, 4, dim, 32, [3, 100, 0, 65], [7, 30, 1, 2], causal=False, scale=0.03)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,heads,group,new", [(64, 2, 3, 5), (128, 1, 8, 1), (128, 2, 4, 9), (96, 1, 5, 7), (256, 1, 3, 3), (64, 1, 1, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 5), (300, 40)])
def test_as_many_rows_in_every_sequence(cuda_device, nnb200_lib, dtype, dim, heads, group, new, window, sinks):
    """Without cu, few row tiles and a short table: a cluster of blocks for each.  With cu, one line for all: the same to a rounding or two."""
    g = _gen(dim + new)
    lens = [new, 0, 1, 777, 1500]
    if heads * group * new > 60:
        lens = lens[2:]
    got = _check_attention(g, dtype, heads, group, dim, 16, lens, [new] * len(lens), window=window, sinks=sinks, uniform=True, engine="rows")
    assert got.isfinite().all()
    _check_attention(_gen(dim + new), dtype, heads, group, dim, 16, lens, [new] * len(lens), window=window, sinks=sinks, engine="rows")


@pytest.mark.parametrize("tokens", [15, 16, 17, 127, 129, 1024, 9000])
def test_one_sequence_of_any_length(cuda_device, nnb200_lib, tokens):
    """A cluster whose blocks have many groups, one or none; a table too wide for clusters; every kernel has it right."""
    for dtype in TYPES:
        _check_attention(_gen(tokens), dtype, 2, 2, 64, 16, [tokens], [1], uniform=True)
    g = _gen(tokens)
    table, pages = _tables(g, [tokens], 16)
    cache = _filled(g, pages, 2, 16, 64)
    q = _randn(g, 1, 4, 64).half()
    want, tol = _attention_reference(q, cache, table, [tokens], [0, 1], 2, True, 0, 0, 1 / 8)
    wide = torch.full((1, 2000), -1, dtype=torch.int32, device="cuda")
    wide[:, : len(table[0])] = _i32(table)
    for engine in ("auto", "rows", "tile"):
        got = ops.attention_i8_cache(q.cuda(), cache, wide, _i32([tokens]), engine=engine)
        assert ((got.cpu().double() - want).abs() <= tol).all(), engine


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,new", [(128, 300), (64, 513), (96, 150), (256, 140)])
def test_prompts(cuda_device, nnb200_lib, dtype, dim, new):
    _check_attention(_gen(new), dtype, 2, 4, dim, 64, [new, new + 77, 1200, 3], [new, new - 1, 129, 3])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("heads,group,tokens", [(1, 1, 16), (2, 4, 64), (3, 7, 32), (2, 16, 128)])
def test_tiles_from_one_row_on(cuda_device, nnb200_lib, dtype, dim, heads, group, tokens):
    """The kernel for many rows, whatever their number: empty tiles, tiles that end inside a token's heads, lengths around a block's."""
    lens = [1, 0, 15, 127, 128, 129, 300, 700, 1000]
    new = [1, 1, 15, 60, 128, 0, 33, 2, 257]
    _check_attention(_gen(dim + group), dtype, heads, group, dim, tokens, lens, new, engine="tile")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,heads,group,tokens", [(64, 2, 3, 16), (128, 1, 8, 128), (96, 2, 5, 64), (256, 1, 4, 32), (128, 3, 1, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 3), (40, 20), (100, 1), (64, 500)])
def test_tiles_with_a_window(cuda_device, nnb200_lib, dtype, dim, heads, group, tokens, window, sinks):
    lens = [5, 333, 0, 64, 200, 31, 90, 700]
    new = [5, 37, 2, 0, 1, 40, 17, 400]
    _check_attention(_gen(dim + window), dtype, heads, group, dim, tokens, lens, new, window=window, sinks=sinks, engine="tile")


@pytest.mark.parametrize("dim", [64, 128])
def test_tiles_without_causality(cuda_device, nnb200_lib, dim):
    _check_attention(_gen(dim), torch.float16, 2, 4, dim, 32, [3, 400, 0, 65], [7, 130, 1, 2], causal=False, scale=0.03, engine="tile")
    _check_attention(_gen(dim), torch.float16, 1, 4, dim, 32, [3, 400, 0, 65], [7, 130, 1, 2], scale=-0.1, engine="tile")


def test_maxima_that_grow_along_the_tokens(cuda_device, nnb200_lib):
    """Logits that rise by far more than the sums are rescaled for, block after block, and fall again."""
    g = _gen(7)
    for engine in ("rows", "tile"):
        cache = _filled(g, 40, 1, 32, 64)
        ramp = torch.cat([torch.linspace(0.01, 4, 20), torch.linspace(4, 0.01, 20)])
        cache.k_scale.copy_(ramp[:, None] / 127)
        table, lens, cu = [list(range(40))], [1280], [0, 300]
        q = (_randn(g, 300, 2, 64) * 8).half()
        got = ops.attention_i8_cache(q.cuda(), cache, _i32(table), _i32(lens), engine=engine).cpu().double()
        want, tol = _attention_reference(q, cache, table, lens, cu, 2, True, 0, 0, 1 / 8)
        assert ((got - want).abs() <= tol).all(), engine


def test_long_context_and_many_sequences(cuda_device, nnb200_lib):
    g = _gen(3)
    _check_attention(g, torch.float16, 2, 4, 128, 128, [40001], [3])
    _check_attention(g, torch.float16, 1, 4, 128, 16, [40001, 39000], [2, 1], window=3000, sinks=4)
    _check_attention(g, torch.float16, 1, 4, 128, 16, [20001, 9000], [70, 64], engine="tile")
    _check_attention(g, torch.float16, 1, 2, 64, 16, [(37 * i) % 300 for i in range(1100)], [i % 3 for i in range(1100)], engine="tile")
    lens = [(37 * i) % 300 for i in range(700)]
    _check_attention(g, torch.bfloat16, 1, 2, 64, 16, lens, [1] * 700, uniform=True)
    _check_attention(g, torch.float16, 1, 2, 64, 16, lens, [i % 4 for i in range(700)])


def test_a_cache_past_32_bits(cuda_device, nnb200_lib):
    """Pages whose codes lie beyond 2^32 bytes: the last ones of a cache of 4.4 GB."""
    tokens, heads, dim = 128, 8, 256
    pages = (1 << 32) // (tokens * heads * dim) + 800
    k = torch.zeros((pages, heads, tokens, dim), dtype=torch.int8, device="cuda")
    cache = ops.CacheI8(k, k, *(torch.zeros((pages, heads), device="cuda") for _ in range(2)))
    g = _gen(9)
    table = [[pages - 1, 3, pages - 700]]
    x = _randn(g, 300, heads, dim).half()
    ops.cache_write_i8(cache, x.cuda(), x.cuda(), _i32(table), _i32([300]))
    got = ops.cache_read_i8(cache, _i32(table), _i32([300]), rows=300)
    plain = _Plain(3, heads, tokens, dim)
    plain.write(x, x, [[0, 1, 2]], [300], [0, 300])
    assert torch.equal(got[0].cpu(), plain.values(0, [0, 1, 2], 300).half())
    q = _randn(g, 2, heads, dim).half()
    o = ops.attention_i8_cache(q.cuda(), cache, _i32(table), _i32([300]))
    small = ops.CacheI8(*(c.cuda() for c in plain.codes), *(s.cuda() for s in plain.scale))
    assert torch.equal(o, ops.attention_i8_cache(q.cuda(), small, _i32([[0, 1, 2]]), _i32([300])))


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_rows_and_pages(cuda_device, nnb200_lib, dtype):
    """Queries out of a fused product, off the 16-byte rule; keys and values of a page next to each other; an output
    with room between its heads."""
    g = _gen(8)
    lens, new, heads, group, dim, tokens = [50, 21], [3, 2], 2, 2, 64, 16
    table, pages = _tables(g, lens, tokens)
    plain = _filled(g, pages, heads, tokens, dim)
    both = torch.stack([plain.k, plain.v], 1)
    scales = torch.stack([plain.k_scale, plain.v_scale], 1)
    cache = ops.CacheI8(both[:, 0], both[:, 1], scales[:, 0], scales[:, 1])
    q = torch.zeros((5, 4, dim + 3), dtype=dtype, device="cuda")[..., 1:dim + 1]
    q.copy_(_randn(g, 5, 4, dim))
    out = torch.full((5, 4, dim + 1), 9.0, dtype=dtype, device="cuda")
    got = ops.attention_i8_cache(q, cache, _i32(table), _i32(lens), cu=_i32(_cu(new)), out=out[..., :dim])
    assert (out[..., dim:] == 9).all()
    assert torch.equal(got, ops.attention_i8_cache(q.contiguous(), plain, _i32(table), _i32(lens), cu=_i32(_cu(new))))


def test_extreme_scales_and_values(cuda_device, nnb200_lib):
    """Blocks of zeros, blocks whose values are a million times others', queries beyond f16, and a first token that sees only itself."""
    g = _gen(4)
    cache = _filled(g, 5, 1, 16, 64)
    cache.k_scale.fill_(0.01)
    for scales in ([1.0, 1e-6, 1e-6, 1e-6, 1.0], [1e-6, 1.0, 1e6, 1.0, 1e-6], [0.0, 1.0, 0.0, 1.0, 1.0]):
        cache.v_scale.copy_(torch.tensor(scales)[:, None])
        for page in range(5):
            if scales[page] == 0:
                cache.v[page] = 0
        table, lens, cu = [[0, 1, 2, 3, 4]], [80], [0, 80]
        for dtype in (torch.float32, torch.bfloat16):
            q = (_randn(g, 80, 2, 64) * 4).to(dtype)
            got = ops.attention_i8_cache(q.cuda(), cache, _i32(table), _i32(lens)).cpu().double()
            want, tol = _attention_reference(q, cache, table, lens, cu, 2, True, 0, 0, 1 / 8)
            assert ((got - want).abs() <= tol).all()
            assert (got[0] - want[0]).abs().max() <= 2.0 ** -7 * want[0].abs().max()
    cache.v_scale.fill_(1.0)
    q = _randn(g, 1, 2, 64) * 1e6
    cache.k_scale.fill_(1e-7)
    got = ops.attention_i8_cache(q.cuda(), cache, _i32([[0, 1]]), _i32([20])).cpu().double()
    want, tol = _attention_reference(q, cache, [[0, 1]], [20], [0, 1], 2, True, 0, 0, 1 / 8)
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype,engine", [*((t, "rows") for t in TYPES), (torch.float16, "tile"), (torch.bfloat16, "tile")])
def test_what_is_masked_may_be_anything(cuda_device, nnb200_lib, dtype, engine):
    """Scales of NaN and infinity on pages that a row does not see, or sees none of; queries that are NaN stay their own."""
    g = _gen(6)
    cache = _filled(g, 4, 1, 16, 64)
    clean = ops.CacheI8(cache.k, cache.v, cache.k_scale.clone(), cache.v_scale.clone())
    q = _randn(g, 60, 2, 64).to(dtype).cuda()
    table = _i32([[0, 1, 2, 3]])
    want = ops.attention_i8_cache(q, clean, table, _i32([60]), engine=engine)
    for bad in (math.nan, math.inf):
        for scale in (cache.k_scale, cache.v_scale):
            cache.k_scale.copy_(clean.k_scale)
            cache.v_scale.copy_(clean.v_scale)
            scale[2] = bad
            got = ops.attention_i8_cache(q, cache, table, _i32([60]), engine=engine)
            assert torch.equal(got[:32], want[:32])
            assert not got[32:].isfinite().any() if scale is cache.v_scale or bad != bad else True
            got = ops.attention_i8_cache(q[50:], cache, table, _i32([60]), window=3, sinks=20, engine=engine)
            assert got.isfinite().all()
    q[7, 1, 3] = math.nan
    got = ops.attention_i8_cache(q, clean, table, _i32([60]), engine=engine)
    assert got[7, 1].isnan().all()
    rest = torch.ones((60, 2), dtype=torch.bool, device="cuda")
    rest[7, 1] = False
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("engine", ["rows", "tile"])
def test_rows_that_see_nothing_whatever_they_hold(cuda_device, nnb200_lib, engine):
    """The padding of a batch: rows before their sequence's first token, and of sequences without one, give zeros."""
    g = _gen(17)
    for dim in (64, 256):
        cache = _filled(g, 4, 1, 16, dim)
        q = _randn(g, 12, 2, dim).half().cuda()
        table, lens, cu = _i32([[0, 1], [2, 3]]), _i32([0, 5]), _i32([0, 4, 12])
        want = ops.attention_i8_cache(q, cache, table, lens, cu=cu, engine=engine)
        assert (want[:7] == 0).all() and (want[7:] != 0).any()
        for bad in (math.nan, math.inf):
            q[:7] = bad
            assert torch.equal(ops.attention_i8_cache(q, cache, table, lens, cu=cu, engine=engine), want)
            assert (ops.attention_i8_cache(q[:4], cache, table[:1], _i32([0]), causal=False, engine=engine) == 0).all()


@pytest.mark.parametrize("engine", ["rows", "tile"])
@pytest.mark.parametrize("window", [100, 2 ** 31, 2 ** 62, 2 ** 63 - 1])
def test_a_window_beyond_everything(cuda_device, nnb200_lib, engine, window):
    g = _gen(18)
    cache = _filled(g, 4, 1, 16, 64)
    q = _randn(g, 60, 2, 64).half().cuda()
    for lens, cu in ((_i32([60]), None), (_i32([50]), None), (_i32([60]), _i32([0, 60]))):    # (50: ten rows stand before the sequence)
        want = ops.attention_i8_cache(q, cache, _i32([[0, 1, 2, 3]]), lens, cu=cu, engine=engine)
        for sinks in (0, 2 ** 63 - 1):
            assert torch.equal(ops.attention_i8_cache(q, cache, _i32([[0, 1, 2, 3]]), lens, cu=cu, window=window, sinks=sinks, engine=engine), want)


def test_no_page_for_a_sequence_that_begins_behind_rows_without_a_token(cuda_device, nnb200_lib):
    """Read: rows before the sequence and rows whose first page is wrong are zeros, all of them."""
    g = _gen(19)
    cache = _filled(g, 3, 2, 16, 64)
    out = tuple(torch.full((40, 2, 64), math.nan, dtype=torch.float16, device="cuda") for _ in range(2))
    ops.cache_read_i8(cache, _i32([[-1, 2]]), _i32([20]), out=out)
    assert capi.take_device_error() == capi.DEVICE_ERROR_BAD_PAGE
    for x in out:
        assert (x[:36] == 0).all() and x.isfinite().all() and (x[36:] != 0).any()


@pytest.mark.parametrize("engine", [1, 2])
def test_rows_that_several_sequences_claim(cuda_device, nnb200_lib, engine):
    """`cu` that goes up and down: what such rows hold is not defined, but the workspace is enough and nobody else's rows change."""
    g = _gen(20)
    seqs, rows = 50, 600
    cache = _filled(g, 4, 1, 16, 64)
    q = _randn(g, rows + 8, 2, 64).half().cuda()
    out = torch.full_like(q, 7.0)
    table, lens, cu = _i32([[0, 1, 2, 3]] * seqs), _i32([64] * seqs), _i32([0, rows] * (seqs // 2) + [0])
    a = capi.block(capi.AttentionI8Args, *ops._sequences(cache, table, lens, cu, rows), q.data_ptr(), out.data_ptr(), *q.stride()[:2], *out.stride()[:2], 2, 0, 0,
                   0.125, 1, capi.FLOAT_F16, engine)
    need = nnb200_lib.nnb200_attention_i8_workspace_bytes(C.byref(a))
    space = torch.full((need + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = space.data_ptr(), need
    capi.check(nnb200_lib.nnb200_attention_i8(C.byref(a), None), "nnb200_attention_i8")
    torch.cuda.synchronize()
    assert (space[need:] == 0x5A).all() and (out[rows:] == 7).all() and out.isfinite().all() and capi.take_device_error() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 96, 256])
def test_strided_rows_in_tiles(cuda_device, nnb200_lib, dtype, dim):
    """Queries and outputs off the 16-byte rule, and off the 32-byte one only; heads before rows."""
    g = _gen(22)
    lens, new, group = [500, 21], [290, 2], 3
    table, pages = _tables(g, lens, 32)
    cache = _filled(g, pages, 2, 32, dim)
    rest = (_i32(table), _i32(lens))
    dense = _randn(g, 292, 6, dim).to(dtype).cuda()
    want = ops.attention_i8_cache(dense, cache, *rest, cu=_i32(_cu(new)), engine="tile")
    for shape, at in (((292, 6, dim + 3), 1), ((292, 6, dim + 8), 8)):
        q = torch.zeros(shape, dtype=dtype, device="cuda")[..., at: at + dim].copy_(dense)
        out = torch.full(shape, 9.0, dtype=dtype, device="cuda")
        got = ops.attention_i8_cache(q, cache, *rest, cu=_i32(_cu(new)), out=out[..., at: at + dim], engine="tile")
        assert torch.equal(got, want) and (out[..., :at] == 9).all() and (out[..., at + dim:] == 9).all()
    turned = dense.transpose(0, 1).contiguous().transpose(0, 1)
    out = torch.empty((6, 292, dim), dtype=dtype, device="cuda").transpose(0, 1)
    for engine in ("tile", "rows"):
        got = ops.attention_i8_cache(turned, cache, *rest, cu=_i32(_cu(new)), out=out, engine=engine)
        assert torch.equal(got, want if engine == "tile" else ops.attention_i8_cache(dense, cache, *rest, cu=_i32(_cu(new)), engine="rows"))


def test_lengths_and_pages_that_are_wrong(cuda_device, nnb200_lib):
    """Nothing outside the arrays is touched: wrong pages are left out and recorded, wrong lengths and rows are cut."""
    g = _gen(2)
    cache = _filled(g, 4, 1, 16, 64)
    q = _randn(g, 1, 2, 64).half().cuda()
    good = ops.attention_i8_cache(q, cache, _i32([[0, 1]]), _i32([32]))
    for page in (-1, 4, 2 ** 31 - 1, -2 ** 31):
        before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
        got = ops.attention_i8_cache(q, cache, _i32([[0, 1, page]]), _i32([48]))
        assert capi.take_device_error() == capi.DEVICE_ERROR_BAD_PAGE
        assert torch.equal(got, good)
        x = torch.ones((48, 1, 64), dtype=torch.float16, device="cuda")
        ops.cache_write_i8(cache, x[:16], x[:16], _i32([[0, 1, page]]), _i32([48]))
        assert capi.take_device_error() == capi.DEVICE_ERROR_BAD_PAGE
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.k, cache.v, cache.k_scale, cache.v_scale)))
        k, _ = ops.cache_read_i8(cache, _i32([[0, page, 1]]), _i32([48]), rows=48)
        assert capi.take_device_error() == capi.DEVICE_ERROR_BAD_PAGE
        assert (k[16:32] == 0).all() and (k[:16] != 0).any() and (k[32:] != 0).any()
    assert torch.equal(ops.attention_i8_cache(q, cache, _i32([[0, 1]]), _i32([10 ** 9])), good)
    assert (ops.attention_i8_cache(q, cache, _i32([[0, 1]]), _i32([-5])) == 0).all()
    out = torch.full_like(q, 3.0)
    for cu in ([5, 9], [-7, -2], [2 ** 31 - 1, 0]):
        ops.attention_i8_cache(q, cache, _i32([[0, 1]]), _i32([32]), cu=_i32(cu), out=out)
        ops.cache_write_i8(cache, q[:, :1], q[:, :1], _i32([[0, 1]]), _i32([32]), cu=_i32(cu))
    assert (out == 3).all() and capi.take_device_error() == 0


# ---- streams, graphs, together ----------------------------------------------------------------------

def test_captured_calls_follow_their_arrays(cuda_device, nnb200_lib):
    """A decode step is captured once and replayed as the sequences grow; eager calls on another stream run meanwhile."""
    g = _gen(12)
    heads, group, dim, tokens, seqs = 2, 4, 128, 16, 3
    table = torch.arange(seqs * 8, dtype=torch.int32, device="cuda").view(seqs, 8)
    cache, plain = ops.CacheI8.empty(seqs * 8, heads, tokens, dim, "cuda"), _Plain(seqs * 8, heads, tokens, dim)
    lens = _i32([13, 30, 1])
    q, k, v = (torch.zeros((seqs, h, dim), dtype=torch.float16, device="cuda") for h in (heads * group, heads, heads))
    prompt = _randn(g, 44, heads, dim).half()
    ops.cache_write_i8(cache, prompt.cuda(), prompt.cuda(), table, lens, cu=_i32([0, 13, 43, 44]))
    plain.write(prompt, prompt, table.tolist(), lens.tolist(), [0, 13, 43, 44])
    big = _filled(g, 64, heads, tokens, dim)
    big_q = _randn(g, 1, heads * group, dim).half().cuda()
    big_table, big_lens = torch.arange(64, dtype=torch.int32, device="cuda")[None], _i32([1000])
    big_want = ops.attention_i8_cache(big_q, big, big_table, big_lens)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.cache_write_i8(cache, k, v, table, lens)
        out = ops.attention_i8_cache(q, cache, table, lens)
    for step in range(20):
        fresh = [(1 + 0.2 * step) * _randn(g, *t.shape) for t in (q, k, v)]
        for t, x in zip((q, k, v), fresh):
            t.copy_(x)
        lens += 1
        with torch.cuda.stream(side):
            big_got = ops.attention_i8_cache(big_q, big, big_table, big_lens)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(big_got, big_want)
        plain.write(fresh[1].half(), fresh[2].half(), table.tolist(), lens.tolist(), [0, 1, 2, 3])
        assert _same(cache, plain)
        want, tol = _attention_reference(fresh[0].half(), cache, table.tolist(), lens.tolist(), [0, 1, 2, 3], group, True, 0, 0, 1 / math.sqrt(dim))
        assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("engine,new", [("tile", 90), ("rows", 2)])
def test_two_graphs_and_eager_calls_between_them(cuda_device, nnb200_lib, engine, new):
    """Captured calls whose tables, lengths and rows change between replays; two graphs on two streams at once, and eager calls on a third:
    each has a workspace of its own."""
    g = _gen(23)
    heads, group, dim, tokens, seqs = 2, 4, 64, 32, 3
    table, pages = _tables(g, [2000, 1500, 900], tokens)
    cache = _filled(g, pages, heads, tokens, dim)
    table = _i32(table)
    streams, graphs, calls = [torch.cuda.Stream() for _ in range(3)], [], []
    for i in range(2):
        lens, cu, q = _i32([1, 1, 1]), _i32([0, 1, 2, 3]), torch.zeros((seqs * new, heads * group, dim), dtype=torch.float16, device="cuda")
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = ops.attention_i8_cache(q, cache, table, lens, cu=cu, engine=engine)
        graphs.append(graph)
        calls.append((q, lens, cu, out))
    for step in range(6):
        want = []
        for i, (q, lens, cu, out) in enumerate(calls):
            q.copy_(_randn(g, *q.shape))
            lens.copy_(torch.tensor([2000 - 300 * step, 10 + 200 * step, 900 - i]))
            cu.copy_(torch.tensor([0, new - step % 2, 2 * new - step % 2, 3 * new]))
            out.zero_()
            want.append(ops.attention_i8_cache(q, cache, table, lens, cu=cu, engine=engine))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = ops.attention_i8_cache(calls[0][0], cache, table, calls[0][1], cu=calls[0][2], engine=engine)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[0]) and all(torch.equal(call[3], w) for call, w in zip(calls, want)), step


@pytest.mark.parametrize("name", ["norm", "norm, residual", "norm, buffers", "write", "read", "attention", "attention, window"])
def test_same_bytes_from_the_python_code(cuda_device, nnb200_lib, monkeypatch, name):
    """The compiled front end takes the call, and the Python code behind it does the same."""
    def calls():
        g = _gen(3)
        x, r, w = _randn(g, 5, 264).half().cuda(), _randn(g, 5, 264).half().cuda(), _randn(g, 264).cuda()
        cache = _filled(g, 6, 2, 16, 64)
        q, k = _randn(g, 4, 4, 64).half().cuda(), _randn(g, 4, 2, 64).half().cuda()
        table, lens, cu = _i32([[1, 2, 3], [4, 5, 0]]), _i32([40, 33]), _i32([0, 1, 4])
        return {
            "norm": lambda: ops.rms_norm_i8(x, w),
            "norm, residual": lambda: ops.rms_norm_i8(x, w.half(), residual=r, eps=1e-3),
            "norm, buffers": lambda: ops.rms_norm_i8(x, w, residual=r, residual_out=r, out=torch.empty((5, 264), dtype=torch.int8, device="cuda"),
                                                     scale=torch.empty(5, device="cuda")),
            "write": lambda: (ops.cache_write_i8(cache, k, k, table, lens, cu=cu), cache.k, cache.v, cache.k_scale, cache.v_scale)[1:],
            "read": lambda: ops.cache_read_i8(cache, table, lens, rows=4, cu=cu, out_dtype=torch.bfloat16),
            "attention": lambda: (ops.attention_i8_cache(q, cache, table, lens),),
            "attention, window": lambda: (ops.attention_i8_cache(q, cache, table, lens, cu=cu, window=7, sinks=2, scale=0.1, out=torch.empty_like(q)),),
        }[name]

    taken = []

    class Recorder:
        def __init__(self, front):
            self.front = front

        def __getattr__(self, f):
            def call(*args):
                made = getattr(self.front, f)(*args)
                taken.append(made is not None)
                return made
            return call

    monkeypatch.setattr(ops, "_native", Recorder(ops._front()))
    got = [t.clone() for t in calls()()]
    assert taken == [True]
    monkeypatch.setattr(ops, "_native", ops._NoFront())
    want = calls()()
    assert len(got) == len(want) and all(torch.equal(a, b) and a.dtype == b.dtype for a, b in zip(got, want))


@pytest.mark.parametrize("captured", [False, True])
@pytest.mark.parametrize("new,ragged", [(1, False), (1, True), (5, True), (90, True), (90, False)])
def test_a_stream_of_steps_without_waiting(cuda_device, nnb200_lib, new, ragged, captured):
    """Kernels that begin while the one before ends: each step's calls read what the last call wrote and write over what the one before it
    read, buffers and scratch the same ones again and again.  With a synchronisation behind each call, without, and as one graph."""
    g = _gen(31 + new)
    seqs, width, heads, group, dim, tokens, steps = 4, 512, 2, 4, 64, 16, 6
    rows = seqs * new
    w_qkv = torch.randint(-127, 128, ((group + 2) * heads * dim, width), generator=g, dtype=torch.int32).to(torch.int8).cuda()
    w_out = torch.randint(-127, 128, (width, heads * group * dim), generator=g, dtype=torch.int32).to(torch.int8).cuda()
    norms = [(1 + 0.1 * _randn(g, width)).half().cuda() for _ in range(2)]
    x0 = _randn(g, rows, width).half().cuda()
    table = _i32(torch.randperm(seqs * 64, generator=g).view(seqs, 64).tolist())
    starts = _i32([3, 200, 17, 64])
    cu = _i32(_cu([new] * seqs)) if ragged else None
    cache = ops.CacheI8.empty(seqs * 64, heads, tokens, dim, "cuda")
    before = _randn(g, 284, heads, dim).half().cuda()
    per_row, zeros = torch.full((rows,), 0.02, device="cuda"), torch.zeros(rows, dtype=torch.int8, device="cuda")

    def chain(after):
        ops.cache_write_i8(cache, before, before, table, starts, cu=_starts)
        after()
        x, lens, seen = x0.clone(), starts.clone(), []
        codes, scale = torch.empty((rows, width), dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
        o = torch.empty((rows, heads * group, dim), dtype=torch.float16, device="cuda")
        for _ in range(steps):
            lens += new
            ops.rms_norm_i8(x, norms[0], out=codes, scale=scale)
            after()
            qkv = ops.gemm_i8(codes, w_qkv, out_kind="f16", scale_a=scale, scale_w=1e-3).view(rows, -1, dim)
            after()
            ops.cache_write_i8(cache, qkv[:, heads * group: -heads], qkv[:, -heads:], table, lens, cu=cu)
            after()
            ops.attention_i8_cache(qkv[:, : heads * group], cache, table, lens, cu=cu, out=o)
            after()
            q = ops.quantize_linear(o.view(rows, -1), per_row, zeros)
            after()
            y = ops.gemm_i8(q, w_out, out_kind="f16", scale_a=0.02, scale_w=1e-3)
            after()
            ops.rms_norm_i8(y, norms[1], residual=x, residual_out=x, out=codes, scale=scale)
            after()
            seen += [codes.clone(), scale.clone(), x.clone(), o.clone(), ops.cache_read_i8(cache, table, lens, rows=rows, cu=cu)[1]]
            after()
        return seen + [cache.k.clone(), cache.v_scale.clone()]

    _starts = _i32(_cu(starts.tolist()))
    want = [t.clone() for t in chain(torch.cuda.synchronize)]
    assert all(t.float().isfinite().all() for t in want) and not torch.equal(want[0], want[5])
    if captured:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            got = chain(lambda: None)
    for _ in range(4):
        if captured:
            graph.replay()
        else:
            got = chain(lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True))


def test_a_block_of_a_model(cuda_device, nnb200_lib):
    """Norm, int8 product into q, k and v, cache, attention, int8 product, norm: a prompt and then tokens one by one."""
    g = _gen(21)
    width, heads, group, dim, tokens = 512, 2, 4, 64, 16
    wide = (group + 2) * heads * dim
    w_qkv = torch.randint(-127, 128, (wide, width), generator=g, dtype=torch.int32).to(torch.int8)
    w_out = torch.randint(-127, 128, (width, heads * group * dim), generator=g, dtype=torch.int32).to(torch.int8)
    s_qkv, s_out = (torch.rand(n, generator=g) * 1e-3 + 5e-4 for n in (wide, width))
    norms = [(1 + 0.1 * _randn(g, width)).half() for _ in range(2)]
    table = [[5, 2, 7, 0]]
    cache, plain = ops.CacheI8.empty(8, heads, tokens, dim, "cuda"), _Plain(8, heads, tokens, dim)
    length = 0
    for n in (37, 1, 1, 1, 5):
        length += n
        x = _randn(g, n, width).half()
        codes, scale = ops.rms_norm_i8(x.cuda(), norms[0].cuda())
        want, _, _ = _norm_reference(x, norms[0], None, 1e-6)
        assert torch.equal(codes.cpu(), want)
        qkv = ops.gemm_i8(codes, w_qkv.cuda(), out_kind="f16", scale_a=scale, scale_w=s_qkv.cuda()).view(n, -1, dim)
        exact = (want.double() @ w_qkv.double().T * scale.cpu().double()[:, None] * s_qkv.double()).view(n, -1, dim)
        assert ((qkv.cpu().double() - exact).abs() <= 2.0 ** -10 * exact.abs() + 2.0 ** -24).all()
        q, k, v = qkv[:, : heads * group], qkv[:, heads * group: -heads], qkv[:, -heads:]
        ops.cache_write_i8(cache, k, v, _i32(table), _i32([length]))
        plain.write(k.cpu(), v.cpu(), table, [length], [0, n])
        assert _same(cache, plain)
        o = ops.attention_i8_cache(q, cache, _i32(table), _i32([length]))
        want, tol = _attention_reference(q.cpu(), cache, table, [length], [0, n], group, True, 0, 0, 1 / 8)
        assert ((o.cpu().double() - want).abs() <= tol).all()
        flat = o.view(n, -1)
        top = flat.float().abs().amax(1) / 127
        oq = ops.quantize_linear(flat, top, torch.zeros(n, dtype=torch.int8, device="cuda"))
        y = ops.gemm_i8(oq, w_out.cuda(), out_kind="f16", scale_a=top, scale_w=s_out.cuda())
        codes, scale, h = ops.rms_norm_i8(y, norms[1].cuda(), residual=x.cuda())
        want, exact, sum_ = _norm_reference(y.cpu(), norms[1], x, 1e-6)
        assert torch.equal(codes.cpu(), want) and torch.equal(h.cpu(), sum_) and ((scale.cpu().double() - exact).abs() <= 2.0 ** -22 * exact).all()


@pytest.mark.parametrize("compiled", [True, False])
def test_a_cache_that_is_given_larger_tensors(cuda_device, nnb200_lib, monkeypatch, compiled):
    """Between two calls a cache gets more pages: what it held is carried over by its owner, and nobody writes to the old tensors again."""
    if not compiled:
        monkeypatch.setattr(ops, "_native", ops._NoFront())
    g = _gen(29)
    cache = ops.CacheI8.empty(2, 2, 16, 64, "cuda")
    x = _randn(g, 70, 2, 64).half().cuda()
    ops.cache_write_i8(cache, x[:30], x[:30], _i32([[1, 0]]), _i32([30]))
    old = cache.k, cache.v, cache.k_scale, cache.v_scale
    kept = [t.clone() for t in old]
    cache.k, cache.v, cache.k_scale, cache.v_scale = (torch.cat([t, torch.zeros_like(t), torch.zeros_like(t)]) for t in old)
    assert cache.pages == 6
    table = _i32([[1, 0, 5, 3, 2]])
    ops.cache_write_i8(cache, x[30:], x[30:], table, _i32([70]))
    q = _randn(g, 1, 4, 64).half().cuda()
    got = ops.attention_i8_cache(q, cache, table, _i32([70]))
    assert all(torch.equal(a, b) for a, b in zip(old, kept))
    whole = ops.CacheI8.empty(6, 2, 16, 64, "cuda")
    for low, high in ((0, 30), (30, 70)):
        ops.cache_write_i8(whole, x[low:high], x[low:high], table, _i32([high]))
    assert torch.equal(cache.k, whole.k) and torch.equal(cache.v_scale, whole.v_scale) and capi.take_device_error() == 0
    assert torch.equal(got, ops.attention_i8_cache(q, whole, table, _i32([70])))
    assert all(torch.equal(a, b) for a, b in zip(ops.cache_read_i8(cache, table, _i32([70]), rows=70), ops.cache_read_i8(whole, table, _i32([70]), rows=70)))


@pytest.mark.parametrize("compiled", [True, False])
@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_rows_without_columns(cuda_device, nnb200_lib, monkeypatch, dtype, compiled):
    """A mean over nothing is no number, and says so: the scale is written whatever stood there."""
    if not compiled:
        monkeypatch.setattr(ops, "_native", ops._NoFront())
    x, scale = torch.empty((5, 0), dtype=dtype, device="cuda"), torch.ones(5, device="cuda")
    for residual in (None, torch.empty((5, 0), dtype=dtype, device="cuda")):
        scale.fill_(1.0)
        got = ops.rms_norm_i8(x, torch.empty(0, dtype=dtype, device="cuda"), residual=residual, scale=scale)
        assert got[1] is scale or got[1].data_ptr() == scale.data_ptr()
        assert scale.isnan().all() and got[0].shape == (5, 0)
