"""Attention over the 8-bit cache where few bits would show: weights far below a row's largest, queries with one loud channel,
large scores, long contexts of which every token counts.  Each row's output is compared as a vector with 64 bits, relative to its own length."""
import math

import pytest
import torch

from nnops_b200 import ops

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
FORMS = [(torch.float16, "rows"), (torch.bfloat16, "rows"), (torch.float32, "rows"), (torch.float16, "tile"), (torch.bfloat16, "tile")]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _exact(q, codes, scales, pages, length, group, window=0, sinks=0, without=None):
    """One sequence in 64 bits: the rows' outputs, and (largest of p vs) * sqrt(sum of codes^2) of each, relative to the output's length:
    what all weights being off by 1 where the largest is 1 come to, if each is off by itself.  `without`: tokens that are left out."""
    n, dim = q.shape[0], q.shape[2]
    ids = torch.tensor(pages, dtype=torch.long)
    k, v = ((c[ids].double() * s[ids].double()[..., None, None]).transpose(1, 2).flatten(0, 1)[:length] for c, s in zip(codes, scales))
    raw = codes[1][ids].double().transpose(1, 2).flatten(0, 1)[:length]
    each = scales[1][ids].double()[:, None].expand(-1, codes[1].shape[2], -1).flatten(0, 1)[:length]
    pos, j = length - n + torch.arange(n), torch.arange(length)
    seen = j[None] <= pos[:, None]
    if window:
        seen &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
    if without is not None:
        seen = seen & ~((j >= without[0]) & (j < without[1]))[None]
    out, least, top = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape[:2], dtype=torch.float64), 0.0
    for a in range(q.shape[1]):
        h = a // group
        z = torch.where(seen, q[:, a].double() @ k[:, h].T / math.sqrt(dim), -math.inf)
        p = torch.softmax(z, 1)
        out[:, a] = p @ v[:, h]
        largest = (p * each[:, h]).amax(1)
        least[:, a] = largest * (seen.double() @ raw[:, h].square().sum(1)).sqrt() / out[:, a].norm(dim=1)
        # Of a row's exponents, in powers of two: the span that its scores and the values' scales take.
        top = max(top, ((z.masked_fill(~seen, 0).abs().amax() * 1.4427) + each[:, h].log2().abs().amax()).item())
    return out, least, top


def _bound(dtype, top, least):
    """Relative to the output's length.  A weight's exponent is the rounded product of a score, a scale and a factor, and a rounded sum: four
    roundings of at most half a step of its size (`top`, up to the next power of two), times ln 2, and ex2's 2^-22; both in the sum of the
    weights and in the products.  The weight itself: one f16 (half a step: 2^-11) or two (2^-22), or half of f16's least step, 2^-25,
    where the largest is at least 2^7 or 2^13.  f32 sums along one path of the tokens: at most 2^9 steps (tiles of 8192 tokens take 16 at a time) of 2^-24.
    Errors of the weights are each one's own, so that their sum grows as the output itself does; twice that for a row's luck."""
    exponent = 4 * 2.0 ** -25 * 2.0 ** math.ceil(math.log2(max(top, 1.0))) * math.log(2) + 2.0 ** -22
    split = dtype is torch.float32
    return (2 * exponent + 2 * (2.0 ** -22 if split else 2.0 ** -11) + (2.0 ** -20 if split else 2.0 ** -15) + HALF_STEP[dtype] +
            2 * least * (2.0 ** -38 if split else 2.0 ** -32))


def _distance(got, want):
    return (got - want).norm(dim=-1) / want.norm(dim=-1)


@pytest.mark.parametrize("dtype,engine", FORMS)
@pytest.mark.parametrize("lead", [8, 12, 14, 17])
@pytest.mark.parametrize("loud", [False, True])
def test_a_first_token_far_above_the_rest(cuda_device, nnb200_lib, dtype, engine, lead, loud):
    """Its score leads by so many nats and its values are zeros (`loud`: but for one channel, which is a thousand times the others'): the output is
    made of the weights of all the others."""
    g = torch.Generator().manual_seed(lead)
    length, dim, tokens, group, n = 8192, 128, 64, 4, 1 if engine == "rows" else 70
    pages = length // tokens
    sign = torch.randint(0, 2, (dim,), generator=g) * 2 - 1
    k, v = (torch.randint(-127, 128, (pages, 1, tokens, dim), generator=g, dtype=torch.int32).to(torch.int8) for _ in range(2))
    spread = 73.3 * math.sqrt(dim)    # of the sum of dim such codes, signs in front
    k[0, 0, 0] = (round(lead * spread / dim) * sign).to(torch.int8)
    v[0, 0, 0] = 0
    k_scale, v_scale = torch.full((pages, 1), math.sqrt(dim) / spread), torch.full((pages, 1), 0.01)
    if loud:
        v[..., 5], v[0, 0, :, :5], v[0, 0, :, 6:] = 0, 0, 0
        v[0, 0, 0, 5], v_scale[0] = 127, 10.0
    q = (sign * torch.tensor([1.0, 0.96875, 0.9375, 0.984375])[None, :, None]).expand(n, 4, dim).to(dtype)
    want, least, top = _exact(q, (k, v), (k_scale, v_scale), list(range(pages)), length, group)
    cache = ops.CacheI8(k.cuda(), v.cuda(), k_scale.cuda(), v_scale.cuda())
    got = ops.attention_i8_cache(q.cuda(), cache, _i32([list(range(pages))]), _i32([length]), engine=engine).cpu().double()
    assert abs(got[..., 5] / want[..., 5] - 1).max() <= _bound(dtype, top, torch.zeros(())) or not loud
    if loud:    # what is left, by itself: the loud channel's share of the largest weight is as large as with the scales alike
        got, want = (torch.cat([t[..., :5], t[..., 6:]], -1) for t in (got, want))
        least = torch.zeros_like(least)
        for a in range(4):
            z = torch.softmax(q[:, a].double() @ (k.double() * k_scale[..., None, None].double()).view(length, dim).T / math.sqrt(dim), 1)
            least[:, a] = (z[:, 0] * 10) * (v.double().square().sum() - 127 ** 2).sqrt() / want[:, a].norm(dim=1)
    off = _distance(got, want)
    assert (off <= _bound(dtype, top, least)).all(), (off.max().item(), _bound(dtype, top, least).min().item())


@pytest.mark.parametrize("dtype,engine", [f for f in FORMS if f[0] is not torch.float16])
@pytest.mark.parametrize("dim", [64, 256])
def test_a_loud_channel_of_the_queries(cuda_device, nnb200_lib, dtype, engine, dim):
    """2^14 (f32) or 2^20 (bf16) times the others, where keys have nothing: the scores are the other channels'."""
    g = torch.Generator().manual_seed(dim)
    length, tokens, group, n = 500, 16, 2, 40
    pages = -(-length // tokens)
    k, v = (torch.randint(-127, 128, (pages, 1, tokens, dim), generator=g, dtype=torch.int32).to(torch.int8) for _ in range(2))
    k[..., 3] = 0
    scales = torch.full((pages, 1), 1 / 73.3), torch.full((pages, 1), 0.01)
    q = torch.randn((n, 2, dim), generator=g)
    q[..., 3] = 2.0 ** 14 if dtype is torch.float32 else 2.0 ** 20
    q = q.to(dtype)
    want, least, top = _exact(q, (k, v), scales, list(range(pages)), length, group)
    cache = ops.CacheI8(k.cuda(), v.cuda(), *(s.cuda() for s in scales))
    got = ops.attention_i8_cache(q.cuda(), cache, _i32([list(range(pages))]), _i32([length]), engine=engine).cpu().double()
    # Besides: a query's values to 2^-22 of each, and its product with a key in dim / 16 steps of 2^-23 of what its terms come to.
    products = (q.double().abs() @ k.double().abs().flatten(0, 2).T / 73.3 / math.sqrt(dim)).amax(-1)
    products[...] = products.amax()
    off = _distance(got, want)
    bound = _bound(dtype, top, least) + 2 * (2.0 ** -22 + dim / 16 * 2.0 ** -23) * products
    assert (off <= bound).all(), (off.max().item(), bound.min().item())


@pytest.mark.parametrize("dtype,engine", [f for f in FORMS if f[0] is not torch.float16])
@pytest.mark.parametrize("power", [-113, -100, -60, 60, 100, 113, 126])
def test_queries_of_any_size(cuda_device, nnb200_lib, dtype, engine, power):
    """Queries of 2^power against keys of 2^-power: the scores of ordinary ones, from the same bits; nothing overflows on the way."""
    g = torch.Generator().manual_seed(5)
    length, dim, tokens, n = 200, 64, 16, 20
    pages = -(-length // tokens)
    k, v = (torch.randint(-127, 128, (pages, 1, tokens, dim), generator=g, dtype=torch.int32).to(torch.int8) for _ in range(2))
    scales = torch.full((pages, 1), 2.0 ** -6), torch.full((pages, 1), 2.0 ** -7)
    q = torch.randn((n, 2, dim), generator=g).clamp(-1.9, 1.9).to(dtype)
    want, least, top = _exact(q, (k, v), scales, list(range(pages)), length, 2)
    cache = ops.CacheI8(k.cuda(), v.cuda(), (scales[0] * 2.0 ** -power).cuda(), scales[1].cuda())
    got = ops.attention_i8_cache((q.double() * 2.0 ** power).to(dtype).cuda(), cache, _i32([list(range(pages))]), _i32([length]), engine=engine)
    products = (q.double().abs() @ k.double().abs().flatten(0, 2).T * 2.0 ** -6 / math.sqrt(dim)).amax()
    off = _distance(got.cpu().double(), want)
    bound = _bound(dtype, top, least) + 2 * (2.0 ** -22 + dim / 16 * 2.0 ** -23) * products
    assert (off <= bound).all(), (off.max().item(), bound.min().item())


@pytest.mark.parametrize("dtype,engine,dim,lens,new,window,sinks", [
    (torch.float16, "rows", 128, [40001], [3], 0, 0),
    (torch.float32, "rows", 128, [40001, 17], [1, 1], 0, 0),
    (torch.float16, "rows", 64, [9000], [1], 0, 0),
    (torch.float32, "rows", 96, [9000, 5000], [4, 4], 0, 0),
    (torch.bfloat16, "rows", 256, [12000, 300], [2, 9], 0, 0),
    (torch.float16, "rows", 128, [40001, 39000], [2, 1], 3000, 4),
    (torch.float16, "tile", 128, [20001, 9000], [70, 64], 0, 0),
    (torch.float16, "tile", 64, [20001, 600], [300, 20], 0, 0),
    (torch.bfloat16, "tile", 96, [7000], [90], 2500, 100),
    (torch.float16, "tile", 256, [9001, 130], [80, 130], 0, 0),
])
@pytest.mark.parametrize("wide", [False, True])
def test_every_token_counts(cuda_device, nnb200_lib, dtype, engine, dim, lens, new, window, sinks, wide):
    """Long contexts whose outputs change by more than the bound when 64 tokens are left out (shown on the exact sums).  `wide`: a table
    with room for more, so that single tokens go by the line and its second kernel too."""
    g = torch.Generator().manual_seed(dim + len(lens))
    tokens, group, heads = 16, 4, 1
    need = [-(-n // tokens) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=g).tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * ((4000 if wide else max(need)) - n))
        at += n
    codes = [torch.randint(-127, 128, (sum(need) + 2, heads, tokens, dim), generator=g, dtype=torch.int32).to(torch.int8) for _ in range(2)]
    scales = [torch.exp(0.3 * torch.randn((sum(need) + 2, heads), generator=g)) / 80 for _ in range(2)]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn((cu[-1], heads * group, dim), generator=g).to(dtype)
    cache = ops.CacheI8(*(c.cuda() for c in codes), *(s.cuda() for s in scales))
    uniform = len(set(new)) == 1
    got = ops.attention_i8_cache(q.cuda(), cache, _i32(table), _i32(lens), cu=None if uniform else _i32(cu), window=window, sinks=sinks, engine=engine)
    got = got.cpu().double()
    for b, length in enumerate(lens):
        x = q[cu[b]:cu[b + 1]]
        want, least, top = _exact(x, codes, scales, table[b][: need[b]], length, group, window, sinks)
        # A product's dim / 16 steps of 2^-23 of its terms, which scores of one deviation stay within 6 deviations of.
        bound = _bound(dtype, top, least) + 2 * (2.0 ** -22 + dim / 16 * 2.0 ** -23) * 6 * math.sqrt(dim)
        off = _distance(got[cu[b]:cu[b + 1]], want)
        assert (off <= bound).all(), (b, off.max().item(), bound.min().item())
        if length > 1000:
            first = length - min(length, window or length) // 2 // tokens * tokens
            lost = _exact(x, codes, scales, table[b][: need[b]], length, group, window, sinks, without=(first, first + 4 * tokens))[0]
            assert (_distance(lost, want) > bound).double().mean() > 0.95


@pytest.mark.parametrize("dtype,engine,size", [(*f, s) for f in FORMS for s in (0, 10, 20, 22, 23, 24, 25, 26, 27, 28, 30, 60)
                                               if f[1] == "rows" or s <= 25])    # tiles: as far as the header says
def test_scores_of_any_size(cuda_device, nnb200_lib, dtype, engine, size):
    """Scores up to 2^size that grow along the tokens in steps of 1 / 127 of it, and stand still where they are largest: the values of three tokens, of
    different pages, are what is left, also where the steps of f32 are larger than any that matters."""
    g = torch.Generator().manual_seed(size)
    dim, tokens, group, length, n = 64, 16, 2, 300, 20
    pages = -(-length // tokens)
    ascending = torch.linspace(-127, 126, length).round()
    ascending[[255, 270, 279]] = 127.0    # seen by all rows
    k = torch.zeros((pages * tokens, dim))
    k[:length, ::2] = ascending[:, None]
    k = k.to(torch.int8).view(pages, 1, tokens, dim)
    v = torch.randint(1, 128, (pages, 1, tokens, dim), generator=g, dtype=torch.int32).to(torch.int8)
    scales = torch.full((pages, 1), 2.0 ** size / 127), torch.full((pages, 1), 0.01)
    q = torch.full((n, 2, dim), 8 * 2.0 ** -5).to(dtype)    # 32 terms, and the call's scale of 1 / 8
    want, least, top = _exact(q, (k, v), scales, list(range(pages)), length, group)
    cache = ops.CacheI8(k.cuda(), v.cuda(), *(s.cuda() for s in scales))
    got = ops.attention_i8_cache(q.cuda(), cache, _i32([list(range(pages))]), _i32([length]), engine=engine).cpu().double()
    if size < 14 or engine == "rows":
        # All exponents have the same factors, so beyond a few thousand what is left are weights that are the same, to the last bit.
        bound = _bound(dtype, top if size < 14 else 1.0, least) + 2.0 ** -22
        assert (_distance(got, want) <= bound).all(), (_distance(got, want).max().item(), bound.min().item())
        return
    # In tiles an exponent is rounded once more where some row does not see all of a block (token 255 lies in another block than the two
    # others): by half a step, 2^-24 of 2^size * 1.44, which is 0.36 of a power of two at 2^22 already.  So the three may
    # have any weights; but they are the only ones (the next score is 2^20 / 127 below), and their sum is 1.
    values = v.double().view(pages * tokens, dim)[[255, 270, 279]] * 0.01
    slack = (2 * 2.0 ** -11 + HALF_STEP[dtype]) * values.amax(0)    # each weight as an f16, then the output
    assert ((got >= values.amin(0) - slack) & (got <= values.amax(0) + slack)).all()
