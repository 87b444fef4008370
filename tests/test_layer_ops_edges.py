"""The operators around the matmul at their edges: what a row may not depend on, counts next to what 32 bits hold, tiles that
rows fill in part, roundings as small as the kernels say they are, buffers that lie in one another."""
import math

import numpy as np
import pytest

import test_layer_ops as T
from test_layer_ops import Cache, check_attention, eng, gpu, md, mem, run_append, run_attention, tmd  # noqa: F401
from onednn_b200 import api, dtypes as dt  # noqa: F401

MMA, TC, GENERIC = "cuda:sm100:kv_attention_mma", "cuda:sm100:kv_attention_tc", "cuda:generic"


# ---- tiles that rows fill in part ------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("news", [1, 31, 33, 63, 65, 127, 129, 161, 255, 257])
@pytest.mark.parametrize("length,dst", [(300, "bf16"), (9000, "f16")])
def test_prompts_whose_rows_fill_a_warp_in_part(gpu, news, length, dst):
    """Whole items (300 tokens) and cut ones (9000, on their own) with 1 .. 31 live lanes in their last warp; rows behind stay."""
    torch, types = T._torch()
    c = Cache([length, 100], [news, 96], 1, 16, 128, "s8", seed=news, behind=3)
    q = torch.randn(c.rows, 1, 128, generator=c.g, device="cuda").to(types[dst])
    out = torch.full_like(q, 3.0)
    kept = out.clone()
    p, _ = run_attention(gpu, c, q, out, 128 ** -0.5, TC)
    assert p.pd.impl_info_str() == TC
    gpu[1].wait()
    check_attention(c, q, 128 ** -0.5, out, kept, dst)


# ---- counts next to what 32 bits hold --------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("impl,news", [(MMA, 1), (MMA, 3), (TC, 48)])
@pytest.mark.parametrize("length", [0x7fffff00, 0x7fffffff])
def test_a_sequence_of_two_thousand_million_tokens(gpu, impl, news, length):
    """One page of 2^20 tokens, 2048 times in the table: positions up to 2^31 - 257 are read, none behind; with more tokens
    than that the rest is left out and reported.  Every page says the same, so the result is the page's own.

    Sums run over 2^31 weights in f32: no chain of additions is longer than 2^18 (2^24 units of 128 tokens over at least 128
    blocks), each off by 2^-22 at most where the matrix unit truncates: 2^-4 of the size, rounded up."""
    torch, _ = T._torch()
    e, s = gpu
    page, dim = 1 << 20, 16
    c = Cache([page], [news], 1, page, dim, "s8", spare=0)
    q = torch.randn(news, 1, dim, generator=c.g, device="cuda").to(torch.bfloat16)
    k, v = c.dense(0, 0, page)[:, 0], c.dense(1, 0, page)[:, 0]
    v_abs = v.abs()
    z = torch.exp(q[:, 0].double() @ k.T * 0.1)
    want, size = z @ v / z.sum(1, keepdim=True), z @ v_abs / z.sum(1, keepdim=True)
    c.table = torch.zeros(1, 2048, dtype=torch.int32, device="cuda")
    c.kv_lens.fill_(length)
    dst = torch.full_like(q, math.nan)
    p, _ = run_attention(gpu, c, q, dst, 0.1, impl)
    assert p.pd.impl_info_str() == impl
    if length > 0x7fffff00:
        T.bad_wait(s)
    else:
        s.wait()
    assert ((dst[:, 0].double() - want).abs() <= size * 2.0 ** -4).all()


# ---- what a row may not depend on, and how closely it is kept --------------------------------------------------

def by_row(c, q, scale, weights=None):
    """(result, sum of p |v|, largest p * value scale * peak, tokens) of every row in 64 bits, the middle two relative to the sum
    of p, over the tokens that the row sees and no others; and the largest sum of |q| |k| that a score has.
    `weights`: what p * value scale (relative to the largest of the row) is rounded to before the product."""
    torch, _ = T._torch()
    group = q.shape[1] // c.heads
    want, size, most = (torch.zeros(q.shape[:2] + (n,), dtype=torch.float64, device="cuda") for n in (c.dim, c.dim, 1))
    tokens, reach = torch.zeros(q.shape[0], 1, 1, dtype=torch.float64, device="cuda"), 0.0
    for b, (n, length) in enumerate(zip(c.news, c.lens)):
        lo = int(c.np_off[b])
        idx = torch.from_numpy(c.np_table[b, :-(-length // c.page)].astype(np.int64)).cuda()
        unit = c.scales[1][idx].double().T.repeat_interleave(c.page, 1)[:, :length].repeat_interleave(group, 0)[:, None]  # (heads, 1, tokens)
        k, v = (c.dense(w, b, length).repeat_interleave(group, 1).transpose(0, 1) for w in (0, 1))
        x = q[lo:lo + n].double().transpose(0, 1)
        at = length - n + torch.arange(n, device="cuda")
        hidden = (torch.arange(length, device="cuda")[None] > at[:, None])[None]
        z = (x @ k.transpose(1, 2) * scale).masked_fill(hidden, -math.inf)
        reach = max(reach, float((x.abs() @ k.abs().transpose(1, 2) * abs(scale)).masked_fill(hidden, 0).max()))
        p = torch.exp(z - z.amax(-1, keepdim=True))
        total = p.sum(-1, keepdim=True)
        pv = p * unit
        top = pv.amax(-1, keepdim=True)
        if weights is not None:
            pv = weights(pv / top) * top
        code = v / unit.transpose(1, 2)
        want[lo:lo + n] = (pv @ code / total).transpose(0, 1)
        size[lo:lo + n] = (p @ v.abs() / total).transpose(0, 1)
        most[lo:lo + n] = (top / total * T.PEAK[c.kind]).transpose(0, 1)
        tokens[lo:lo + n] = at[:, None, None].double() + 1
    return want, size, most, tokens, reach


def closeness(c, q, scale, kind):
    """Off by at most (all of it over the tokens that the row sees): the weights' rounding, 2^-11 of each where the result is
    bf16, 2^-11 of what that left where it is f16 (2^-22), and half f16's smallest step, 2^-25, where the row's largest weight
    is kept at 2^-1 or above: 2^-24 of that per token; logarithm and exponential of the value scales 2^-21 together; a score's
    error, as in check_attention, twice; sums of `tokens` / 16 instructions' results, 2^-22 each; half a step of the result."""
    want, size, most, tokens, reach = by_row(c, q, scale)
    score = (c.dim + 8) * 2.0 ** -22 * reach + 64 * T.U
    weight = 2.0 ** -11 if kind == "bf16" else 2.0 ** -22
    tol = size * (weight + 2.0 ** -21 + 2 * score + (tokens / 16 + 4) * 2.0 ** -22) + most * tokens * 2.0 ** -24
    return want, tol + want.abs() * T.HALF[kind] + (2.0 ** -25 if kind == "f16" else 2.0 ** -134)


# (lens, news, page): the newest tokens lie in several pages, so that rows of one tile see different ones
SPREAD = {"step": ([700, 33, 256], [1, 1, 1], 16), "draft": ([64, 131, 40], [9, 7, 11], 8), "uneven": ([90, 45], [8, 20], 5),
          "prompt": ([400, 300], [200, 300], 32), "runs of 8": ([300, 129], [150, 129], 24)}


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
@pytest.mark.parametrize("kind", ["s8", "e4m3"])
@pytest.mark.parametrize("shape", list(SPREAD))
@pytest.mark.parametrize("what", ["last page large", "every other page large", "large pages without weight", "first page small",
                                  "first pages of zeros", "zeros everywhere else", "rising", "all small", "all large"])
def test_value_scales_of_pages_that_do_not_count(gpu, impl, kind, shape, what):
    """Pages whose values are 2^20 .. 2^60 times the others', which rows do not see, or give no weight, or do: every row is
    held to what it sees itself."""
    torch, _ = T._torch()
    lens, news, page = SPREAD[shape]
    for dim, power in ((128, 24), (64, 40), (80, 60)):
        c = Cache(lens, news, 2, page, dim, kind, seed=power)
        q = torch.randn(c.rows, 8, dim, generator=c.g, device="cuda")
        big = 2.0 ** power
        for b, n in enumerate(lens):
            ids = torch.from_numpy(c.np_table[b, :-(-n // page)].astype(np.int64)).cuda()
            v = c.scales[1]
            if what == "last page large":
                v[ids[-1]] *= big
            elif what == "every other page large":
                v[ids[::2]] *= big
            elif what == "large pages without weight":
                # scores of some -100 there, of some 0 elsewhere: weights of 2^-144, values of 2^power
                q = q.abs()
                c.codes[0].view(torch.int8)[ids[1::3]] = -64 if kind == "s8" else -0x80 + 0x68  # -64, both
                c.scales[0][ids[1::3]] = 100 / (64 * 0.1 * 0.79 * dim)
                v[ids[1::3]] *= big
            elif what == "first page small":
                v[ids[0]] /= big
            elif what == "first pages of zeros":
                for w in (0, 1):
                    c.codes[w][ids[:2]] = 0
                    c.scales[w][ids[:2]] = T.TINY
            elif what == "zeros everywhere else":
                c.codes[1][ids[::2]] = 0
                v[ids[::2]] = T.TINY
            elif what == "rising":
                v[ids] *= torch.exp2(torch.linspace(-power, 10, len(ids), device="cuda")).floor()[:, None].clamp_min(2.0 ** -power)
            elif what == "all small":
                v[ids] /= big
            else:
                v[ids] *= big
        q = q.to(torch.bfloat16)
        dst = torch.full_like(q, math.nan)
        run_attention(gpu, c, q, dst, 0.1, impl)
        gpu[1].wait()
        want, tol = closeness(c, q, 0.1, "bf16")
        err = (dst.double() - want).abs()
        assert not torch.isnan(dst).any()
        assert (err <= tol).all(), "%s: %g of the tolerance" % (power, float((err / tol).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("impl,seqs,news", [(MMA, 64, 1), (MMA, 64, 3), (TC, 40, 48)])
@pytest.mark.parametrize("rise", [0.7, 0.95, 8.9])
def test_scores_that_rise_step_by_step_behind_a_large_page(gpu, impl, seqs, news, rise):
    """A first page of large values and low scores, then pages whose scores rise by 2^rise each: in the end the first page has no
    weight.  Whatever stood for it in a row's exponent is to be gone by then."""
    torch, _ = T._torch()
    page, pages, heads, dim = 128, 56, 8, 64
    c = Cache([page * pages] * seqs, [news] * seqs, heads, page, dim, "s8", seed=8)
    c.codes[0].zero_()
    c.codes[0][..., 0] = 64
    for b in range(seqs):
        ids = torch.from_numpy(c.np_table[b].astype(np.int64)).cuda()
        c.scales[0][ids] = (torch.arange(pages, device="cuda")[:, None] + 1) * (rise * math.log(2) / 64 / 0.125)
        c.scales[1][ids[0]] *= 2.0 ** min(60, rise * 44)
    q = torch.zeros(c.rows, heads, dim, device="cuda")
    q[..., 0] = 1
    q = q.to(torch.bfloat16)
    dst = torch.full_like(q, math.nan)
    run_attention(gpu, c, q, dst, 0.125, impl)
    gpu[1].wait()
    want, tol = closeness(c, q, 0.125, "bf16")
    err = (dst.double() - want).abs()
    assert not torch.isnan(dst).any()
    assert (err <= tol).all(), "%g of the tolerance, %d of %d" % (float((err / tol).max()), int((err > tol).sum()), err.numel())


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
@pytest.mark.parametrize("scale", [1e3, -1e3, 1e6, -1e7, 2e7, 1e9, 1e15, 1e30])
@pytest.mark.parametrize("large", [1.0, 2.0 ** 30])
def test_scores_of_any_size(gpu, impl, scale, large):
    """Every token a key of its own: the row's result is the value of the best one that it sees, however large scores are.  One
    weight, rounded to f16, then the result's rounding.  The prompts' kernel takes scores, times log2 e, to
    2^26 (here scale * 127 / 8 * log2 e); a row beyond is NaN, none is wrong."""
    torch, _ = T._torch()
    lens, news = [250, 130], [100, 60]
    c = Cache(lens, news, 1, 32, 64, "s8", seed=9)
    q = torch.zeros(c.rows, 1, 64, device="cuda")
    q[..., 0] = 1
    q = q.to(torch.bfloat16)
    c.codes[0].zero_()
    c.scales[0].fill_(0.125)
    c.scales[1][1::2] *= large
    want = torch.zeros(c.rows, 64, dtype=torch.float64, device="cuda")
    for b, n in enumerate(lens):
        key = torch.randperm(255, generator=c.g, device="cuda")[:n] - 127
        ids = torch.from_numpy(c.np_table[b, :-(-n // 32)].astype(np.int64)).cuda()
        page = torch.zeros(len(ids) * 32, dtype=torch.int8, device="cuda")
        page[:n] = key.to(torch.int8)
        c.codes[0][ids, 0, :, 0] = page.view(-1, 32)
        value = c.dense(1, b, n)[:, 0]
        for i in range(news[b]):
            seen = n - news[b] + i + 1
            want[int(c.np_off[b]) + i] = value[int((key[:seen] * (1 if scale > 0 else -1)).argmax())]
    dst = torch.full_like(q, math.nan)
    run_attention(gpu, c, q, dst, scale, impl)
    gpu[1].wait()
    right = (dst[:, 0].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -20)
    if impl == TC and abs(scale) * 127 / 8 * 1.4427 > 2.0 ** 26:
        right |= torch.isnan(dst[:, 0])
    assert right.all()


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
@pytest.mark.parametrize("kind", ["s8", "e4m3"])
@pytest.mark.parametrize("page", [16, 24])
def test_f16_results_come_from_unrounded_weights(gpu, impl, kind, page):
    """What is left of a weight after its rounding to f16 counts where the result is f16.  The allowance is small enough to tell:
    the definition with weights rounded to f16 does not meet it."""
    torch, _ = T._torch()
    c = Cache([70, 96], [60, 90], 1, page, 128, kind, seed=page)
    q = torch.randn(c.rows, 2, 128, generator=c.g, device="cuda").to(torch.float16)
    scale = 0.002  # scores around 0.01, so that their own errors stay below 2^-18
    dst = torch.full_like(q, math.nan)
    run_attention(gpu, c, q, dst, scale, impl)
    gpu[1].wait()
    want, tol = closeness(c, q, scale, "f16")
    assert ((dst.double() - want).abs() <= tol).all(), "%g of the tolerance" % float(((dst.double() - want).abs() / tol).max())
    rounded = by_row(c, q, scale, weights=lambda w: (w * 8192).half().double() / 8192)[0].to(torch.float16)
    assert ((rounded.double() - want).abs() > tol).any()


@pytest.mark.gpu
def test_a_token_of_two_to_the_thirty_elements(gpu):
    """2^30 - 1 in all heads together, next to the largest that the descriptors take, element by element."""
    torch, _ = T._torch()
    heads, dim = 32767, 32769
    e, s = gpu
    n = heads * dim
    buf = [torch.randint(-127, 128, (n + 1,), dtype=torch.int8, device="cuda") for _ in range(2)]
    c = Cache([1], [1], 1, 1, 16, "s8", spare=0)
    c.codes = [b[1:].view(1, heads, 1, dim) for b in buf]
    c.scales = [torch.rand(1, heads, device="cuda") + 0.5 for _ in range(2)]
    out = [torch.full((1 + n,), 9, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    k, v = (o[1:].view(1, heads, dim) for o in out)
    p = api.Primitive(api.kv_cache_read_primitive_desc(e, tmd(c.codes[0]), tmd(k), tmd(c.table)))
    p.execute(s, {**c.args(e), api.ARG_DST: mem(k, e), api.ARG_DST_1: mem(v, e)})
    s.wait()
    assert all(float(o[0]) == 9 for o in out)
    for i, got in enumerate((k, v)):
        for h in range(0, heads, 256):
            want = (c.codes[i][0, h:h + 256, 0].float() * c.scales[i][0, h:h + 256, None]).to(torch.bfloat16)
            assert torch.equal(got[0, h:h + 256], want)
    # and appended: the same codes again, from values that they stand for
    x = [(c.codes[i][:, :, 0].to(torch.bfloat16)) for i in range(2)]
    for i in range(2):
        x[i][:, :, 0] = 127  # every head's scale is 127 / 127
    c.codes = [torch.zeros_like(t) for t in c.codes]
    run_append(gpu, c, x[0], x[1])
    s.wait()
    one = (torch.full((), 127.0) * torch.tensor(1 / 127.0)).item()  # in f32
    for i in range(2):
        assert (c.scales[i] == one).all()
        assert torch.equal(c.codes[i][:, :, 0], x[i].to(torch.int8))


# ---- buffers that lie in one another ---------------------------------------------------------------------------

@pytest.mark.gpu
def test_outputs_that_share_places_are_refused(gpu):
    """Keys' and values' caches, scales or rows that share elements without being the same memory; ones that lie in each
    other's gaps are taken."""
    torch, _ = T._torch()
    e, s = gpu
    heads, page, dim = 2, 16, 32
    c = Cache([20, 3], [2, 3], heads, page, dim, "s8")
    x = torch.randn(c.rows, heads, dim, generator=c.g, device="cuda")
    both = torch.zeros(2 * c.pages, heads, page, 2, dim, dtype=torch.int8, device="cuda")
    scales = torch.zeros(2 * c.pages, heads, device="cuda")
    rows = torch.zeros(64, heads, 2, dim, device="cuda")

    def cache_at(first):
        return api.Memory(tmd(both[:c.pages, :, :, 0]), e, both.data_ptr() + first)

    def append(key_at, value_at, key_scale=0, value_scale=c.pages * heads):
        f32 = tmd(scales[:c.pages])
        p = api.Primitive(api.kv_cache_append_primitive_desc(e, tmd(x), tmd(both[:c.pages, :, :, 0]), tmd(c.table)))
        p.execute(s, {**c.args(e), api.ARG_SRC: mem(x, e), api.ARG_SRC_1: mem(x, e), api.ARG_B200_KEY_CACHE: cache_at(key_at),
                      api.ARG_B200_VALUE_CACHE: cache_at(value_at), api.ARG_B200_KEY_SCALES: api.Memory(f32, e, scales.data_ptr() + 4 * key_scale),
                      api.ARG_B200_VALUE_SCALES: api.Memory(f32, e, scales.data_ptr() + 4 * value_scale)})

    def refused(f, *a):
        with pytest.raises(api.Error) as err:
            f(*a)
        assert err.value.name == "invalid_arguments"
    slot, head = 2 * dim, 2 * dim * page
    one = head * heads  # bytes of a page
    for a, b in ((0, 0), (0, 1), (0, dim - 1), (0, slot), (5 * slot, 0), (0, head), (0, one), (0, (c.pages - 1) * one + head), (one, 1), (0, slot + dim - 1),
                 (0, head - slot + dim + 1)):
        refused(append, a, b)
    for a, b in ((0, 1), (heads, 0), (0, c.pages * heads - 1)):
        refused(append, 0, dim, a, b)
    s.wait()
    assert not both.any() and not scales.any()
    # values in the gaps between keys, and on the other side of them; behind one another
    want = [T.expected_append(c, x, torch.zeros(c.pages, heads, page, dim, dtype=torch.int8, device="cuda"), scales[:c.pages])[0] for _ in range(2)]
    for a, b in ((0, dim), (dim, 0), (0, c.pages * one), (0, c.pages * one + dim)):
        both.zero_()
        scales.zero_()
        append(a, b)
        s.wait()
        flat = both.view(-1)
        for at, w in ((a, want[0]), (b, want[1])):
            got = flat.as_strided((c.pages, heads, page, dim), (one, head, slot, 1), at)
            assert torch.equal(got, w)
    p = api.Primitive(api.kv_cache_read_primitive_desc(e, tmd(c.codes[0]), tmd(rows[:5, :, 0]), tmd(c.table)))

    def read(first, second):
        d = tmd(rows[:5, :, 0])
        p.execute(s, {**c.args(e), api.ARG_DST: api.Memory(d, e, rows.data_ptr() + 4 * first), api.ARG_DST_1: api.Memory(d, e, rows.data_ptr() + 4 * second)})
    for a, b in ((0, 0), (0, 1), (2 * dim, 0), (0, 4 * heads * 2 * dim)):
        refused(read, a, b)
    for a, b in ((0, dim), (0, 5 * heads * 2 * dim)):
        read(a, b)
    s.wait()
    r = torch.randn(4, 64, device="cuda")
    h = torch.zeros_like(r)
    norm = api.Primitive(api.rms_norm_primitive_desc(e, tmd(r), tmd(r), 1e-5, residual_md=tmd(r)))
    refused(norm.execute, s, {api.ARG_SRC: mem(r, e), api.ARG_SRC_1: mem(r, e), api.ARG_DST: mem(h, e), api.ARG_DST_1: mem(h, e)})
    s.wait()


# ---- batches and layouts ---------------------------------------------------------------------------------------

STEP = dict(lens=[700, 33, 256], news=[1, 1, 1], heads=2, page=16, dim=128, kind="s8")
PROMPT = dict(lens=[700, 300], news=[200, 300], heads=2, page=32, dim=128, kind="s8")


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
def test_lengths_beyond_the_table_leave_exactly_the_tokens_that_it_holds(gpu, impl):
    """Every row stands behind the table's end and sees all slots of the pages that the table names inside the cache; the
    rest is left out and reported."""
    torch, _ = T._torch()
    e, s = gpu
    spec = PROMPT if impl == TC else STEP
    c = Cache(**spec, seed=11)
    q = torch.randn(c.rows, 8, c.dim, generator=c.g, device="cuda").to(torch.bfloat16)
    c.kv_lens += 100000
    dst = torch.full_like(q, math.nan)
    run_attention(gpu, c, q, dst, 0.1, impl)
    T.bad_wait(s)
    for b, n in enumerate(c.news):
        rows = slice(int(c.np_off[b]), int(c.np_off[b]) + n)
        pages = [int(v) for v in c.np_table[b] if 0 <= v < c.pages]
        one = Cache([len(pages) * c.page], [n], c.heads, c.page, c.dim, c.kind)
        one.codes, one.scales, one.np_table, one.pages = c.codes, c.scales, np.asarray([pages], dtype=np.int32), c.pages
        k, v = (one.dense(w, 0, one.lens[0]).repeat_interleave(4, 1).transpose(0, 1) for w in (0, 1))
        z = q[rows].double().transpose(0, 1) @ k.transpose(1, 2) * 0.1
        reach = float((q[rows].double().abs().transpose(0, 1) @ k.abs().transpose(1, 2) * 0.1).max())
        p = torch.softmax(z, -1)
        want, size = (p @ v).transpose(0, 1), (p @ v.abs()).transpose(0, 1)
        # as in closeness(): weights, scores, sums, result, and 2^-24 of the largest value for each of up to 2^10 tokens
        tol = size * (2.0 ** -11 + 2 * ((c.dim + 8) * 2.0 ** -22 * reach + 64 * T.U) + 64 * 2.0 ** -22) + want.abs() * 2.0 ** -8 + float(v.abs().max()) * 2.0 ** -14
        assert ((dst[rows].double() - want).abs() <= tol).all()  # NaN, what was there before, does not pass


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
@pytest.mark.parametrize("news", [[0, 0, 0], [1, 0, 1], [0, 40, 0]])
def test_descriptors_larger_than_the_batch(gpu, impl, news):
    """A primitive for 4096 rows takes batches of none, of a step, of a prompt piece; the rows behind stay."""
    torch, types = T._torch()
    c = Cache([90, 300, 17], news, 2, 16, 64, "e4m3", before=2, behind=4094 - sum(news), seed=3)
    q = torch.randn(c.rows, 4, 64, generator=c.g, device="cuda").to(torch.bfloat16)
    dst = torch.full_like(q, 3.0)
    kept = dst.clone()
    run_attention(gpu, c, q, dst, 0.1, impl)
    gpu[1].wait()
    check_attention(c, q, 0.1, dst, kept, "bf16")
    x = torch.randn(c.rows, 2, 64, generator=c.g, device="cuda").to(torch.bfloat16)
    want = [T.expected_append(c, x, c.codes[i], c.scales[i]) for i in range(2)]
    run_append(gpu, c, x, x)
    gpu[1].wait()
    for i in range(2):
        assert torch.equal(c.scales[i], want[i][1]) and torch.equal(c.codes[i].contiguous().view(torch.int8), want[i][0])


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
@pytest.mark.parametrize("lens,news,page,dim", [([130, 61], [100, 61], 16, 64), ([40, 97], [1, 2], 1, 64), ([75, 20], [3, 20], 24, 128)])
def test_token_major_pages_and_head_major_rows(gpu, impl, lens, news, page, dim):
    """Other orders of the same dims: pages (token, head, dim) in memory, queries and results (head, row, dim), a table with rows
    wider than its columns."""
    torch, types = T._torch()
    e, s = gpu
    c = Cache(lens, news, 2, page, dim, "s8", seed=page)
    c.codes = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in c.codes]
    wide = torch.full((len(lens), c.table.shape[1] + 3), -1, dtype=torch.int32, device="cuda")
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide[:, :c.table.shape[1]]
    x = torch.randn(2, c.rows, dim, generator=c.g, device="cuda").to(torch.float16).transpose(0, 1)  # (rows, heads, dim), head-major
    want = [T.expected_append(c, x, c.codes[i], c.scales[i]) for i in range(2)]
    run_append(gpu, c, x, x)
    s.wait()
    for i in range(2):
        assert torch.equal(c.scales[i], want[i][1]) and torch.equal(c.codes[i].contiguous(), want[i][0])
    q = torch.randn(8, c.rows, dim, generator=c.g, device="cuda").to(torch.bfloat16).transpose(0, 1)
    dst = torch.full((8, c.rows, dim), 3.0, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    run_attention(gpu, c, q, dst, 0.1, impl)
    s.wait()
    check_attention(c, q, 0.1, dst, dst, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
def test_sequences_that_share_pages(gpu, impl):
    """A common prefix, and the same sequence twice."""
    torch, _ = T._torch()
    c = Cache([200, 200, 200], [70, 70, 70], 2, 32, 64, "s8", seed=4)
    t = c.np_table.copy()
    t[1, :4] = t[0, :4]
    t[2] = t[0]
    c.np_table, c.table = t, torch.from_numpy(t).cuda()
    q = torch.randn(c.rows, 4, 64, generator=c.g, device="cuda").to(torch.bfloat16)
    dst = torch.full_like(q, math.nan)
    run_attention(gpu, c, q, dst, 0.1, impl)
    gpu[1].wait()
    check_attention(c, q, 0.1, dst, dst, "bf16")


@pytest.mark.gpu
def test_many_sequences(gpu):
    """Five thousand of them, most of one token, some without: append, read and attention find each row's."""
    torch, types = T._torch()
    e, s = gpu
    n = 5000
    lens = [1 + i * 7 % 23 for i in range(n)]
    news = [0 if i % 11 == 0 else 1 for i in range(n)]
    c = Cache(lens, news, 1, 8, 16, "s8", seed=6, behind=5)
    x = torch.randn(c.rows, 1, 16, generator=c.g, device="cuda")
    want = [T.expected_append(c, x, c.codes[i], c.scales[i]) for i in range(2)]
    run_append(gpu, c, x, x)
    s.wait()
    for i in range(2):
        assert torch.equal(c.scales[i], want[i][1]) and torch.equal(c.codes[i], want[i][0])
    q = torch.randn(c.rows, 2, 16, generator=c.g, device="cuda").to(torch.bfloat16)
    outs = []
    for impl in (MMA, GENERIC):
        dst = torch.full_like(q, 3.0)
        run_attention(gpu, c, q, dst, 0.25, impl)
        s.wait()
        outs.append(dst)
    kept = torch.full_like(q, 3.0)
    check_attention(c, q, 0.25, outs[0], kept, "bf16")
    check_attention(c, q, 0.25, outs[1], kept, "bf16")


# ---- the norm's plans for many rows ----------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,src,residual,gamma,dst", [
    (300, 264, "bf16", "bf16", "f32", "s8"), (300, 512, "f16", "", "bf16", "f16"), (257, 1024, "bf16", "f32", "f32", "e4m3"),
    (300, 1032, "f32", "bf16", "", "s8"), (300, 4096, "bf16", "bf16", "f32", "e4m3"), (270, 8192, "f16", "f32", "f16", "s8"),
    (300, 5003, "bf16", "bf16", "f32", "s8"), (1031, 64, "f32", "", "f32", "s8"), (1025, 136, "bf16", "f16", "f32", "bf16")])
def test_norm_of_many_rows(gpu, rows, cols, src, residual, gamma, dst):
    torch, types = T._torch()
    torch.manual_seed(rows + cols)
    x = (torch.randn(rows, cols, device="cuda") * 3).to(types[src])
    r = (torch.randn(rows, cols, device="cuda") * 5).to(types[residual]) if residual else None
    g = (torch.rand(cols, device="cuda") + 0.5).to(types[gamma]) if gamma else None
    out = torch.zeros(rows, cols, dtype=types[dst], device="cuda")
    total, scales = T.run_norm(gpu, x, r, g, out, 1e-5)
    T.check_norm(x, r, g, out, 1e-5, total, scales, dst)


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
@pytest.mark.parametrize("group,news", [(130, [1, 1]), (71, [1, 3]), (33, [2, 0])])
def test_many_query_heads_on_one_key_head(gpu, impl, group, news):
    torch, _ = T._torch()
    c = Cache([300, 41], news, 1, 16, 64, "s8", seed=group)
    q = torch.randn(c.rows, group, 64, generator=c.g, device="cuda").to(torch.bfloat16)
    dst = torch.full_like(q, math.nan)
    run_attention(gpu, c, q, dst, 0.125, impl)
    gpu[1].wait()
    check_attention(c, q, 0.125, dst, dst, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 20])
def test_read_with_more_rows_than_tokens(gpu, dim):
    """Rows that stand for tokens before a sequence's first are zero, the others its tokens."""
    torch, _ = T._torch()
    e, s = gpu
    c = Cache([3, 0, 9], [5, 2, 9], 2, 8, dim, "s8", behind=2)
    out = torch.full((2, c.rows, 2, dim), 7.0, device="cuda")
    p = api.Primitive(api.kv_cache_read_primitive_desc(e, tmd(c.codes[0]), tmd(out[0]), tmd(c.table)))
    p.execute(s, {**c.args(e), api.ARG_DST: mem(out[0], e), api.ARG_DST_1: mem(out[1], e)})
    s.wait()
    for i in range(2):
        assert (out[i, :2] == 0).all() and (out[i, 5:7] == 0).all() and (out[i, 16:] == 7).all()
        for rows, b, n in ((slice(2, 5), 0, 3), (slice(7, 16), 2, 9)):
            assert torch.equal(out[i, rows], c.dense(i, b, n).float())


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(7, 128), (300, 512), (5, 4096), (3, 257), (2, 20000)])
def test_norm_in_the_memory_of_its_inputs(gpu, rows, cols):
    """The sum written over src, and the result over src: each element is read before anything is written in its place."""
    torch, _ = T._torch()
    e, s = gpu
    torch.manual_seed(cols)
    x = torch.randn(rows, cols, device="cuda").to(torch.bfloat16)
    r = torch.randn(rows, cols, device="cuda").to(torch.bfloat16)
    for over in ("sum", "result"):
        src, codes, scales = x.clone(), torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
        if over == "sum":
            p = api.Primitive(api.rms_norm_primitive_desc(e, tmd(x), tmd(codes), 1e-5, residual_md=tmd(r)))
            p.execute(s, {api.ARG_SRC: mem(src, e), api.ARG_SRC_1: mem(r, e), api.ARG_DST_1: mem(src, e), api.ARG_DST: mem(codes, e),
                          api.ARG_ATTR_SCALES | api.ARG_DST: mem(scales, e)})
            s.wait()
            T.check_norm(x, r, None, codes, 1e-5, src, scales, "s8")
        else:
            p = api.Primitive(api.rms_norm_primitive_desc(e, tmd(x), tmd(x), 1e-5))
            p.execute(s, {api.ARG_SRC: mem(src, e), api.ARG_DST: mem(src, e)})
            s.wait()
            T.check_norm(x, None, None, src, 1e-5, None, None, "bf16")
