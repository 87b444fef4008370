"""The operators around the matmul as programs use them: dispatch, scratchpads, captured graphs, streams, pages and values
that have no business in a result, memory beyond 4 GiB, and a whole layer's run of them with the matmuls between."""
import math

import numpy as np
import pytest

import test_layer_ops as T
from test_layer_ops import Cache, check_attention, check_norm, eng, expected_append, gpu, md, mem, run_append, run_attention, tmd  # noqa: F401
from onednn_b200 import api, dtypes as dt

MMA, TC, GENERIC = "cuda:sm100:kv_attention_mma", "cuda:sm100:kv_attention_tc", "cuda:generic"


# ---- dispatch (no GPU needed) ----------------------------------------------------------------------------------

def _impls(eng, rows, seqs, heads=2, group=4, page=16, dim=64, q="bf16", dst=None, cache="s8", cache_strides=None, q_strides=None):
    x = md((rows, heads * group, dim), q, q_strides)
    pd = api.kv_cache_attention_primitive_desc(eng, x, md((9, heads, page, dim), cache, cache_strides),
                                               md((rows, heads * group, dim), dst or q), md((seqs, 4), "s32"), 0.1)
    names = [pd.impl_info_str()]
    while pd.next_impl():
        names.append(pd.impl_info_str())
    return names


def test_attention_dispatch(eng):
    """Prompts on tcgen05, steps on mma.sync, whatever neither takes on the generic kernel, which every list ends with."""
    assert _impls(eng, 8, 8) == [MMA, GENERIC]
    assert _impls(eng, 96, 8, group=4) == [TC, MMA, GENERIC]        # 12 tokens x 4 heads: 48 rows
    assert _impls(eng, 95, 8, group=4) == [MMA, GENERIC]
    assert _impls(eng, 100, 1, page=24) == [TC, MMA, GENERIC]
    assert _impls(eng, 100, 1, page=20) == [MMA, GENERIC]           # pages that 8 does not divide
    assert _impls(eng, 100, 1, dim=144) == [MMA, GENERIC]           # heads wider than 128
    assert _impls(eng, 100, 1, dim=256, cache="e4m3") == [MMA, GENERIC]
    assert _impls(eng, 100, 1, dim=72) == [GENERIC]                 # rows of codes that 16 bytes do not divide
    assert _impls(eng, 100, 1, q="f32") == [GENERIC]
    assert _impls(eng, 100, 1, q="bf16", dst="f32") == [GENERIC]
    assert _impls(eng, 100, 1, q="bf16", dst="f16") == [TC, MMA, GENERIC]
    assert _impls(eng, 8, 8, cache_strides=(2 * 16 * 72, 16 * 72, 72, 1)) == [GENERIC]
    assert _impls(eng, 8, 8, cache_strides=(2 * 16 * 80, 16 * 80, 80, 1)) == [MMA, GENERIC]
    assert _impls(eng, 8, 8, q_strides=(8 * 68, 68, 1)) == [GENERIC]


def test_primitives_are_told_apart_by_what_they_are(eng):
    """Descriptors that differ in the softmax scale or epsilon alone must not share a primitive cache entry."""
    import ctypes as C
    x, c, t = md((8, 4, 64), "bf16"), md((5, 2, 16, 64), "s8"), md((8, 4), "s32")
    L = api.lib()

    def cached(pd):
        r = C.c_int(-1)
        assert L.dnnl_b200_primitive_cache_contains(pd.h, None, C.byref(r)) == 0
        return r.value
    a = api.kv_cache_attention_primitive_desc(eng, x, c, x, t, 0.5)
    assert cached(a) == 0
    if api.Engine.get_count() > 0:
        keep = api.Primitive(a)  # noqa: F841
        assert cached(a) == 1
        assert cached(api.kv_cache_attention_primitive_desc(eng, x, c, x, t, 0.25)) == 0
        y = md((8, 64), "bf16")
        keep2 = api.Primitive(api.rms_norm_primitive_desc(eng, y, y, 1e-5))  # noqa: F841
        assert cached(api.rms_norm_primitive_desc(eng, y, y, 1e-5)) == 1
        assert cached(api.rms_norm_primitive_desc(eng, y, y, 1e-6)) == 0
        assert cached(api.rms_norm_primitive_desc(eng, y, y, 1e-5, residual_md=y)) == 0
    else:
        with pytest.raises(api.Error) as e:
            api.Primitive(a)
        assert e.value.name == "runtime_error"


# ---- on the GPU ------------------------------------------------------------------------------------------------

def side_stream(e):
    """A stream of torch's, and the framework's around it (made before any capture on it)."""
    torch, _ = T._torch()
    st = torch.cuda.Stream()
    return st, api.Stream(e, cuda_stream=st.cuda_stream)


STEP = dict(lens=[700, 33, 256], news=[1, 1, 1], heads=2, page=16, dim=128, kind="s8")
PROMPT = dict(lens=[700, 300], news=[200, 300], heads=2, page=32, dim=128, kind="s8")
SHORT = dict(lens=[40, 41], news=[1, 2], heads=2, page=5, dim=24, kind="e4m3")  # generic


def _case(spec, group=4, src="bf16", seed=5, **more):
    torch, types = T._torch()
    c = Cache(**{**spec, **more}, seed=seed)
    q = torch.randn(c.rows, c.heads * group, c.dim, generator=c.g, device="cuda").to(types[src])
    return c, q


@pytest.mark.gpu
def test_execution_refusals(gpu):
    torch, _ = T._torch()
    e, s = gpu
    c, q = _case(STEP)
    dst = torch.zeros_like(q)
    p, args = run_attention(gpu, c, q, dst, 0.1)
    s.wait()

    def refused(change):
        a = dict(args)
        change(a)
        with pytest.raises(api.Error) as err:
            p.execute(s, a)
        assert err.value.name == "invalid_arguments"
    for k in list(args):
        refused(lambda a: a.pop(k))
    refused(lambda a: a.update({api.ARG_B200_KV_LENS: mem(torch.zeros(2, dtype=torch.int32, device="cuda"), e)}))
    refused(lambda a: a.update({api.ARG_B200_KV_LENS: mem(torch.zeros(3, device="cuda"), e)}))
    refused(lambda a: a.update({api.ARG_B200_KEY_SCALES: mem(c.scales[0][:, :1], e)}))
    refused(lambda a: a.update({api.ARG_DST: mem(dst[:1], e)}))
    refused(lambda a: a.update({api.ARG_DST: api.Memory(tmd(dst), e, 0)}))
    u = api.PrimitiveAttr()
    u.set_scratchpad_mode(1)
    pu = api.Primitive(api.kv_cache_attention_primitive_desc(e, tmd(q), tmd(c.codes[0]), tmd(dst), tmd(c.table), 0.1, attr=u))
    with pytest.raises(api.Error) as err:
        pu.execute(s, args)
    assert err.value.name == "invalid_arguments"


@pytest.mark.gpu
@pytest.mark.parametrize("spec,impl", [(STEP, MMA), (PROMPT, TC), (PROMPT, MMA), (SHORT, GENERIC)])
def test_scratchpads_and_repetition(gpu, spec, impl):
    """The same bits each time, in the library's scratchpad and in a dirty one of the caller's, whose surroundings stay."""
    torch, _ = T._torch()
    e, s = gpu
    c, q = _case(spec)
    first = torch.zeros_like(q)
    p, args = run_attention(gpu, c, q, first, 0.1, impl)
    again = torch.zeros_like(q)
    for _ in range(3):
        p.execute(s, {**args, api.ARG_DST: mem(again, e)})
    s.wait()
    assert torch.equal(T.bits(first), T.bits(again))
    a = api.PrimitiveAttr()
    a.set_scratchpad_mode(1)
    pd = api.kv_cache_attention_primitive_desc(e, tmd(q), tmd(c.codes[0]), tmd(first), tmd(c.table), 0.1, attr=a)
    while pd.impl_info_str() != impl:
        assert pd.next_impl()
    n = pd.scratchpad_desc().get_size()
    assert (n > 0) == (impl != GENERIC)
    buf = torch.full((n + 1024,), 0xA5, dtype=torch.uint8, device="cuda")
    mine = {**args, api.ARG_DST: mem(again, e)}
    if n:
        mine[api.ARG_SCRATCHPAD] = api.Memory(pd.scratchpad_desc(), e, buf.data_ptr() + 512)
    pu = api.Primitive(pd)
    for _ in range(2):
        again.zero_()
        pu.execute(s, mine)
        s.wait()
        assert torch.equal(T.bits(first), T.bits(again))
        assert (buf[:512] == 0xA5).all() and (buf[512 + n:] == 0xA5).all()
    # after an error was reported the library's scratchpads are cleared and used again
    assert api.lib().dnnl_b200_debug_mark_scratchpads_dirty() == 0
    again.zero_()
    p.execute(s, {**args, api.ARG_DST: mem(again, e)})
    s.wait()
    assert torch.equal(T.bits(first), T.bits(again))


@pytest.mark.gpu
@pytest.mark.parametrize("spec,impl", [(STEP, MMA), (PROMPT, TC)])
def test_two_graphs_of_one_primitive_side_by_side(gpu, spec, impl):
    """Captured executions have scratch of their own: two graphs of one primitive on two streams, and an eager execution
    of the same primitive between, all at once, many times."""
    torch, _ = T._torch()
    e, s = gpu
    cases = [_case(spec, seed=i) for i in (1, 2, 3)]
    p, _ = run_attention(gpu, *cases[0], torch.zeros_like(cases[0][1]), 0.1, impl)
    s.wait()
    outs, wants, graphs, streams = [], [], [], []
    for c, q in cases:
        out = torch.zeros_like(q)
        args = {**c.args(e), api.ARG_SRC: mem(q, e), api.ARG_DST: mem(out, e)}
        p.execute(s, args)
        s.wait()
        outs.append((out, args))
        wants.append(out.clone())
    torch.cuda.synchronize()
    for out, args in outs[:2]:
        st, wrapped = side_stream(e)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            p.execute(wrapped, args)
        graphs.append(g)
        streams.append((st, wrapped))
    for _ in range(20):
        for out, _a in outs:
            out.zero_()
        torch.cuda.synchronize()
        for g, (st, _w) in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        p.execute(s, outs[2][1])
        torch.cuda.synchronize()
        for (out, _a), want in zip(outs, wants):
            assert torch.equal(T.bits(out), T.bits(want))
    # a graph reads offsets and lengths when it runs: one token less
    c, q = cases[0]
    c.kv_lens -= 1
    c.lens = [n - 1 for n in c.lens]
    with torch.cuda.stream(streams[0][0]):
        graphs[0].replay()
    torch.cuda.synchronize()
    check_attention(c, q, 0.1, outs[0][0], outs[0][0], "bf16")
    s.wait()
    del graphs


@pytest.mark.gpu
def test_append_read_and_norm_captured(gpu):
    torch, _ = T._torch()
    e, s = gpu
    c = Cache([50, 20], [3, 20], 2, 16, 64, "s8")
    x = torch.randn(23, 2, 64, generator=c.g, device="cuda").to(torch.bfloat16)
    want = [expected_append(c, x, c.codes[i], c.scales[i]) for i in range(2)]
    start = [t.clone() for t in c.codes + c.scales]
    out = torch.zeros(2, 23, 2, 64, dtype=torch.bfloat16, device="cuda")
    h, y, rs = torch.randn(23, 256, device="cuda"), torch.zeros(23, 256, dtype=torch.int8, device="cuda"), torch.zeros(23, device="cuda")
    append = api.Primitive(api.kv_cache_append_primitive_desc(e, tmd(x), tmd(c.codes[0]), tmd(c.table)))
    read = api.Primitive(api.kv_cache_read_primitive_desc(e, tmd(c.codes[0]), tmd(out[0]), tmd(c.table)))
    norm = api.Primitive(api.rms_norm_primitive_desc(e, tmd(h), tmd(y), 1e-5))
    st, w = side_stream(e)
    g = torch.cuda.CUDAGraph()
    a1 = api.ExecArgs({**c.args(e), api.ARG_SRC: mem(x, e), api.ARG_SRC_1: mem(x, e)})
    a2 = api.ExecArgs({**c.args(e), api.ARG_DST: mem(out[0], e), api.ARG_DST_1: mem(out[1], e)})
    a3 = api.ExecArgs({api.ARG_SRC: mem(h, e), api.ARG_DST: mem(y, e), api.ARG_ATTR_SCALES | api.ARG_DST: mem(rs, e)})
    with torch.cuda.graph(g, stream=st):
        append.execute(w, a1)
        read.execute(w, a2)
        norm.execute(w, a3)
    for _ in range(2):
        for t, v in zip(c.codes + c.scales, start):
            t.copy_(v)
        g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(c.codes[i].contiguous(), want[i][0]) and torch.equal(c.scales[i], want[i][1])
        check_norm(h, None, None, y, 1e-5, None, rs, "s8")
        assert (out != 0).any()


@pytest.mark.gpu
@pytest.mark.parametrize("spec,impl", [(STEP, MMA), (PROMPT, TC)])
def test_another_stream_than_the_current_one(gpu, spec, impl):
    torch, _ = T._torch()
    e, _ = gpu
    _, other = side_stream(e)
    c, q = _case(spec)
    dst = torch.zeros_like(q)
    torch.cuda.synchronize()
    run_attention(gpu, c, q, dst, 0.1, impl, stream=other)
    other.wait()
    check_attention(c, q, 0.1, dst, dst, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "e4m3"])
@pytest.mark.parametrize("spec,impl", [(STEP, MMA), (PROMPT, TC), (PROMPT, GENERIC)])
def test_what_lies_behind_the_last_token_does_not_show(gpu, spec, impl, kind):
    """Slots behind a sequence's last token hold NaN (e4m3) or the largest codes, unused pages NaN scales; queries of rows
    behind the last sequence are NaN."""
    torch, _ = T._torch()
    c, q = _case(spec, kind=kind, behind=3)
    raw = [t.view(torch.int8) for t in c.codes]
    used = torch.zeros(c.pages, dtype=torch.bool)
    for b, n in enumerate(c.lens):
        for j in range(-(-n // c.page)):
            used[int(c.np_table[b, j])] = True
        if n % c.page:
            for t in raw:
                t[int(c.np_table[b, n // c.page]), :, n % c.page:] = 127
    for t, sc in zip(raw, c.scales):
        t[~used.cuda()] = 127
        sc[~used.cuda()] = math.nan
    q[-3:] = math.nan
    dst = torch.full_like(q, 2.0)
    kept = dst.clone()
    run_attention(gpu, c, q, dst, 0.1, impl)
    gpu[1].wait()
    check_attention(c, q[:-3], 0.1, dst[:-3], kept[:-3], "bf16")
    assert torch.equal(dst[-3:], kept[-3:])


@pytest.mark.gpu
@pytest.mark.parametrize("spec,impl", [(STEP, MMA), (PROMPT, TC), (PROMPT, MMA), (STEP, GENERIC)])
def test_nan_and_infinite_queries_stay_in_their_rows(gpu, spec, impl):
    torch, _ = T._torch()
    c, q = _case(spec)
    clean = torch.zeros_like(q)
    run_attention(gpu, c, q, clean, 0.1, impl)
    bad = q.clone()
    bad[0, 1, 3] = math.nan
    bad[1, 2, 5] = math.inf
    dst = torch.zeros_like(q)
    run_attention(gpu, c, bad, dst, 0.1, impl)
    gpu[1].wait()
    assert torch.isnan(dst[0, 1]).all() and torch.isnan(dst[1, 2]).all()
    other = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    other[0, 1] = other[1, 2] = False
    assert torch.equal(T.bits(dst[other]), T.bits(clean[other]))


@pytest.mark.gpu
@pytest.mark.parametrize("spec,impl", [(STEP, MMA), (PROMPT, TC), (PROMPT, MMA), (STEP, GENERIC)])
@pytest.mark.parametrize("what", ["sharp", "negative", "flat", "pages of zeros", "scales far apart", "small queries"])
def test_scores_and_scales_far_from_the_ordinary(gpu, spec, impl, what):
    torch, _ = T._torch()
    c, q = _case(spec)
    scale = 0.1
    if what == "sharp":       # scores of some hundred: one token has all the weight
        scale = 4.0
    elif what == "negative":
        scale = -0.3
    elif what == "flat":
        scale = 0.0
    elif what == "pages of zeros":
        for t, sc in zip(c.codes, c.scales):
            t[::2] = 0
            sc[::2] = T.TINY
    elif what == "scales far apart":
        for sc in c.scales:
            sc *= torch.exp2(torch.randint(-12, 5, sc.shape, generator=c.g, device="cuda").float())
    else:
        q = (q.float() * 1e-30).to(q.dtype)
    dst = torch.zeros_like(q)
    run_attention(gpu, c, q, dst, scale, impl)
    gpu[1].wait()
    check_attention(c, q, scale, dst, dst, "bf16")


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [MMA, TC, GENERIC])
def test_attention_leaves_bad_pages_out_and_reports_them(gpu, impl):
    """Tokens of pages outside the cache, and beyond the table, count as not there; the stream's next wait fails."""
    torch, _ = T._torch()
    e, s = gpu
    spec = PROMPT if impl == TC else STEP
    c, q = _case(spec)
    t = c.table.clone()
    t[0, 1], t[1, 0] = -5, c.pages
    c.table = t
    dst = torch.zeros_like(q)
    run_attention(gpu, c, q, dst, 0.1, impl)
    T.bad_wait(s)
    # the definition, without these tokens
    good = Cache(**spec, seed=5)
    c.np_table = good.np_table
    want = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    group = q.shape[1] // c.heads
    hide = {0: (c.page, 2 * c.page), 1: (0, c.page)}
    for b, (n, length) in enumerate(zip(c.news, c.lens)):
        begin = int(c.np_off[b])
        k, v = (c.dense(w, b, length).repeat_interleave(group, 1).transpose(0, 1) for w in (0, 1))
        z = q[begin:begin + n].double().transpose(0, 1) @ k.transpose(1, 2) * 0.1
        at = length - n + torch.arange(n, device="cuda")
        tok = torch.arange(length, device="cuda")
        hidden = tok[None] > at[:, None]
        if b in hide:
            hidden = hidden | ((tok >= hide[b][0]) & (tok < hide[b][1]))[None]
        pr = torch.exp(z - z.masked_fill(hidden, -1e300).amax(-1, keepdim=True).clamp_min(-1e3)).masked_fill(hidden, 0)
        l = pr.sum(-1, keepdim=True)
        want[begin:begin + n] = (pr @ v / l.clamp_min(1e-300)).transpose(0, 1)  # rows that see nothing: 0
    # 2^-11 for the weights, 2^-8 for the result, both of values up to the largest
    top = max(float(c.dense(1, b, n).abs().max()) for b, n in enumerate(c.lens) if n)
    assert ((dst.double() - want).abs() <= want.abs() * 2.0 ** -8 + top * 2.0 ** -10).all()
    # lengths that the table does not hold: only the tokens that it holds are seen, and it is reported
    c2, q2 = _case(spec)
    c2.kv_lens += 100000
    run_attention(gpu, c2, q2, dst, 0.1, impl)
    T.bad_wait(s)
    assert not torch.isnan(dst).any()


@pytest.mark.gpu
@pytest.mark.parametrize("spec", [STEP, PROMPT])
def test_buffers_that_vector_accesses_cannot_start_at(gpu, spec):
    """Queries one element behind a 16-byte boundary: the primitive's kernel cannot take them, the generic one does."""
    torch, _ = T._torch()
    e, s = gpu
    c, q = _case(spec)
    wide = torch.zeros(q.numel() + 8, dtype=q.dtype, device="cuda")
    off = wide[1:1 + q.numel()].view(q.shape)
    off.copy_(q)
    dst = torch.zeros_like(q)
    run_attention(gpu, c, off, dst, 0.1)
    s.wait()
    check_attention(c, q, 0.1, dst, dst, "bf16")


@pytest.mark.gpu
def test_addresses_within_an_element_are_refused(gpu):
    """Refused on the host: a buffer that starts inside an element of its type, a scratchpad that 16 bytes do not divide."""
    torch, _ = T._torch()
    e, s = gpu
    c, q = _case(STEP)
    dst = torch.zeros_like(q)
    a = api.PrimitiveAttr()
    a.set_scratchpad_mode(1)
    pd = api.kv_cache_attention_primitive_desc(e, tmd(q), tmd(c.codes[0]), tmd(dst), tmd(c.table), 0.1, attr=a)
    n = pd.scratchpad_desc().get_size()
    buf = torch.zeros(n + 1024, dtype=torch.uint8, device="cuda")
    p = api.Primitive(pd)
    args = {**c.args(e), api.ARG_SRC: mem(q, e), api.ARG_DST: mem(dst, e),
            api.ARG_SCRATCHPAD: api.Memory(pd.scratchpad_desc(), e, buf.data_ptr())}

    def refused(prim, a):
        with pytest.raises(api.Error) as err:
            prim.execute(s, a)
        assert err.value.name == "invalid_arguments"
    for off in (1, 4, 8):
        refused(p, {**args, api.ARG_SCRATCHPAD: api.Memory(pd.scratchpad_desc(), e, buf.data_ptr() + off)})
    for arg, t in ((api.ARG_SRC, q), (api.ARG_DST, dst), (api.ARG_B200_KEY_SCALES, c.scales[0]), (api.ARG_B200_PAGE_TABLE, c.table),
                   (api.ARG_B200_SEQ_OFFSETS, c.offsets), (api.ARG_B200_KV_LENS, c.kv_lens)):
        refused(p, {**args, arg: api.Memory(tmd(t), e, t.data_ptr() + 1)})
    p.execute(s, args)
    s.wait()
    check_attention(c, q, 0.1, dst, dst, "bf16")

    x, y = torch.randn(8, 64, device="cuda"), torch.zeros(8, 64, dtype=torch.int8, device="cuda")
    scales = torch.zeros(8, device="cuda")
    norm = api.Primitive(api.rms_norm_primitive_desc(e, tmd(x), tmd(y), 1e-5))
    where = api.ARG_ATTR_SCALES | api.ARG_DST
    good = {api.ARG_SRC: mem(x, e), api.ARG_DST: mem(y, e), where: mem(scales, e)}
    refused(norm, {**good, where: api.Memory(tmd(scales), e, scales.data_ptr() + 2)})
    refused(norm, {**good, api.ARG_SRC: api.Memory(tmd(x), e, x.data_ptr() + 2)})
    norm.execute(s, good)
    s.wait()


@pytest.mark.gpu
def test_append_wants_two_caches(gpu):
    """Keys and values written into one cache, or two caches with one set of scales, would race."""
    torch, _ = T._torch()
    e, s = gpu
    c = Cache([20, 3], [2, 3], 2, 16, 64, "s8")
    x = torch.randn(c.rows, 2, 64, generator=c.g, device="cuda")
    before = [t.clone() for t in c.codes + c.scales]
    p = api.Primitive(api.kv_cache_append_primitive_desc(e, tmd(x), tmd(c.codes[0]), tmd(c.table)))
    args = {**c.args(e), api.ARG_SRC: mem(x, e), api.ARG_SRC_1: mem(x, e)}
    for one, other in ((api.ARG_B200_KEY_CACHE, api.ARG_B200_VALUE_CACHE), (api.ARG_B200_KEY_SCALES, api.ARG_B200_VALUE_SCALES)):
        with pytest.raises(api.Error) as err:
            p.execute(s, {**args, other: args[one]})
        assert err.value.name == "invalid_arguments"
    s.wait()
    for was, now in zip(before, c.codes + c.scales):
        assert torch.equal(T.bits(was), T.bits(now))


@pytest.mark.gpu
def test_a_cache_beyond_four_gigabytes(gpu):
    """Pages whose codes lie behind 2^32 bytes: append, read and both attention kernels find them."""
    torch, _ = T._torch()
    e, s = gpu
    heads, page, dim = 8, 16, 128
    pages = (1 << 32) // (heads * page * dim) + 64
    c = Cache([100, 60], [40, 1], heads, page, dim, "s8")
    small = [t.clone() for t in c.codes + c.scales]
    big = [torch.zeros(pages, heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, heads, device="cuda") for _ in range(2)]
    shift = pages - c.pages
    for i in range(2):
        big[i][shift:] = c.codes[i]
        scales[i][shift:] = c.scales[i]
    x = torch.randn(41, heads, dim, generator=c.g, device="cuda").to(torch.bfloat16)
    want = [expected_append(c, x, c.codes[i], c.scales[i]) for i in range(2)]
    c.codes, c.scales, c.pages = big, scales, pages
    c.np_table = np.where(c.np_table < 1 << 20, c.np_table + shift, c.np_table).astype(np.int32)
    c.table = torch.from_numpy(c.np_table).cuda()
    run_append(gpu, c, x, x)
    s.wait()
    for i in range(2):
        assert torch.equal(c.codes[i][shift:], want[i][0]) and torch.equal(c.scales[i][shift:], want[i][1])
        assert not c.codes[i][:shift].any()
    out = torch.zeros(2, 41, heads, dim, dtype=torch.bfloat16, device="cuda")
    p = api.Primitive(api.kv_cache_read_primitive_desc(e, tmd(c.codes[0]), tmd(out[0]), tmd(c.table)))
    p.execute(s, {**c.args(e), api.ARG_DST: mem(out[0], e), api.ARG_DST_1: mem(out[1], e)})
    s.wait()
    new = torch.cat([c.dense(0, 0, 100)[60:], c.dense(0, 1, 60)[59:]])
    assert ((out[0].double() - new).abs() <= new.abs() * 2.0 ** -8).all()
    for impl in (TC, MMA, GENERIC):
        q = torch.randn(41, 4 * heads, dim, generator=c.g, device="cuda").to(torch.bfloat16)
        dst = torch.zeros_like(q)
        run_attention(gpu, c, q, dst, 0.1, impl)
        s.wait()
        check_attention(c, q, 0.1, dst, dst, "bf16")
    del small


@pytest.mark.gpu
def test_a_layer_from_norm_to_norm(gpu):
    """norm -> int8 matmul with the row scales that the norm wrote -> its columns into the cache -> attention -> 4-bit weights
    matmul -> norm of the result and the residual stream, twice: a prompt in two sequences, then a step.  Every operator
    is checked on what the one before left on the device."""
    torch, _ = T._torch()
    e, s = gpu
    hidden, heads, group, dim, page = 512, 2, 4, 64, 16
    q_heads, width = heads * group, (heads * group + 2 * heads) * dim
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    gamma = torch.rand(hidden, generator=g, device="cuda") + 0.5
    wq = torch.randint(-127, 128, (hidden, width), generator=g, device="cuda", dtype=torch.int8)
    wq_scale = (torch.rand(width, generator=g, device="cuda") + 0.5) / 2000
    wo = torch.randint(-8, 8, (q_heads * dim, hidden), generator=g, device="cuda", dtype=torch.int32)
    packed = ((wo[:, 0::2] & 15) | (wo[:, 1::2] & 15) << 4).to(torch.uint8).contiguous()  # two columns per byte
    wo_scale = ((torch.rand(q_heads * dim // 64, hidden, generator=g, device="cuda") + 0.5) / 50).to(torch.bfloat16)
    c = Cache([70, 45], [70, 45], heads, page, dim, "s8", columns=8)
    stream = torch.randn(115, hidden, generator=g, device="cuda") * 2

    def weights(pd, plain_md, plain):
        if pd.weights_desc() == plain_md:
            return plain
        m = api.Memory(pd.weights_desc(), e)
        api.Primitive(api.reorder_primitive_desc(e, plain_md, e, pd.weights_desc())).execute(s, {api.ARG_FROM: plain, api.ARG_TO: m})
        return m

    def layer(rows, residual, delta):
        """delta: what the layer before adds to the residual stream, bf16"""
        codes, scales, total = torch.zeros(rows, hidden, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda"), residual.clone()
        n = api.Primitive(api.rms_norm_primitive_desc(e, tmd(delta), tmd(codes), 1e-5, scale_md=tmd(gamma), residual_md=tmd(total)))
        n.execute(s, {api.ARG_SRC: mem(delta, e), api.ARG_SRC_1: mem(total, e), api.ARG_DST_1: mem(total, e), api.ARG_SCALE: mem(gamma, e),
                      api.ARG_DST: mem(codes, e), api.ARG_ATTR_SCALES | api.ARG_DST: mem(scales, e)})
        qkv = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
        a = api.PrimitiveAttr()
        a.set_scales(api.ARG_SRC, 3, (1, hidden), dt.F32)
        a.set_scales(api.ARG_WEIGHTS, 2, (), dt.F32)
        plain = md((hidden, width), "s8")
        pd = api.matmul_primitive_desc(e, tmd(codes), api.MemoryDesc((hidden, width), dt.S8, api.TAG_ANY), tmd(qkv), attr=a)
        assert pd.impl_info_str() == "cuda:sm100:tcgen05_i8"
        w = weights(pd, plain, mem(wq, e))
        api.Primitive(pd).execute(s, {api.ARG_SRC: mem(codes, e), api.ARG_WEIGHTS: w, api.ARG_DST: mem(qkv, e),
                                      api.ARG_ATTR_SCALES | api.ARG_SRC: mem(scales, e), api.ARG_ATTR_SCALES | api.ARG_WEIGHTS: mem(wq_scale, e)})
        v = qkv.view(rows, q_heads + 2 * heads, dim)
        q, k, val = v[:, :q_heads], v[:, q_heads:q_heads + heads], v[:, q_heads + heads:]
        s.wait()
        want_cache = [expected_append(c, x, c.codes[i], c.scales[i]) for i, x in enumerate((k, val))]
        run_append(gpu, c, k, val)
        out = torch.zeros(rows, q_heads, dim, dtype=torch.bfloat16, device="cuda")
        run_attention(gpu, c, q, out, dim ** -0.5)
        y = torch.zeros(rows, hidden, dtype=torch.bfloat16, device="cuda")
        a2 = api.PrimitiveAttr()
        a2.set_fpmath_mode(1, True)
        a2.set_scales(api.ARG_WEIGHTS, 3, (64, 1), dt.BF16)
        flat = out.view(rows, q_heads * dim)
        pd2 = api.matmul_primitive_desc(e, tmd(flat), api.MemoryDesc((q_heads * dim, hidden), dt.S4, api.TAG_ANY), tmd(y), attr=a2)
        plain2 = api.MemoryDesc((q_heads * dim, hidden), dt.S4, api.TAG_AB)
        w2 = weights(pd2, plain2, api.Memory(plain2, e, packed.data_ptr()))
        api.Primitive(pd2).execute(s, {api.ARG_SRC: mem(flat, e), api.ARG_WEIGHTS: w2, api.ARG_DST: mem(y, e),
                                       api.ARG_ATTR_SCALES | api.ARG_WEIGHTS: mem(wo_scale.view(-1), e)})
        s.wait()
        check_norm(delta, residual, gamma, codes, 1e-5, total, scales, "s8")
        exact = (codes.double() @ wq.double()) * scales.double()[:, None] * wq_scale.double()
        assert ((qkv.double() - exact).abs() <= exact.abs() * (2.0 ** -8 + 4 * T.U) + 1e-30).all()  # exact sums, one rounding to bf16
        for i in range(2):
            assert torch.equal(c.codes[i].contiguous(), want_cache[i][0]) and torch.equal(c.scales[i], want_cache[i][1])
        check_attention(c, q, dim ** -0.5, out, out, "bf16")
        dense = wo.double() * wo_scale.double().repeat_interleave(64, 0)
        ref, size = flat.double() @ dense, flat.double().abs() @ dense.abs()
        # weights rounded to bf16 where the kernel does that (2^-8 each at most), the result once more
        assert ((y.double() - ref).abs() <= size * 2.0 ** -8 + ref.abs() * 2.0 ** -8).all()
        return total, y

    residual, delta = layer(115, stream, torch.zeros(115, hidden, dtype=torch.bfloat16, device="cuda"))
    assert torch.equal(residual, stream)
    # a step: each sequence's last row goes on
    last = torch.tensor([69, 114], device="cuda")
    c.lens, c.news = [71, 46], [1, 1]
    c.np_off = np.array([0, 1, 2], dtype=np.int32)
    c.offsets = torch.from_numpy(c.np_off).cuda()
    c.kv_lens = torch.tensor([71, 46], dtype=torch.int32, device="cuda")
    total, _ = layer(2, residual[last].contiguous(), delta[last].contiguous())
    assert torch.equal(total, residual[last] + delta[last].float())


@pytest.mark.gpu
def test_norm_in_front_of_an_fp8_matmul(gpu):
    """The fp8 matmul takes the row scales as a binary multiplication over (rows, 1)."""
    torch, _ = T._torch()
    e, s = gpu
    rows, hidden, width = 48, 256, 128
    x = torch.randn(rows, hidden, device="cuda").to(torch.bfloat16)
    codes, scales = torch.zeros(rows, hidden, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(rows, device="cuda")
    api.Primitive(api.rms_norm_primitive_desc(e, tmd(x), tmd(codes), 1e-5)).execute(
        s, {api.ARG_SRC: mem(x, e), api.ARG_DST: mem(codes, e), api.ARG_ATTR_SCALES | api.ARG_DST: mem(scales, e)})
    w = torch.randn(hidden, width, device="cuda").to(torch.float8_e4m3fn)
    y = torch.zeros(rows, width, dtype=torch.bfloat16, device="cuda")
    po = api.PostOps()
    by_row = scales.view(rows, 1)
    po.append_binary(0x1fff1, tmd(by_row))
    a = api.PrimitiveAttr()
    a.set_post_ops(po)
    pd = api.matmul_primitive_desc(e, tmd(codes), tmd(w), tmd(y), attr=a)
    assert pd.impl_info_str() == "cuda:sm100:tcgen05_f8"
    api.Primitive(pd).execute(s, {api.ARG_SRC: mem(codes, e), api.ARG_WEIGHTS: mem(w, e), api.ARG_DST: mem(y, e),
                                  api.arg_post_op(0) | api.ARG_SRC_1: mem(by_row, e)})
    s.wait()
    a64, b64 = codes.float().double(), w.float().double()
    exact = (a64 @ b64) * scales.double()[:, None]
    size = (a64.abs() @ b64.abs()) * scales.double()[:, None]
    # f32 sums in the matrix unit, which keeps some 13 bits below the largest product of an instruction; one rounding to bf16
    assert ((y.double() - exact).abs() <= size * 2.0 ** -11 + exact.abs() * 2.0 ** -8).all()
