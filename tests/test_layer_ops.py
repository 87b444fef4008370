"""The operators around the matmul of a transformer's layer: fused norm with an 8-bit destination, the paged 8-bit cache
of keys and values, attention over it -- against their definitions in 64 bits, and their refusals.

Tolerances count roundings: u = 2^-24 for one f32 operation, half a step of the destination's type for the last one.
"""
import ctypes as C
import math
import os

import numpy as np
import pytest

os.environ.setdefault("ONEDNN_B200_ALLOW_NO_DEVICE", "1")

from onednn_b200 import api, dtypes as dt  # noqa: E402

U = 2.0 ** -24
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative: finfo(type).eps / 2
CODE = {"f32": dt.F32, "bf16": dt.BF16, "f16": dt.F16, "s8": dt.S8, "e4m3": dt.F8_E4M3, "s32": dt.S32}
PEAK = {"s8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -126


def _torch():
    import torch
    t = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "s8": torch.int8, "e4m3": torch.float8_e4m3fn,
         "s32": torch.int32}
    return torch, t


# ---- descriptors and refusals (no GPU needed) -----------------------------------------------------------------

@pytest.fixture(scope="module")
def eng():
    return api.Engine()


def md(shape, kind, strides=None):
    if strides is None:
        strides = [int(np.prod(shape[i + 1:], dtype=np.int64)) for i in range(len(shape))]
    return api.MemoryDesc(tuple(shape), CODE[kind], strides=tuple(strides))


def refused(status, f, *a, **k):
    with pytest.raises(api.Error) as e:
        f(*a, **k)
    assert e.value.name == status


def test_norm_descriptors_and_refusals(eng):
    f = api.rms_norm_primitive_desc
    x, g = md((4, 64), "bf16"), md((64,), "f32")
    pd = f(eng, x, md((4, 64), "s8"), 1e-5, scale_md=g, residual_md=md((4, 64), "f32"))
    assert pd.impl_info_str() == "cuda:rms_norm"
    assert pd.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_ATTR_SCALES | api.ARG_DST).dims == [4]
    assert pd.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_DST_1).data_type == dt.F32
    assert pd.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_BIAS).ndims == 0
    L = api.lib()
    assert L.dnnl_primitive_desc_query_s32(pd.h, 3, 0) == 3 and L.dnnl_primitive_desc_query_s32(pd.h, 4, 0) == 3
    plain = f(eng, x, md((4, 64), "bf16"), 0.0)
    assert plain.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_ATTR_SCALES | api.ARG_DST).ndims == 0
    assert L.dnnl_primitive_desc_query_s32(plain.h, 3, 0) == 1 and L.dnnl_primitive_desc_query_s32(plain.h, 4, 0) == 1
    assert not plain.next_impl()
    # rows that fold, whatever the rank: a slice of every head; and rows that do not
    f(eng, md((2, 3, 5, 8), "f16", (240, 80, 16, 1)), md((2, 3, 5, 8), "f16"), 1e-5)
    refused("unimplemented", f, eng, md((2, 3, 8), "f16", (100, 8, 1)), md((2, 3, 8), "f16"), 1e-5)
    refused("unimplemented", f, eng, md((4, 64), "bf16", (1, 4)), md((4, 64), "bf16"), 1e-5)
    refused("invalid_arguments", f, eng, x, md((4, 65), "bf16"), 1e-5)
    refused("invalid_arguments", f, eng, x, md((2, 2, 64), "bf16"), 1e-5)
    refused("invalid_arguments", f, eng, x, x, 1e-5, scale_md=md((4,), "f32"))
    refused("invalid_arguments", f, eng, x, x, 1e-5, residual_md=md((1, 64), "bf16"))
    refused("invalid_arguments", md, (4, 64), "bf16", (32, 1))  # rows on one another: no descriptor
    for eps in (-1e-6, math.nan, math.inf):
        refused("invalid_arguments", f, eng, x, x, eps)
    refused("unimplemented", f, eng, md((4, 64), "s8"), x, 1e-5)
    refused("unimplemented", f, eng, x, md((4, 64), "s32"), 1e-5)
    refused("unimplemented", f, eng, x, x, 1e-5, residual_md=md((4, 64), "s8"))
    refused("unimplemented", f, eng, x, api.MemoryDesc((4, 64), dt.U8, api.TAG_AB), 1e-5)
    refused("unimplemented", f, eng, api.MemoryDesc((4, 64), dt.BF16, api.TAG_ANY), x, 1e-5)
    a = api.PrimitiveAttr()
    a.set_scales(api.ARG_DST, 0)
    refused("unimplemented", f, eng, x, md((4, 64), "s8"), 1e-5, attr=a)
    refused("unimplemented", f, api.Engine(kind=1), x, x, 1e-5)


def test_cache_descriptors_and_refusals(eng):
    x, c, t = md((6, 2, 64), "bf16"), md((5, 2, 16, 64), "s8"), md((3, 4), "s32")
    append, read, attend = api.kv_cache_append_primitive_desc, api.kv_cache_read_primitive_desc, api.kv_cache_attention_primitive_desc
    L = api.lib()
    for pd, ins, outs, name in ((append(eng, x, c, t), 5, 4, "cuda:kv_append"), (read(eng, c, x, t), 7, 2, "cuda:kv_read"),
                                (attend(eng, md((6, 8, 64), "bf16"), c, md((6, 8, 64), "bf16"), t, 0.125), 8, 1, None)):
        assert name is None or pd.impl_info_str() == name
        assert (L.dnnl_primitive_desc_query_s32(pd.h, 3, 0), L.dnnl_primitive_desc_query_s32(pd.h, 4, 0)) == (ins, outs)
        assert pd.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_B200_KEY_SCALES).dims == [5, 2]
        assert pd.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_B200_SEQ_OFFSETS).dims == [4]
        assert pd.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_B200_KV_LENS).dims == [3]
        assert pd.query_md(api.QUERY_EXEC_ARG_MD, api.ARG_B200_VALUE_CACHE) == c
    for f in (lambda x, c, t: append(eng, x, c, t), lambda x, c, t: read(eng, c, x, t),
              lambda x, c, t: attend(eng, x, c, x, t, 1.0)):
        refused("invalid_arguments", f, x, md((5, 2, 16), "s8"), t)
        refused("invalid_arguments", f, x, c, md((3,), "s32"))
        refused("invalid_arguments", f, x, c, md((3, 4), "f32"))
        refused("invalid_arguments", f, md((6, 2, 32), "bf16"), c, t)
        refused("invalid_arguments", f, md((6, 128), "bf16"), c, t)
        refused("invalid_arguments", f, md((6, 3, 64), "bf16"), c, t)
        refused("unimplemented", f, md((6, 2, 64), "s8"), c, t)
        refused("unimplemented", f, x, md((5, 2, 16, 64), "bf16"), t)
        refused("unimplemented", f, x, md((5, 2, 16, 64), "s8", (2048, 1024, 1, 16)), t)
        refused("unimplemented", f, md((6, 2, 64), "bf16", (128, 1, 2)), c, t)
    q = md((6, 8, 64), "bf16")
    refused("invalid_arguments", attend, eng, q, c, md((5, 8, 64), "bf16"), t, 1.0)
    refused("invalid_arguments", attend, eng, q, c, md((6, 4, 64), "bf16"), t, 1.0)
    refused("invalid_arguments", attend, eng, q, c, q, t, math.inf)
    refused("unimplemented", attend, eng, md((6, 2, 272), "bf16"), md((5, 2, 16, 272), "s8"), md((6, 2, 272), "bf16"), t, 1.0)
    # sizes that 32-bit counts inside the kernels do not hold
    for pages, h, page, dim in ((1, 1, 1 << 20, 2048), (1, 65535, 1, 1 << 15), (1, 1, (1 << 20) + 1, 16), (1, 65536, 1, 16)):
        refused("unimplemented", read, eng, md((pages, h, page, dim), "s8"), md((1, h, dim), "bf16"), t)
    refused("unimplemented", attend, eng, md((1 << 30, 4, 64), "bf16"), md((5, 2, 16, 64), "s8"), md((1 << 30, 4, 64), "bf16"), t, 1.0)
    a = api.PrimitiveAttr()
    po = api.PostOps()
    po.append_eltwise(0x20)
    a.set_post_ops(po)
    refused("unimplemented", attend, eng, q, c, q, t, 1.0, attr=a)


# ---- helpers for the GPU ---------------------------------------------------------------------------------------

@pytest.fixture(scope="module")
def gpu():
    torch, _ = _torch()
    e = api.Engine()
    return e, api.Stream(e, cuda_stream=torch.cuda.current_stream().cuda_stream)


def tmd(t):
    _, types = _torch()
    kind = {v: k for k, v in types.items()}[t.dtype]
    return md(tuple(t.shape), kind, tuple(t.stride()))


def mem(t, e):
    return api.Memory(tmd(t), e, t.data_ptr())


def bits(t):
    torch, _ = _torch()
    return t.contiguous().view(torch.uint8)


# ---- norm ------------------------------------------------------------------------------------------------------

def run_norm(gpu, src, residual, gamma, dst, eps, in_place=False):
    torch, _ = _torch()
    e, s = gpu
    args = {api.ARG_SRC: mem(src, e), api.ARG_DST: mem(dst, e)}
    scales = total = None
    if gamma is not None:
        args[api.ARG_SCALE] = mem(gamma, e)
    if residual is not None:
        total = residual if in_place else torch.full_like(residual, 7).as_strided(residual.shape, residual.stride())
        args.update({api.ARG_SRC_1: mem(residual, e), api.ARG_DST_1: mem(total, e)})
    if dst.dtype in (torch.int8, torch.float8_e4m3fn):
        rows = dst.numel() // dst.shape[-1]
        scales = torch.full((rows,), -1.0, device="cuda")
        args[api.ARG_ATTR_SCALES | api.ARG_DST] = mem(scales, e)
    pd = api.rms_norm_primitive_desc(e, tmd(src), tmd(dst), eps, scale_md=None if gamma is None else tmd(gamma),
                                     residual_md=None if residual is None else tmd(residual))
    p = api.Primitive(pd)
    p.execute(s, args)
    s.wait()
    return total, scales


def check_norm(src, residual_before, gamma, dst, eps, total, scales, dst_kind):
    """Against the definition.  The sum of squares is a chain of at most cols / 32 + 10 f32 additions of positive terms
    (a warp per row; longer rows have shorter chains per thread); half of its error remains behind the root."""
    torch, types = _torch()
    h = src.double()
    if residual_before is not None:
        h = h + residual_before.double()
        kind = {v: k for k, v in types.items()}[residual_before.dtype]
        f32 = src.float() + residual_before.float()
        assert torch.equal(bits(total), bits(f32.to(types[kind])))  # one addition, one rounding: no slack
    cols = src.shape[-1]
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    if gamma is not None:
        y = y * gamma.double()
    rel = (min(cols, 1056) / 32 / 2 + 10) * U * 2
    if dst_kind not in PEAK:
        err = (dst.double() - y).abs()
        floor = 2.0 ** -25 if dst_kind == "f16" else 2.0 ** -133  # half the smallest step
        assert (err <= y.abs() * (HALF[dst_kind] * (1 + rel) + rel) + floor).all()
        return
    top = y.abs().amax(-1)
    want = torch.clamp(top / PEAK[dst_kind], min=TINY).reshape(-1)
    assert ((scales.double() - want).abs() <= want * (rel + 3 * U)).all()
    t = y / want.view(*y.shape[:-1], 1)
    code = dst.float().double()
    slack = PEAK[dst_kind] * (2 * rel + 6 * U)
    half = 0.5 if dst_kind == "s8" else torch.clamp(t.abs() * 2.0 ** -4, min=2.0 ** -10)
    assert ((code - t).abs() <= half + slack).all()
    assert code.abs().max() <= PEAK[dst_kind]


NORMS = [  # rows, cols, src, residual, gamma, dst
    (1, 1, "f32", "f32", "f32", "s8"), (3, 7, "bf16", "", "", "bf16"), (5, 64, "bf16", "bf16", "f32", "s8"),
    (4, 128, "f16", "", "f16", "f16"), (17, 256, "bf16", "f32", "bf16", "e4m3"), (9, 257, "f16", "f16", "f32", "s8"),
    (2, 1000, "f32", "bf16", "f32", "e4m3"), (6, 1024, "bf16", "bf16", "f32", "bf16"), (3, 1032, "f16", "f32", "", "e4m3"),
    (5, 2050, "bf16", "bf16", "bf16", "f16"), (130, 4096, "bf16", "bf16", "f32", "s8"), (2, 8192, "f32", "f32", "f32", "f32"),
    (3, 8200, "bf16", "bf16", "f32", "s8"), (2, 8193, "f16", "f32", "f16", "s8"), (2, 32768, "bf16", "f32", "f32", "e4m3"),
    (2, 20001, "f16", "", "f32", "bf16"), (3, 33000, "bf16", "bf16", "f32", "s8"), (2, 40000, "f32", "", "", "f16"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,src,residual,gamma,dst", NORMS)
def test_norm(gpu, rows, cols, src, residual, gamma, dst):
    torch, types = _torch()
    torch.manual_seed(rows * 100003 + cols)
    x = (torch.randn(rows, cols, device="cuda") * 3).to(types[src])
    r = (torch.randn(rows, cols, device="cuda") * 5).to(types[residual]) if residual else None
    g = (torch.rand(cols, device="cuda") + 0.5).to(types[gamma]) if gamma else None
    out = torch.zeros(rows, cols, dtype=types[dst], device="cuda")
    total, scales = run_norm(gpu, x, r, g, out, 1e-5)
    check_norm(x, r, g, out, 1e-5, total, scales, dst)


@pytest.mark.gpu
@pytest.mark.parametrize("off,pitch", [(0, 160), (1, 160), (3, 137)])
def test_norm_strided_rows_in_place_and_untouched_neighbours(gpu, off, pitch):
    """Rows inside wider ones, at offsets that 16-byte accesses can and cannot start at; the residual stream updated in
    its own memory; nothing beside the rows written."""
    torch, types = _torch()
    torch.manual_seed(off)
    rows, cols = 21, 128
    wide = torch.randn(rows, pitch, device="cuda").to(torch.bfloat16)
    res = torch.randn(rows, pitch, device="cuda")
    out = torch.full((rows, pitch), 99, dtype=torch.int8, device="cuda")
    x, r, d = (t[:, off:off + cols] for t in (wide, res, out))
    r0, res0 = r.clone(), res.clone()
    g = torch.rand(cols, device="cuda") + 0.5
    total, scales = run_norm(gpu, x, r, g, d, 1e-6, in_place=True)
    check_norm(x, r0, g, d, 1e-6, total, scales, "s8")
    beside = torch.ones(pitch, dtype=torch.bool)
    beside[off:off + cols] = False
    beside = beside.cuda()
    assert (out[:, beside] == 99).all() and torch.equal(res[:, beside], res0[:, beside])


@pytest.mark.gpu
def test_norm_heads_of_a_projection(gpu):
    """(tokens, heads, dim) as a slice of a wider row: the leading dims fold although the rows are not dense."""
    torch, _ = _torch()
    qkv = torch.randn(11, 10, 64, device="cuda").to(torch.float16)
    x = qkv.view(11, 5, 2, 64)[:, :, 0]
    out = torch.zeros(11, 5, 64, dtype=torch.float16, device="cuda")
    run_norm(gpu, x, None, None, out, 1e-5)
    check_norm(x, None, None, out, 1e-5, None, None, "f16")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "e4m3"])
def test_norm_rows_of_zeros_infinities_and_nan(gpu, kind):
    """A row of zeros and one of the smallest values: the smallest scale, codes 0.  NaN, or an infinity (whose row has
    an infinite mean square: inf * 0), makes the row's scale NaN and leaves the other rows alone."""
    torch, types = _torch()
    x = torch.randn(6, 300, device="cuda")
    x[0] = 0
    x[1] = 1e-42
    x[2, 17] = math.nan
    x[3, 299] = math.inf
    out = torch.zeros(6, 300, dtype=types[kind], device="cuda")
    _, scales = run_norm(gpu, x, None, None, out, 0.25)
    assert scales[0] == TINY and scales[1] == TINY
    assert (out[:2].float() == 0).all()
    assert torch.isnan(scales[2:4]).all()
    check_norm(x[4:], None, None, out[4:], 0.25, None, scales[4:], kind)


@pytest.mark.gpu
def test_norm_no_rows(gpu):
    torch, _ = _torch()
    e, s = gpu
    x = api.MemoryDesc((0, 64), dt.BF16, api.TAG_AB)
    p = api.Primitive(api.rms_norm_primitive_desc(e, x, x, 1e-5))
    p.execute(s, {})
    s.wait()


# ---- the cache -------------------------------------------------------------------------------------------------

class Cache:
    """A paged cache with a shuffled table, in memory that may be strided, and the batch's offsets and lengths."""

    def __init__(self, lens, news, heads, page, dim, kind, seed=0, spare=2, pitch=None, before=0, behind=0, columns=None):
        torch, types = _torch()
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)
        self.lens, self.news, self.heads, self.page, self.dim, self.kind = list(lens), list(news), heads, page, dim, kind
        need = [max(0, -(-n // page)) for n in lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=self.g, device="cuda").cpu().tolist()
        cols = columns or max(need + [1])
        # entries that no token needs are never to be read: far outside the cache
        table = np.full((len(lens), cols), 0x7fffff00, dtype=np.int32)
        k = 0
        for b, n in enumerate(need):
            for j in range(min(n, cols)):
                table[b, j] = order[k]
                k += 1
        self.np_table = table
        self.table = torch.from_numpy(table).cuda()
        self.rows = before + sum(news) + behind
        off = before + np.concatenate([[0], np.cumsum(news)])
        self.np_off = off.astype(np.int32)
        self.offsets = torch.from_numpy(self.np_off).cuda()
        self.kv_lens = torch.from_numpy(np.asarray(lens, dtype=np.int32)).cuda()
        pitch = pitch or dim
        self.codes, self.scales = [], []
        for _ in range(2):
            raw = torch.randn(self.pages, heads, page, pitch, generator=self.g, device="cuda") * (40 if kind == "s8" else 120)
            raw = raw.round().clamp(-127, 127).to(torch.int8) if kind == "s8" else raw.clamp(-448, 448).to(torch.float8_e4m3fn)
            self.codes.append(raw[..., :dim])
            self.scales.append((torch.rand(self.pages, heads, generator=self.g, device="cuda") + 0.5) / 50)

    def args(self, e):
        return {api.ARG_B200_KEY_CACHE: mem(self.codes[0], e), api.ARG_B200_VALUE_CACHE: mem(self.codes[1], e),
                api.ARG_B200_KEY_SCALES: mem(self.scales[0], e), api.ARG_B200_VALUE_SCALES: mem(self.scales[1], e),
                api.ARG_B200_PAGE_TABLE: mem(self.table, e), api.ARG_B200_SEQ_OFFSETS: mem(self.offsets, e),
                api.ARG_B200_KV_LENS: mem(self.kv_lens, e)}

    def dense(self, which, b, n):
        """(n, heads, dim) in 64 bits: the sequence's first n tokens."""
        torch, _ = _torch()
        idx = torch.from_numpy(self.np_table[b, :-(-n // self.page)].astype(np.int64)).cuda()
        x = self.codes[which].contiguous().view(torch.int8)[idx].view(self.codes[which].dtype).double() * self.scales[which][idx].double()[..., None, None]
        return x.transpose(1, 2).reshape(-1, self.heads, self.dim)[:n]


def quantised(x, kind):
    """f32 values in units of the scale -> raw codes; every step here is one f32 operation, as in the kernel."""
    torch, types = _torch()
    x = torch.nan_to_num(x, nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-PEAK[kind], PEAK[kind])
    return x.round().to(torch.int8) if kind == "s8" else x.to(torch.float8_e4m3fn)


def expected_append(c, x, codes, scales):
    """The append restated in f32 torch operations, page by page, on copies."""
    torch, _ = _torch()
    raw, scales = codes.contiguous().view(torch.int8).clone(), scales.clone()
    for b, (n, length) in enumerate(zip(c.news, c.lens)):
        begin = int(c.np_off[b])
        i = max(0, n - length)
        while i < n:
            at = length - n + i
            phys, slot = int(c.np_table[b, at // c.page]), at % c.page
            count = min(c.page - slot, n - i)
            v = x[begin + i:begin + i + count].float().transpose(0, 1)  # (heads, count, dim)
            mag = torch.where(v.abs() < math.inf, v.abs(), torch.zeros_like(v)).amax((1, 2))
            one = torch.ones((), device="cuda")
            s = torch.maximum(mag * (one / PEAK[c.kind]).float(), torch.full_like(mag, TINY))
            if slot:
                old = scales[phys]
                s = torch.maximum(s, old)
                grown = s > old
                again = quantised(raw[phys, :, :slot].view(codes.dtype).float() * (old / s)[:, None, None], c.kind).view(torch.int8)
                raw[phys, :, :slot] = torch.where(grown[:, None, None], again, raw[phys, :, :slot])
            scales[phys] = s
            raw[phys, :, slot:slot + count] = quantised(v * s.reciprocal()[:, None, None], c.kind).view(torch.int8)
            i += count
    return raw, scales


def run_append(gpu, c, keys, values):
    e, s = gpu
    p = api.Primitive(api.kv_cache_append_primitive_desc(e, tmd(keys), tmd(c.codes[0]), tmd(c.table)))
    p.execute(s, {**c.args(e), api.ARG_SRC: mem(keys, e), api.ARG_SRC_1: mem(values, e)})
    return p


CACHES = [  # lens, news, heads, page, dim, kind, src, pitch, before, behind
    ([1], [1], 1, 1, 16, "s8", "f32", None, 0, 0),
    ([5, 17, 16, 1], [1, 1, 1, 1], 2, 16, 64, "s8", "bf16", None, 0, 0),
    ([100, 3, 64], [40, 3, 0], 3, 16, 128, "s8", "bf16", None, 0, 3),
    ([90, 0, 51], [90, 0, 2], 2, 24, 80, "e4m3", "f16", None, 2, 5),
    ([33, 200], [33, 70], 2, 7, 20, "s8", "f32", None, 0, 0),
    ([33, 9], [10, 9], 1, 64, 13, "e4m3", "bf16", 15, 1, 1),
    ([300], [300], 8, 128, 128, "e4m3", "bf16", 144, 0, 0),
    ([40, 41], [7, 8], 2, 32, 256, "s8", "f16", 256, 0, 0),
    ([3, 20], [5, 2], 2, 8, 32, "s8", "f32", None, 0, 0),  # more rows than tokens: the first two rows stand for none
    (list(range(1, 161)), [1] * 160, 1, 16, 64, "s8", "bf16", None, 0, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news,heads,page,dim,kind,src,pitch,before,behind", CACHES)
def test_append_and_read(gpu, lens, news, heads, page, dim, kind, src, pitch, before, behind):
    """Append restated in f32 step by step gives the same bytes; nothing else of the cache changes; read back is
    code * scale rounded once."""
    torch, types = _torch()
    e, s = gpu
    c = Cache(lens, news, heads, page, dim, kind, seed=sum(lens), pitch=pitch, before=before, behind=behind)
    # keys and values as slices of one projection
    kv = (torch.randn(c.rows, 2 * heads + 1, dim, generator=c.g, device="cuda") * torch.rand(c.rows, 1, 1, generator=c.g, device="cuda") * 4).to(types[src])
    keys, values = kv[:, :heads], kv[:, heads:2 * heads]
    want = [expected_append(c, x, c.codes[i], c.scales[i]) for i, x in enumerate((keys, values))]
    beside = [t.as_strided((c.pages, heads, page, (pitch or dim) - dim), t.stride(), t.storage_offset() + dim).clone() for t in c.codes] if pitch and pitch > dim else None
    run_append(gpu, c, keys, values)
    s.wait()
    for i in range(2):
        assert torch.equal(c.scales[i], want[i][1])
        assert torch.equal(c.codes[i].contiguous().view(torch.int8), want[i][0])
        if beside:
            now = c.codes[i].as_strided(beside[i].shape, c.codes[i].stride(), c.codes[i].storage_offset() + dim)
            assert torch.equal(bits(now), bits(beside[i]))
    # the same tokens again: nothing grows, nothing changes
    run_append(gpu, c, keys, values)
    s.wait()
    for i in range(2):
        assert torch.equal(c.scales[i], want[i][1]) and torch.equal(c.codes[i].contiguous().view(torch.int8), want[i][0])

    # everything back, into rows wider than a head, with rows in front and behind that stay as they were
    front, back = 2, 3
    off = front + np.concatenate([[0], np.cumsum(lens)])
    c.offsets = torch.from_numpy(off.astype(np.int32)).cuda()
    rows = front + sum(lens) + back
    for to in ("f32", "bf16", "f16"):
        pad = 8 if dim % 8 == 0 else 1
        out = torch.full((2, rows, heads, dim + pad), 9, dtype=types[to], device="cuda")
        k, v = out[0, :, :, :dim], out[1, :, :, :dim]
        p = api.Primitive(api.kv_cache_read_primitive_desc(e, tmd(c.codes[0]), tmd(k), tmd(c.table)))
        p.execute(s, {**c.args(e), api.ARG_DST: mem(k, e), api.ARG_DST_1: mem(v, e)})
        s.wait()
        assert (out[..., dim:] == 9).all() and (out[:, :front] == 9).all() and (out[:, rows - back:] == 9).all()
        for i, got in enumerate((k, v)):
            for b, n in enumerate(lens):
                idx = torch.from_numpy(c.np_table[b, :-(-n // page)].astype(np.int64)).cuda()
                f = c.codes[i].contiguous().view(torch.int8)[idx].view(c.codes[i].dtype).float() * c.scales[i][idx][..., None, None]
                f = f.transpose(1, 2).reshape(-1, heads, dim)[:n].to(types[to])
                assert torch.equal(bits(got[off[b]:off[b + 1]]), bits(f))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "e4m3"])
def test_append_one_by_one_keeps_every_token_close(gpu, kind):
    """Tokens of growing size, one per call: the page's scale grows and the older codes are rounded again each time.
    Every rounding is off by at most half a step of a scale that is at most the last one's."""
    torch, _ = _torch()
    e, s = gpu
    page, heads, dim, n = 16, 2, 64, 40
    c = Cache([n], [1], heads, page, dim, kind)
    x = torch.randn(n, heads, dim, device="cuda") * torch.linspace(0.1, 6, n, device="cuda")[:, None, None]
    for i in range(n):
        c.kv_lens.fill_(i + 1)
        run_append(gpu, c, x[i:i + 1], -x[i:i + 1])
    s.wait()
    for which, sign in ((0, 1), (1, -1)):
        back = c.dense(which, 0, n) * sign
        for j in range(0, n, page):
            k = min(page, n - j)
            top = x[j:j + k].double().abs().amax((0, 2))  # per head: the page's last scale times the peak
            roundings = k
            if kind == "s8":
                step = (top / 127)[None, :, None]
                assert ((back[j:j + k] - x[j:j + k].double()).abs() <= 0.5 * roundings * step * 1.0001).all()
            else:
                # 2^-4 of the value per rounding (compounded), or half the subnormal step
                tol = x[j:j + k].double().abs() * ((1 + 2.0 ** -4) ** roundings - 1) + (top / 448 * 2.0 ** -10)[None, :, None] * roundings * 2
                assert ((back[j:j + k] - x[j:j + k].double()).abs() <= tol).all()
            assert torch.allclose(c.scales[which][int(c.np_table[0, j // page])].double(), top / PEAK[kind], rtol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["s8", "e4m3"])
def test_append_zeros_infinities_and_nan(gpu, kind):
    torch, _ = _torch()
    e, s = gpu
    c = Cache([8, 8], [8, 8], 1, 8, 32, kind)
    x = torch.randn(16, 1, 32, device="cuda")
    x[:8] = 0
    x[9, 0, 3], x[10, 0, 5], x[11, 0, 7] = math.inf, -math.inf, math.nan
    want = expected_append(c, x, c.codes[0], c.scales[0])
    run_append(gpu, c, x, x)
    s.wait()
    first, second = int(c.np_table[0, 0]), int(c.np_table[1, 0])
    assert c.scales[0][first, 0] == TINY and (c.codes[0][first].float() == 0).all()
    got = c.codes[0][second, 0].float()
    assert got[1, 3] == PEAK[kind] and got[2, 5] == -PEAK[kind] and got[3, 7] == 0
    assert torch.equal(c.codes[0].contiguous().view(torch.int8), want[0]) and torch.equal(c.scales[0], want[1])


def bad_wait(s):
    with pytest.raises(api.Error) as err:
        s.wait()
    assert err.value.name == "runtime_error"
    s.wait()  # reported once


@pytest.mark.gpu
def test_pages_outside_the_cache_are_reported_and_left_alone(gpu):
    """Indices below zero, one past the end and far outside, and lengths that the table does not hold."""
    torch, _ = _torch()
    e, s = gpu
    heads, page, dim = 2, 8, 32
    c = Cache([20, 20, 20, 100], [20, 20, 20, 6], heads, page, dim, "s8", columns=3)
    t = c.table.clone()
    t[0, 1], t[1, 0], t[2, 2] = -1, c.pages, 0x7fffffff
    c.table = t
    c.np_table = t.cpu().numpy()
    before = [x.clone() for x in c.codes]
    x = torch.randn(66, heads, dim, device="cuda").to(torch.bfloat16)
    run_append(gpu, c, x, x)
    bad_wait(s)
    touched = sorted({int(v) for v in t[:3].flatten().tolist() if 0 <= v < c.pages})
    others = [i for i in range(c.pages) if i not in touched]
    for i in range(2):
        assert torch.equal(bits(c.codes[i][others]), bits(before[i][others]))
    out = torch.full((2, 66, heads, dim), 5.0, device="cuda")
    p = api.Primitive(api.kv_cache_read_primitive_desc(e, tmd(c.codes[0]), tmd(out[0]), tmd(c.table)))
    p.execute(s, {**c.args(e), api.ARG_DST: mem(out[0], e), api.ARG_DST_1: mem(out[1], e)})
    bad_wait(s)
    assert (out[:, 8:16] == 0).all() and (out[:, 20:28] == 0).all() and (out[:, 56:60] == 0).all() and (out[:, 60:] == 0).all()
    assert (out[0, 0:8] != 0).any()


# ---- attention -------------------------------------------------------------------------------------------------

def run_attention(gpu, c, q, dst, scale, impl=None, stream=None, scratchpad="library"):
    e, s = gpu
    s = stream or s
    a = api.PrimitiveAttr()
    if scratchpad == "user":
        a.set_scratchpad_mode(1)
    pd = api.kv_cache_attention_primitive_desc(e, tmd(q), tmd(c.codes[0]), tmd(dst), tmd(c.table), scale, attr=a)
    while impl is not None and pd.impl_info_str() != impl:
        if not pd.next_impl():
            pytest.skip("%s does not take this case" % impl)
    args = {**c.args(e), api.ARG_SRC: mem(q, e), api.ARG_DST: mem(dst, e)}
    if scratchpad == "user" and pd.scratchpad_desc().ndims:
        args[api.ARG_SCRATCHPAD] = api.Memory(pd.scratchpad_desc(), e)
    p = api.Primitive(pd)
    p.execute(s, args)
    return p, args


def expected_attention(c, q, scale):
    """(result, sum of p |v| over sum of p, largest score in magnitude's terms), in 64 bits; rows of no sequence: None."""
    torch, _ = _torch()
    group = q.shape[1] // c.heads
    want = torch.full(q.shape, math.nan, dtype=torch.float64, device="cuda")
    size, reach = torch.zeros_like(want), torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device="cuda")
    for b, (n, length) in enumerate(zip(c.news, c.lens)):
        if not n:
            continue
        begin = int(c.np_off[b])
        x = q[begin:begin + n].double()
        if length == 0:
            want[begin:begin + n] = 0
            continue
        k, v = (c.dense(w, b, length).repeat_interleave(group, 1).transpose(0, 1) for w in (0, 1))
        z = x.transpose(0, 1) @ k.transpose(1, 2) * scale
        zabs = x.abs().transpose(0, 1) @ k.abs().transpose(1, 2) * abs(scale)
        at = length - n + torch.arange(n, device="cuda")
        hidden = torch.arange(length, device="cuda")[None] > at[:, None]
        z = z.masked_fill(hidden, -math.inf)
        p = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-1e300))
        p = p.masked_fill(hidden, 0)
        l = p.sum(-1, keepdim=True).clamp_min(1e-300)
        want[begin:begin + n] = (p @ v / l).transpose(0, 1)
        size[begin:begin + n] = (p @ v.abs() / l).transpose(0, 1)
        reach[begin:begin + n] = zabs.masked_fill(hidden, 0).amax(-1, keepdim=True).transpose(0, 1)
    return want, size, reach


def check_attention(c, q, scale, got, untouched, kind):
    """Products of the scores are exact in f32 (8 x 11 bits) and summed in f32: off by at most (dim + 8) u times the sum
    of their magnitudes, a little more where the matrix unit truncates (2^-22 instead of 2^-24); a score's error is its
    weight's relative error, in the numerator and the sum.  Weights may be rounded to f16 against the largest: 2^-11
    each, and 2^-25 of the largest for the very small ones, of which there are at most `length`.  The last rounding
    is the destination's."""
    torch, _ = _torch()
    want, size, reach = expected_attention(c, q, scale)
    seen = ~torch.isnan(want)
    longest = max(c.lens)
    score = (q.shape[2] + 8) * 2.0 ** -22 * reach + 64 * U
    vmax = torch.zeros_like(size)
    for b, (n, length) in enumerate(zip(c.news, c.lens)):
        if n and length:
            begin = int(c.np_off[b])
            vmax[begin:begin + n] = c.dense(1, b, length).abs().amax(0).repeat_interleave(q.shape[1] // c.heads, 0)[None]
    tol = size * (2.0 ** -11 + 2 * score + longest * U) + vmax * longest * 2.0 ** -25 + want.abs().nan_to_num() * HALF[kind] + 2.0 ** -24
    err = (got.double() - want).abs()
    assert not torch.isnan(got).any()
    assert (err[seen] <= tol[seen]).all(), "%g of the tolerance" % float((err[seen] / tol[seen]).max())
    assert torch.equal(bits(got[~seen]), bits(untouched[~seen]))


ATTEND = [  # lens, news, heads, group, page, dim, cache kind, q kind, before, behind
    ([1], [1], 1, 1, 1, 16, "s8", "bf16", 0, 0),
    ([37], [1], 2, 4, 16, 64, "e4m3", "f16", 0, 0),
    ([5, 300, 64, 1], [1, 1, 1, 1], 2, 8, 16, 64, "s8", "bf16", 0, 2),
    ([129, 1000, 33], [1, 1, 1], 4, 4, 64, 128, "s8", "bf16", 0, 0),
    ([500, 77], [1, 1], 2, 16, 24, 128, "e4m3", "bf16", 0, 0),
    ([260, 31, 0, 90], [5, 31, 0, 2], 2, 5, 24, 80, "e4m3", "f16", 3, 4),
    ([4, 10], [6, 3], 2, 2, 8, 32, "s8", "bf16", 0, 0),  # rows that see no token
    ([0, 12], [2, 1], 1, 3, 8, 48, "s8", "f16", 0, 0),  # a sequence without tokens
    ([200, 333], [200, 100], 2, 4, 16, 128, "s8", "bf16", 0, 0),
    ([150], [150], 1, 1, 128, 256, "e4m3", "bf16", 0, 0),
    ([700], [3], 1, 32, 200, 112, "s8", "f16", 0, 0),
    ([4097], [1], 1, 1, 128, 64, "s8", "bf16", 0, 0),
    ([3000, 11], [130, 1], 2, 2, 32, 176, "e4m3", "bf16", 0, 1),
    ([61, 62], [1, 2], 2, 3, 7, 20, "s8", "f16", 0, 0),  # rows of 20 bytes
    ([90, 45], [40, 45], 3, 7, 13, 96, "s8", "bf16", 1, 0),
    ([129], [129], 1, 1, 16, 128, "s8", "bf16", 0, 0),  # one row more than a tile of rows
    ([128, 257], [128, 257], 1, 2, 64, 64, "e4m3", "bf16", 0, 0),
    ([40, 1000], [3, 300], 2, 3, 48, 96, "s8", "f16", 0, 2),
    ([900, 10, 0], [257, 20, 3], 1, 4, 128, 128, "e4m3", "f16", 2, 0),  # rows that see no token
    ([5000], [64], 2, 1, 32, 128, "s8", "bf16", 0, 0),  # one item in many parts
    ([2100, 2100], [700, 650], 3, 2, 16, 80, "s8", "bf16", 0, 0),
    ([300, 77, 129], [150, 77, 129], 2, 2, 8, 128, "s8", "bf16", 0, 0),  # runs of 8 tokens
    ([1000, 300], [200, 300], 1, 4, 24, 64, "e4m3", "f16", 1, 1),
    ([613], [333], 2, 1, 200, 112, "e4m3", "bf16", 0, 0),
    ([50] * 70, [1] * 70, 1, 8, 16, 64, "s8", "bf16", 0, 0),
    ([1 + i * 37 % 200 for i in range(300)], [i % 3 for i in range(300)], 2, 2, 16, 64, "s8", "bf16", 0, 0),  # more than a block's threads
    ([30 + i * 7 % 90 for i in range(530)], [30 if i % 5 else 0 for i in range(530)], 1, 2, 16, 64, "s8", "f16", 1, 0),
    ([3000] + [2] * 130, [700] + [1] * 130, 1, 2, 8, 128, "e4m3", "bf16", 0, 0),  # a prompt among steps
]


@pytest.mark.gpu
@pytest.mark.parametrize("impl", [None, "cuda:sm100:kv_attention_mma", "cuda:generic"])
@pytest.mark.parametrize("lens,news,heads,group,page,dim,kind,src,before,behind", ATTEND)
def test_attention(gpu, impl, lens, news, heads, group, page, dim, kind, src, before, behind):
    torch, types = _torch()
    c = Cache(lens, news, heads, page, dim, kind, seed=len(lens) + dim, before=before, behind=behind)
    q = torch.randn(c.rows, heads * group, dim, generator=c.g, device="cuda").to(types[src])
    dst = torch.full_like(q, 3.0)
    kept = dst.clone()
    p, args = run_attention(gpu, c, q, dst, dim ** -0.5, impl)
    gpu[1].wait()
    check_attention(c, q, dim ** -0.5, dst, kept, src)


@pytest.mark.gpu
def test_attention_f32_rows(gpu):
    torch, _ = _torch()
    c = Cache([40, 9], [2, 1], 2, 16, 64, "s8")
    q = torch.randn(3, 4, 64, generator=c.g, device="cuda")
    dst = torch.zeros_like(q)
    run_attention(gpu, c, q, dst, 0.125)
    gpu[1].wait()
    check_attention(c, q, 0.125, dst, dst, "f32")
