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
