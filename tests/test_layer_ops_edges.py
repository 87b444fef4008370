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
