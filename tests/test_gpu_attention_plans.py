"""Plans of many rows: built in several launches."""
import numpy as np
import pytest

import fusedmm_amd as fa

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,degree,shared", [(1300000, 2, False), (4400000, 1, True)])
def test_a_plan_in_several_launches(rows, degree, shared):
    """More chunks than one launch takes: blocks of 16 rows without common columns, blocks of 64 rows with one column each; a
    long row near either end."""
    import torch
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(3)
    n = rows if not shared else 1000
    lengths = torch.full((rows,), degree, dtype=torch.int64, device=dev)
    lengths[5] = lengths[rows - 3] = 1500
    lengths[7::1000] = 0
    ptr = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), lengths.cumsum(0)])
    nnz = int(ptr[-1])
    row = torch.repeat_interleave(torch.arange(rows, device=dev), lengths)
    if shared:
        indx = (row // 64 * 7) % n
        long = (row == 5) | (row == rows - 3)
        indx = torch.where(long, torch.arange(nnz, device=dev) % n, indx)
    else:
        indx = torch.randint(0, n, (nnz,), generator=gen, device=dev)
    i32 = lambda x: x.to(torch.int32)
    plan = fa.AttnPlan(rows, n, nnz, i32(indx), i32(ptr[:-1]), i32(ptr[1:]))
    q, k, v = [torch.randn((x, 8), generator=gen, device=dev) for x in (rows, n, n)]
    d = fa.AttnDesc(type=fa.TYPE_F32, maps=1, m=rows, n=n, heads=1, kv_heads=1, d=8, dv=8, scale=0.5, ldq=8, hdq=8, ldk=8, hdk=8, ldv=8, hdv=8,
                    ldo=8, hdo=8)
    size = fa.fusedMM_attn_workspace(d, plan)
    work = torch.empty(max(size, 16), dtype=torch.uint8, device=dev)
    o = torch.full((rows, 8), 7.5, device=dev)
    assert fa.fusedMM_attn_forward(d, plan, q, k, v, None, o, None, None, work, size) == 0
    # scores are at most 40 in size: their exponentials need no maximum in 64 bits
    w = torch.exp(0.5 * (q.double()[row] * k.double()[indx]).sum(1))
    total = torch.zeros(rows, dtype=torch.float64, device=dev).index_add_(0, row, w)
    want = torch.zeros((rows, 8), dtype=torch.float64, device=dev).index_add_(0, row, w[:, None] * v.double()[indx])
    want = torch.where(lengths[:, None] > 0, want / total.clamp(min=1e-300)[:, None], torch.zeros_like(want))
    # fp32: scores of up to 8 products off by 16 * 2^-24 of their size (at most 40), sums of up to 1500 weights, values up to 6
    assert float((o.double() - want).abs().max()) <= 6 * (40 * 16 + 1500 + 32) * 2.0 ** -24
