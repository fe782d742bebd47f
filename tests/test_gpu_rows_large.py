"""GPU: tables larger than the caches, whose codes are read in another way, against products in 64 bits of the decoded rows;
encoding by blocks of 16 rows (many rows, short rows) and of four (few long rows)."""
import numpy as np
import pytest
import torch

from vectordb_amd import rows as R

import rows_reference as ref

pytestmark = pytest.mark.gpu


def _tolerance(v, q, d, metric):
    """rows_reference.distance_tolerance for f64 tensors v [n, dim], q [nq, dim], d [nq, n]: the f32 rounding of the result,
    the query's fixed point (2^-30 of its largest magnitude per component), f64 sums of fewer than 4096 terms on both sides."""
    fixed = 2.0 ** -30 * q.abs().amax(1)[:, None] * v.abs().sum(1)[None, :]
    mag = q.abs() @ v.abs().t().contiguous()
    vv, qq = (v * v).sum(1)[None, :], (q * q).sum(1)[:, None]
    scale = 1.0 / torch.sqrt(vv * qq) if metric == "cosine" else 2.0 if metric == "l2" else 1.0
    extra = 1.0 + mag * scale if metric == "cosine" else vv + qq + 2 * mag if metric == "l2" else mag
    return 2.0 ** -24 * d.abs() + fixed * scale + 2 * 4096 * 2.0 ** -53 * extra + 2.0 ** -149


def _distances(v, q, metric):
    p = q @ v.t().contiguous()
    vv, qq = (v * v).sum(1)[None, :], (q * q).sum(1)[:, None]
    return -p if metric == "dot" else 1.0 - p / torch.sqrt(vv * qq) if metric == "cosine" else (vv + qq - 2.0 * p).clamp_min(0.0)


# codes of more than 256 MB: rows of one unit, of six, of seven (an odd last unit); queries that are one pass (up to four),
# and a few that are not
@pytest.mark.parametrize("n,dim,group,nq,metric", [(8_500_003, 64, 32, 1, "l2"), (8_500_003, 50, 64, 3, "cosine"), (1_500_001, 384, 128, 1, "dot"),
                                                   (1_500_001, 384, 32, 4, "cosine"), (1_300_007, 400, 64, 2, "l2"), (1_300_007, 400, 128, 6, "l2")])
def test_distances_of_large_tables(gpu, n, dim, group, nq, metric):
    dev = torch.device("cuda", gpu)
    gen = torch.Generator(device=dev)
    gen.manual_seed(n + dim)
    table, step = R.Int4Rows.empty(n, dim, group, dev), 250_000
    for a in range(0, n, step):
        table.encode_device(torch.randn((min(step, n - a), dim), generator=gen, device=dev), first_row=a)
    q = torch.randn((nq, dim), generator=gen, device=dev)
    got = table.distances_device(q, metric)
    for a in range(0, n, step):
        v = table.lookup_device(torch.arange(a, min(a + step, n), device=dev)).double()
        want = _distances(v, q.double(), metric)
        assert bool(((got[:, a:a + step].double() - want).abs() <= _tolerance(v, q.double(), want, metric)).all()), a


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim,group", [(129, 32), (300, 128), (768, 64), (1537, 32)])
def test_encode_few_and_many_rows_alike(gpu, dim, group, dtype):
    """9000 rows at once (16 per block) and in pieces (four per block) are the same codes and scales; norms add the same
    terms in another order."""
    dev = torch.device("cuda", gpu)
    gen = torch.Generator(device=dev)
    gen.manual_seed(dim)
    n = 9000
    x = (torch.randn((n, dim), generator=gen, device=dev) * torch.exp(torch.randn((n, 1), generator=gen, device=dev))).to(dtype)
    whole, parts = R.int4_encode_device(x, group), R.Int4Rows.empty(n, dim, group, dev)
    for a, b in ((0, 1), (1, 5000), (5000, 5003), (5003, 9000)):
        parts.encode_device(x[a:b], first_row=a)
    assert torch.equal(whole.decode_device(), parts.decode_device()) and torch.equal(whole.scales, parts.scales)
    values = ref.encode(x[:300].double().cpu().numpy(), group)
    assert np.array_equal(whole.decode_device()[:300].double().cpu().numpy(), values[2])
    for r in (whole, parts):
        v = r.decode_device().double()
        want = (v * v).sum(1)
        # at most dim f64 terms of one sign in each sum
        assert bool(((r.sqnorm - want).abs() <= 2 * dim * 2.0 ** -52 * want).all())
