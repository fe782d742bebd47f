"""GPU: the embedding table (vectordb_amd/rows.py) against its definitions in 64 bits (rows_reference.py)."""
import numpy as np
import pytest
import torch

from vectordb_amd import _ffi
from vectordb_amd import rows as R

import rows_reference as ref
from helpers import clustered

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _np(t):
    return t.detach().cpu().double().numpy()


def _rows(n, d, seed, dtype=F32, gpu=0):
    """Rows of several magnitudes, in the given type, on the GPU (the reference sees the same rounded values)."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, d)) * 10.0 ** rng.uniform(-3, 2, (n, 1))
    x[rng.random((n, d)) < 0.05] = 0.0
    return torch.from_numpy(x.astype(np.float32)).to(dtype).to(torch.device("cuda", gpu))


# ---- encoding ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,d", [(1, 1), (1, 64), (15, 33), (16, 128), (17, 65), (40, 960), (33, 129), (5, 200), (3, 1537)])
def test_encode_and_decode(gpu, n, d, group, dtype):
    x = _rows(n, d, n * 1000 + d + group, dtype)
    codes, scales, values, sq = ref.encode(_np(x), group)
    r = R.int4_encode_device(x, group)
    assert np.array_equal(_np(r.group_scales), scales.astype(np.float64))
    assert not _np(r.scales)[:, scales.shape[1]:].any()
    assert np.array_equal(_np(r.decode_device()), values)  # 12 significant bits: exact in f32
    # a sum of at most 2 * groups f64 terms of one sign, in another order than the reference's
    assert np.all(np.abs(_np(r.sqnorm) - sq) <= 4 * scales.shape[1] * 2.0 ** -52 * sq)
    for t in (F16, BF16):
        assert torch.equal(r.decode_device(t).cpu(), torch.from_numpy(values).to(F32).to(t))


def test_encode_special_groups(gpu):
    x = np.zeros((20, 130), dtype=np.float32)
    x[1, :4] = [7.0, 0.5, 1.5, -2.5]               # scale 1: halves to even
    x[2, 3], x[2, 100] = np.nan, 1.0               # one group NaN, the next fine
    x[3, 70] = -np.inf
    x[4] = 1e-45                                   # scale rounds to zero
    x[5] = 1e-39                                   # subnormal scale
    x[6, :] = np.linspace(-3.4e38, 3.4e38, 130)
    x[7, :64] = np.arange(64) * 1e-38
    x[8, :64] = -(np.arange(64) % 15 - 7) * np.float32(2.0 ** -133)
    x[9, 129] = 3.0
    for group in (32, 64, 128):
        codes, scales, values, sq = ref.encode(x, group)
        r = R.int4_encode_device(torch.from_numpy(x).cuda(gpu), group)
        assert np.array_equal(_np(r.group_scales), scales.astype(np.float64), equal_nan=True)
        assert np.array_equal(_np(r.decode_device()), values.astype(np.float32).astype(np.float64), equal_nan=True)
        assert np.array_equal(np.isnan(_np(r.sqnorm)), np.isnan(sq))
        q = torch.ones((2, 130), device=r.device)
        for metric in ("l2", "cosine", "dot"):
            d = _np(r.distances_device(q, metric))
            assert np.isnan(d[:, 2]).all() and np.isnan(d[:, 3]).all() and np.isfinite(d[:, 1]).all()
            if metric == "cosine":
                assert np.isnan(d[:, 0]).all()  # a zero vector has no direction


def test_encode_in_pieces_and_strides(gpu):
    x = _rows(100, 96, 3)
    whole = R.int4_encode_device(x, 32)
    wide = torch.full((100, 131), 7.0, device=x.device)
    wide[:, 5:101] = x
    strided = R.int4_encode_device(wide[:, 5:101], 32)  # rows 131 apart, not 16-byte aligned
    turned = R.int4_encode_device(x.t().contiguous().t(), 32)
    parts = R.Int4Rows.empty(100, 96, 32, x.device)
    for a, b in ((33, 70), (0, 1), (70, 100), (1, 33)):
        parts.encode_device(x[a:b], first_row=a)
    for o in (strided, turned, parts):
        assert torch.equal(o.decode_device(), whole.decode_device())
        assert torch.equal(o.scales, whole.scales) and torch.equal(o.sqnorm, whole.sqnorm)
    # what is not asked for stays
    before = whole.codes.clone()
    whole.encode_device(x[40:40], first_row=40)
    whole.encode_device(x[50:51], first_row=50)
    assert torch.equal(before, whole.codes)


# ---- distances --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("metric", ["l2", "cosine", "dot"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,d,nq", [(1, 1, 1), (5, 64, 1), (16, 33, 2), (100, 128, 1), (257, 960, 3), (1000, 96, 4), (129, 200, 5), (70, 768, 17),
                                    (333, 1537, 9), (2100, 64, 33), (50, 129, 64), (4100, 128, 130)])
def test_distances(gpu, n, d, nq, group, metric):
    x = _rows(n, d, n + d)
    q = _rows(nq, d, n + d + 1)
    x[0], q[0] = x[0] + 1.0, q[0] + 1.0  # no zero vector
    r = R.int4_encode_device(x, group)
    values = ref.encode(_np(x), group)[2]
    want = ref.distances(values, _np(q), metric)
    got = _np(r.distances_device(q, metric))
    tol = ref.distance_tolerance(values, _np(q), want, metric)
    ok = np.isfinite(want)
    assert np.array_equal(np.isnan(got), ~ok)
    assert np.all((np.abs(got - want) <= tol)[ok]), float((np.abs(got - want) / tol)[ok].max())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,d,nq", [(300, 2100, 20), (270, 4100, 36), (520, 330, 20), (40, 1100, 100), (290, 190, 97), (5000, 130, 40), (17, 2500, 12)])
def test_distances_many_queries(gpu, n, d, nq, group):
    """Five and eight quartets of queries per pass, whole in LDS and in parts, odd last units, waves without rows."""
    x, q = _rows(n, d, n + d), _rows(nq, d, n + d + 1)
    r = R.int4_encode_device(x, group)
    values = ref.encode(_np(x), group)[2]
    want = ref.distances(values, _np(q), "l2")
    got = _np(r.distances_device(q, "l2"))
    ok = np.isfinite(want)
    assert np.array_equal(np.isnan(got), ~ok)
    assert np.all((np.abs(got - want) <= ref.distance_tolerance(values, _np(q), want, "l2"))[ok])
    for i in (0, nq // 2, nq - 1):  # a query's distances do not depend on its neighbours
        assert np.array_equal(_np(r.distances_device(q[i:i + 1], "l2"))[0], got[i], equal_nan=True)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_distances_query_types(gpu, dtype):
    x, q = _rows(300, 192, 5), _rows(6, 192, 6, dtype)
    r = R.int4_encode_device(x, 64)
    values = ref.encode(_np(x), 64)[2]
    for metric in ("l2", "dot"):
        want = ref.distances(values, _np(q), metric)
        assert np.all(np.abs(_np(r.distances_device(q, metric)) - want) <= ref.distance_tolerance(values, _np(q), want, metric))


def test_distances_of_extreme_queries(gpu):
    x = _rows(40, 70, 8)
    r = R.int4_encode_device(x, 32)
    values = ref.encode(_np(x), 32)[2]
    q = _rows(8, 70, 9)
    q[0] = 0.0
    q[1] *= 1e30
    q[2] *= 1e-36
    q[3, 7] = 1e6     # one component far above the others
    q[4, 0] = float("nan")
    q[5, 69] = float("inf")
    q[6] = 1e-45
    got = _np(r.distances_device(q, "dot"))
    want = ref.distances(values, _np(q), "dot")
    fine = [0, 1, 2, 3, 6, 7]
    assert np.all(np.abs(got - want)[fine] <= ref.distance_tolerance(values, _np(q), want, "dot")[fine])
    assert np.isnan(got[[4, 5]]).all()
    assert not got[0].any()
    d = _np(r.distances_device(torch.from_numpy(values.astype(np.float32)).cuda(gpu), "l2"))  # the rows themselves
    own = ref.distances(values, values, "l2")
    assert (d >= 0).all() and np.all(np.abs(d - own) <= ref.distance_tolerance(values, values, own, "l2"))


def test_distances_of_extreme_rows(gpu):
    """Rows from 1e-36 to 1e36 against queries from 1e-9 to 1e9: products that f32 holds come out, others are infinite."""
    rng = np.random.default_rng(12)
    x = rng.standard_normal((73, 100)) * 10.0 ** np.linspace(-36, 36, 73)[:, None]
    q = rng.standard_normal((7, 100)) * 10.0 ** np.linspace(-9, 9, 7)[:, None]
    x, q = x.astype(np.float32), q.astype(np.float32)
    for group in (32, 64, 128):
        values = ref.encode(x, group)[2]
        r = R.int4_encode_device(torch.from_numpy(x).cuda(gpu), group)
        for metric in ("dot", "cosine", "l2"):
            want = ref.distances(values, q, metric)
            got = _np(r.distances_device(torch.from_numpy(q).cuda(gpu), metric))
            fits = np.abs(want) < 3.4e38
            tol = ref.distance_tolerance(values, q, want, metric)
            assert np.all((np.abs(got - want) <= tol)[fits]) and np.isinf(got[np.abs(want) > 3.41e38]).all()


def test_whole_numbers_are_exact(gpu):
    """SIFT-like rows whose groups all reach 7 * 2^j: scales are powers of two, every distance is a whole number."""
    rng = np.random.default_rng(2)
    c = rng.integers(-7, 8, (500, 128))
    c[:, ::32] = 7
    x = (c * 16.0).astype(np.float32)
    q = rng.integers(0, 256, (11, 128)).astype(np.float32)
    r = R.int4_encode_device(torch.from_numpy(x).cuda(gpu), 32)
    got = _np(r.distances_device(torch.from_numpy(q).cuda(gpu), "l2"))
    assert np.array_equal(got, ((q[:, None, :].astype(np.float64) - x[None].astype(np.float64)) ** 2).sum(2))


# ---- search -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n,d,nq,k,metric", [(1, 8, 2, 1, "l2"), (7, 64, 3, 10, "cosine"), (100, 32, 1, 100, "dot"), (8192, 64, 2, 10, "l2"),
                                             (8193, 64, 5, 1, "l2"), (20000, 48, 3, 1024, "cosine"), (100_000, 32, 2, 1000, "l2"), (70_000, 64, 9, 33, "dot"),
                                             (16384, 16, 1, 7, "l2"), (3000, 130, 40, 64, "l2"), (400_000, 16, 1, 200, "l2"), (50_000, 24, 1, 100, "cosine"),
                                             (30_000, 8, 3, 16, "dot")])
def test_search(gpu, n, d, nq, k, metric):
    x = torch.from_numpy(clustered(n, d, 30, n + d)).cuda(gpu)
    q = torch.from_numpy(clustered(nq, d, 30, n + d + 1) + 0.01).cuda(gpu)
    r = R.int4_encode_device(x, 64)
    dist = _np(r.distances_device(q, metric))
    ids, got, count = r.search_batch_device(q, k, metric)
    m = min(k, n)
    assert count.tolist() == [m] * nq
    order = np.argsort(dist, axis=1, kind="stable")[:, :m]  # by distance, equal ones by row
    assert np.array_equal(ids[:, :m].cpu().numpy(), order)
    assert np.array_equal(_np(got)[:, :m], np.take_along_axis(dist, order, 1))
    assert (ids[:, m:] == -1).all() and torch.isinf(got[:, m:]).all()


def _check_search(r, q, k, metric):
    d = r.distances_device(q, metric)
    ids, got, count = r.search_batch_device(q, k, metric)
    order = torch.argsort(d, dim=1, stable=True)[:, :k]  # NaN last, equal ones by row
    assert torch.equal(ids, order)
    assert np.array_equal(_np(got), _np(torch.gather(d, 1, order)), equal_nan=True)
    assert count.tolist() == [k] * q.shape[0]


@pytest.mark.parametrize("n,nq,k,metric", [(300_007, 128, 10, "l2"), (1_000_001, 36, 1, "cosine"), (600_000, 64, 100, "dot"), (9_000_000, 4, 33, "l2"),
                                           (300_000, 130, 1024, "l2")])
def test_search_by_sample(gpu, n, nq, k, metric):
    """So many distances that the answer comes from a sampled bound and a collection (k = 1024: not sampled)."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(n)
    x = torch.randn((n, 16), generator=gen, device="cuda")
    x = x[torch.argsort(x[:, 0])].contiguous()  # an order that a plain prefix would be misled by
    _check_search(R.int4_encode_device(x, 32), torch.randn((nq, 16), generator=gen, device="cuda"), k, metric)


@pytest.mark.parametrize("k", [10, 1024])
def test_search_in_rounds(gpu, k):
    """More distances than a search holds at a time: the answers of all queries are those of a part of them at a time."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(k)
    n, nq = 3_000_000, 402
    r = R.int4_encode_device(torch.randn((n, 16), generator=gen, device="cuda"), 32)
    q = torch.randn((nq, 16), generator=gen, device="cuda")
    ids, dist, count = r.search_batch_device(q, k, "l2")
    for at in range(0, nq, 67):
        part = r.search_batch_device(q[at:at + 67], k, "l2")
        assert all(torch.equal(w[at:at + 67], p) for w, p in zip((ids, dist, count), part))
    _check_search(r, q[-6:], k, "l2")


@pytest.mark.parametrize("n,nq,k", [(10_000_000, 10, 8), (4_000_000, 9, 1), (9_000_000, 6, 7), (2_000_000, 40, 100)])
def test_search_by_small_sample(gpu, n, nq, k):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(nq)
    x = torch.randn((n, 16), generator=gen, device="cuda")
    _check_search(R.int4_encode_device(x, 32), torch.randn((nq, 16), generator=gen, device="cuda"), k, "l2")


def test_search_by_sample_overflow_ties_nan(gpu):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    n = 300_000
    few = torch.randn((40, 16), generator=gen, device="cuda")
    x = few[torch.randint(0, 40, (n,), generator=gen, device="cuda")].contiguous()  # 7500 rows each: the bound's ties alone fill the collection
    q = torch.randn((120, 16), generator=gen, device="cuda")
    q[5] = float("nan")   # every row ties
    q[6] = 0.0
    _check_search(R.int4_encode_device(x, 32), q, 50, "l2")
    _check_search(R.int4_encode_device(x, 32), q, 50, "dot")
    x = torch.randn((n, 16), generator=gen, device="cuda")
    x[torch.rand((n,), generator=gen, device="cuda") < 0.9999] = float("nan")  # about 30 rows with a distance, 100 asked for
    _check_search(R.int4_encode_device(x, 32), q, 100, "l2")


def test_search_ties_nan_and_host_forms(gpu):
    x = np.tile(clustered(50, 40, 5, 1), (400, 1))  # 20 000 rows, every one 400 times
    x[11::50] = np.nan
    r = R.int4_encode_device(torch.from_numpy(x).cuda(gpu), 32)
    q = x[3:4] + np.float32(0.01)
    ids, dist, count = r.search_batch(q, 500, "l2")
    assert ids.dtype == np.uint64 and count[0] == 500
    assert ids[0, :400].tolist() == list(range(3, 20000, 50))  # equal distances in row order, across chunks
    assert np.array_equal(np.unique(dist[0, :400]).size, 1)
    assert r.search(q[0], 2) == [(3, float(dist[0, 0])), (53, float(dist[0, 0]))]
    few = R.int4_encode_device(torch.from_numpy(x[:60]).cuda(gpu), 32)
    ids, dist, _ = few.search_batch(q, 60, "cosine")
    assert ids[0, -1] == 11 and np.isnan(dist[0, -1])  # NaN rows come last
    assert np.isfinite(dist[0, :-1]).all()
    nan_q = np.full((1, 40), np.nan, dtype=np.float32)
    ids, dist, _ = r.search_batch(nan_q, 5)
    assert ids[0].tolist() == [0, 1, 2, 3, 4] and np.isnan(dist).all()


def test_empty_inputs(gpu):
    dev = torch.device("cuda", gpu)
    r = R.int4_encode_device(torch.zeros((0, 24), device=dev), 32)
    q = torch.ones((3, 24), device=dev)
    assert r.distances_device(q).shape == (3, 0) and r.decode_device().shape == (0, 24)
    ids, dist, count = r.search_batch_device(q, 4)
    assert (ids == -1).all() and torch.isinf(dist).all() and count.tolist() == [0, 0, 0]
    one = R.int4_encode_device(torch.ones((1, 24), device=dev), 32)
    assert one.distances_device(q[:0]).shape == (0, 1)
    assert one.search_batch_device(q[:0], 4)[0].shape == (0, 4)
    none = torch.zeros((0,), dtype=torch.int64, device=dev)
    assert one.lookup_device(none).shape == (0, 24)
    assert not one.lookup_device(torch.tensor([[-1, 1]], device=dev)).any()
    table = torch.ones((0, 24), device=dev)
    assert R.rows_lookup_device(table, none).shape == (0, 24)
    assert not R.rows_lookup_device(table, torch.tensor([0, 5], device=dev)).any()
    assert not R.rows_grad_device(torch.ones((0, 24), device=dev), none, 6).any()
    assert R.rows_grad_device(torch.ones((2, 24), device=dev), torch.tensor([0, 1], device=dev), 0).shape == (0, 24)
    with pytest.raises(_ffi.CuddleError):
        r.search_batch_device(q, 0)
    with pytest.raises(_ffi.CuddleError):
        r.search_batch_device(q, 1025)
    with pytest.raises(ValueError):
        r.search_batch_device(q[:, :5], 1)


# ---- lookup -----------------------------------------------------------------------------------------------------
def _ids(n, shape, seed, dtype, gpu):
    rng = np.random.default_rng(seed)
    ids = rng.integers(0, max(n, 1), shape)
    ids[rng.random(shape) < 0.1] = -1
    ids.reshape(-1)[-1] = n  # one past the end: no row either
    return torch.from_numpy(ids).to(dtype).cuda(gpu)


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
@pytest.mark.parametrize("n,d,shape", [(1, 1, (1,)), (10, 7, (3, 5)), (100, 64, (257,)), (33, 960, (9,)), (1000, 130, (2, 2, 30)), (5, 2056, (3,))])
def test_rows_lookup(gpu, n, d, shape, idt, dtype):
    table = _rows(n, d, n + d, dtype)
    ids = _ids(n, shape, n + d, idt, gpu)
    for scale in (1.0, 27.5, -0.3):
        got = R.rows_lookup_device(table, ids, scale)
        ok = ((ids >= 0) & (ids < n))[..., None].cpu()
        at = torch.where(ok[..., 0], ids.cpu().long(), 0)
        want = torch.where(ok, table.cpu()[at].float() * torch.tensor(scale, dtype=F32), torch.zeros(())).to(dtype)
        assert torch.equal(got.cpu(), want)
    wide = torch.zeros((n, d + 3), dtype=dtype, device=table.device)
    wide[:, 1:d + 1] = table
    assert torch.equal(R.rows_lookup_device(wide[:, 1:d + 1], ids, 1.0), R.rows_lookup_device(table, ids, 1.0))


@pytest.mark.parametrize("out", [F32, F16, BF16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("d", [1, 64, 130, 960])
def test_int4_lookup(gpu, d, group, out):
    x = _rows(70, d, d)
    r = R.int4_encode_device(x, group)
    values = ref.encode(_np(x), group)[2]
    ids = _ids(70, (4, 25), d, torch.int64, gpu)
    got = r.lookup_device(ids, 2.5, out)
    exact = ref.lookup(values, ids.cpu().numpy(), 2.5)
    # 12 bits times a 2-bit scale: the product is exact in f32, one rounding to the output's type
    assert torch.equal(got.cpu(), torch.from_numpy(exact).to(F32).to(out))


# ---- gradient ---------------------------------------------------------------------------------------------------
def _check_grad(got, g, ids, n, scale, out, prev=None):
    want, mag, cnt = ref.grad(_np(g), ids.cpu().numpy(), n, scale)
    eps = torch.finfo(out).eps
    # an f32 sum of m terms in any order: at most m - 1 roundings of partial sums no larger than the sum of magnitudes,
    # then the product with scale (f32) and one rounding to the type; f16 also has a smallest step of 2^-24
    tol = (cnt[:, None] + 1) * 2.0 ** -24 * mag * 1.001 + eps / 2 * (np.abs(want) + (0 if prev is None else np.abs(prev))) * 1.001 + 2.0 ** -149
    if out == F16:
        tol += 2.0 ** -25
    if prev is not None:
        want = want + prev
        tol += 2.0 ** -24 * np.abs(want)
    err = np.abs(_np(got) - want)
    assert np.all(err <= tol), float((err / tol).max())


@pytest.mark.parametrize("dtype,out", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F32, BF16), (F16, BF16)])
@pytest.mark.parametrize("n,d,t", [(1, 1, 1), (1, 64, 300), (10, 33, 5), (50, 128, 2048), (300, 130, 2049), (70_000, 16, 5000), (3, 960, 700), (257, 8, 10_000), (40, 24, 3840), (40, 24, 8192), (40, 24, 8193), (40, 24, 16_384), (40, 24, 16_385), (100_000, 8, 16_383),
                                   (900_000, 8, 66_000), (3_000_000, 4, 30_000), (1_000, 8, 70_000),
                                   (1_200_000, 4, 140_000), (2, 520, 200_000)])
def test_rows_grad(gpu, n, d, t, dtype, out):
    rng = np.random.default_rng(n + d + t)
    g = torch.from_numpy(rng.standard_normal((t, d)).astype(np.float32)).to(dtype).cuda(gpu)
    ids = _ids(n, (t,), n + t, torch.int64, gpu)
    got = R.rows_grad_device(g, ids, n, 0.75, out)
    assert got.dtype == out
    _check_grad(got, g, ids, n, 0.75, out)
    again = R.rows_grad_device(g, ids.int(), n, 0.75, out)
    assert torch.equal(got, again)  # the same bits, run after run
    base = torch.from_numpy(rng.standard_normal((n, d)).astype(np.float32)).to(out).cuda(gpu)
    acc = base.clone()
    assert R.rows_grad_device(g, ids, n, 0.75, out=acc) is acc
    _check_grad(acc, g, ids, n, 0.75, out, _np(base))
    named = torch.zeros(n, dtype=torch.bool)
    keep = ids.cpu()[(ids.cpu() >= 0) & (ids.cpu() < n)]
    named[keep] = True
    assert torch.equal(acc.cpu()[~named], base.cpu()[~named])
    assert not got.cpu()[~named].any()


def test_rows_grad_skewed_and_strided(gpu):
    """One id takes half of the places (its run spans many blocks), gradients are a strided view."""
    rng = np.random.default_rng(4)
    t, n, d = 40_000, 500, 72
    wide = torch.from_numpy(rng.standard_normal((t, d + 9)).astype(np.float32)).cuda(gpu)
    ids = rng.integers(0, n, t)
    ids[rng.random(t) < 0.5] = 123
    ids[5:900] = -1
    ids = torch.from_numpy(ids).cuda(gpu)
    got = R.rows_grad_device(wide[:, 4:4 + d], ids, n, 1.0)
    _check_grad(got, wide[:, 4:4 + d], ids, n, 1.0, F32)
    assert not R.rows_grad_device(wide[:, :d], torch.full_like(ids, -7), n).any()
    same = R.rows_grad_device(wide[:, :d], torch.zeros_like(ids), n)
    _check_grad(same, wide[:, :d], torch.zeros_like(ids), n, 1.0, F32)


def test_rows_grad_broadcast_and_shapes(gpu):
    """One gradient row handed to every place (an expanded tensor), ids of two dimensions, a transposed gradient."""
    dev = torch.device("cuda", gpu)
    ids = torch.tensor([[3, 1, 3], [-1, 0, 3]], device=dev)
    one = torch.arange(8, device=dev, dtype=F32)
    want = torch.zeros((5, 8), device=dev)
    want[3], want[1], want[0] = 3 * one, one, one
    assert torch.equal(R.rows_grad_device(one.expand(2, 3, 8), ids, 5), want)
    g = torch.randn((8, 6), device=dev)
    got = R.rows_grad_device(g.t(), ids.reshape(-1), 5)
    _check_grad(got, g.t(), ids.reshape(-1), 5, 1.0, F32)
    with pytest.raises(ValueError):
        R.rows_grad_device(one.expand(2, 2, 8), ids, 5)
    with pytest.raises(ValueError):
        R.rows_grad_device(one.expand(2, 3, 8), ids, 5, out=torch.zeros((5, 9), device=dev))
    with pytest.raises(ValueError):
        R.rows_grad_device(one.expand(2, 3, 8), ids.float(), 5)


def test_gradient_against_differences(gpu):
    """The lookup is linear in the table, so <w, L(T + E) - L(T)> = <grad(w), E> up to rounding, for any E: with T, E and w
    small whole numbers every quantity is exact."""
    rng = np.random.default_rng(9)
    n, d, t = 40, 24, 300
    dev = torch.device("cuda", gpu)
    table = torch.from_numpy(rng.integers(-50, 50, (n, d)).astype(np.float32)).to(dev)
    step = torch.from_numpy(rng.integers(-3, 4, (n, d)).astype(np.float32)).to(dev)
    w = torch.from_numpy(rng.integers(-9, 10, (t, d)).astype(np.float32)).to(dev)
    ids = _ids(n, (t,), 1, torch.int32, gpu)
    diff = (w.double() * (R.rows_lookup_device(table + step, ids, 4.0) - R.rows_lookup_device(table, ids, 4.0)).double()).sum()
    grad = R.rows_grad_device(w, ids, n, 4.0)
    assert float(diff) == float((grad.double() * step.double()).sum())


# ---- together, streams, graphs ------------------------------------------------------------------------------------
def test_run_together(gpu):
    """A collection trained, encoded, searched and read back: one step on the rows that a batch named moves them towards
    the batch's targets, the table is encoded, and each target's nearest row is the one that was moved."""
    rng = np.random.default_rng(7)
    n, d, t = 2000, 96, 64
    dev = torch.device("cuda", gpu)
    table = torch.from_numpy(rng.standard_normal((n, d)).astype(np.float32)).to(dev)
    ids = torch.from_numpy(rng.choice(n, t, replace=False)).to(dev)
    target = torch.from_numpy(rng.standard_normal((t, d)).astype(np.float32)).to(dev)
    out = R.rows_lookup_device(table, ids)
    grad = R.rows_grad_device(out - target, ids, n)  # of half the squared error
    table = table - grad
    moved = R.rows_lookup_device(table, ids)
    assert float((moved - target).abs().max()) < 1e-5  # a - (a - b): two roundings of values below 8
    r = R.int4_encode_device(table, 32)
    nearest = r.search_batch_device(target, 1)[0][:, 0]
    assert torch.equal(nearest, ids)
    back = r.lookup_device(nearest)
    s = r.group_scales.float()[ids].repeat_interleave(32, dim=1)
    assert bool(((back - moved).abs() <= s * 0.54).all())  # half a step, and the scale's rounding at the largest value


def test_other_stream_and_graph(gpu):
    dev = torch.device("cuda", gpu)
    x, q = _rows(3000, 100, 1), _rows(5, 100, 2)
    g = _rows(700, 100, 3)
    ids = _ids(3000, (700,), 4, torch.int64, gpu)
    r = R.int4_encode_device(x, 64)

    def step(stream=None):
        d = r.distances_device(q, "l2", stream=stream)
        s = r.search_batch_device(q, 12, "cosine", stream=stream)
        v = r.lookup_device(ids, 0.5, BF16, stream=stream)
        gr = R.rows_grad_device(g, ids, 3000, 2.0, stream=stream)
        e = R.int4_encode_device(x, 32, stream=stream)
        return [d, *s, v, gr, e.decode_device(stream=stream), R.rows_lookup_device(x, ids, 3.0, stream=stream)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    got = step(side)
    torch.cuda.current_stream(dev).wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        q.add_(0.25)  # new inputs in place
        g.mul_(-1.5)
        ids.copy_(torch.roll(ids, 3))
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(held, eager)), turn


def test_graph_of_large_calls(gpu):
    """The sampled search (with and without an overflow of its collection) and the sort over many tiles, replayed."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    n, t = 300_000, 70_000
    x = torch.randn((n, 16), generator=gen, device="cuda")
    r = R.int4_encode_device(x, 32)
    q = torch.randn((128, 16), generator=gen, device="cuda")
    g = torch.randn((t, 24), generator=gen, device="cuda")
    ids = torch.randint(-5, 900, (t,), generator=gen, device="cuda")

    def step():
        return [*r.search_batch_device(q, 10), R.rows_grad_device(g, ids, n)]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for turn in range(4):
        q.mul_(1.25)
        g.mul_(-1.5)
        ids.copy_(torch.roll(ids, 3))
        if turn == 2:
            r.encode_device(x[:1].expand(n, 16).contiguous())  # every row the same: the collections overflow
        if turn == 3:
            r.encode_device(x)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, step())), turn
        if turn == 2:
            assert torch.equal(held[0], torch.arange(10, device="cuda").expand(128, 10))


def test_two_host_threads(gpu):
    import threading

    x = _rows(5000, 64, 1)
    r = R.int4_encode_device(x, 64)
    qs = [_rows(3, 64, 10 + i) for i in range(4)]
    want = [[t.clone() for t in r.search_batch_device(q, 20)] for q in qs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        s = torch.cuda.Stream()
        for _ in range(20):
            got = r.search_batch_device(qs[i], 20, stream=s)
            s.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_beyond_32_bits(gpu):
    """A table of more than 2^32 elements and codes of more than 2^31 bytes: the last rows are found and fetched."""
    dev = torch.device("cuda", gpu)
    n, d = 4_400_000, 1024
    r = R.Int4Rows.empty(n, d, 128, dev)
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    part = torch.randn((100_000, d), generator=gen, device=dev)
    for a in range(0, n, 100_000):
        r.encode_device(part.roll(a // 100_000, dims=1), first_row=a)
    last = part.roll(43, dims=1)[-3:]
    r.encode_device(last * 1.5, first_row=n - 3)
    ids, dist, _ = r.search_batch_device(last * 1.5, 1)
    assert ids[:, 0].tolist() == [n - 3, n - 2, n - 1]
    small = R.int4_encode_device(last * 1.5, 128)
    assert torch.equal(r.lookup_device(torch.arange(n - 3, n, device=dev)), small.decode_device())
    del r, part
    table = torch.zeros((n, d), dtype=BF16, device=dev)
    table[-2:] = 3.0
    at = torch.tensor([n - 1, n - 2, 0], device=dev)
    assert R.rows_lookup_device(table, at, 2.0).float().mean(1).tolist() == [6.0, 6.0, 0.0]
    grad = R.rows_grad_device(torch.ones((3, d), dtype=BF16, device=dev), at, n, 1.0, out=table)
    assert grad[-1].float().tolist() == [4.0] * d and grad[-3].float().tolist() == [0.0] * d and grad[0].float().tolist() == [1.0] * d
