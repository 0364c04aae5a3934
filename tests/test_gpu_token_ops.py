"""The operators on token ids on the GPU, through the C ABI, against plain statements in 64 bits (tests/token_ops_ref.py).

Tolerances, from arithmetic.  With u = 2^-24 (half a step of 32 bits) and h = half a step of the stored type (2^-24 / 2^-11 /
2^-8), s the spacing of the type's subnormal numbers:
  lookup     one product in 32 bits, one rounding:          |x| (u + h) (1 + 2u) + s / 2 + 2^-149
  gradient   m terms, any order, then scale and the old value: m + 2 roundings of partial results none of which is larger than
             A = |old| + scale * sum |g|:                   (m + 2) u A (1 + (m + 2) u) + h |x| + s / 2 + 2^-149
Whole numbers are equal."""
import numpy as np
import pytest

from tests import corpus, token_ops_ref as ref
from tests.test_token_ops_host import random_cache
from tokenizer_amd import capi

pytestmark = pytest.mark.gpu

F32, F16, BF16 = capi.L3_F32, capi.L3_F16, capi.L3_BF16
HALF = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
STEP0 = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}
U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    c = capi.Context(device=0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def _t(torch, code):
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[code]


def _matrix(torch, values, code, stride, shift=0, fill=0.0):
    """float64 (n, d) -> (what the GPU holds as float64, the buffer, pointer of the first element); `shift` elements off an aligned address"""
    n, d = values.shape
    buf = torch.full((shift + n * stride + 8,), fill, dtype=_t(torch, code), device="cuda")
    view = buf[shift:shift + n * stride].view(n, stride)[:, :d]
    view.copy_(torch.from_numpy(values).cuda())
    return view.double().cpu().numpy(), buf, buf.data_ptr() + shift * buf.element_size(), view


def _ids(rng, n, rows):
    ids = rng.integers(0, rows, n)
    odd = rng.random(n) < 0.15
    ids[odd] = rng.choice([-1, rows, -2 ** 31, 2 ** 31 - 1], int(odd.sum()))
    return ids.astype(np.int32)


# ---- lookup -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 517])
@pytest.mark.parametrize("dim", [1, 7, 8, 9, 64, 511, 513, 1001, 2048])
def test_embed_sizes(ctx, torch, n, dim):
    rng = np.random.default_rng(n * 10007 + dim)
    types = [F32, F16, BF16]
    T, O = types[(n + dim) % 3], types[(n * 3 + dim // 2) % 3]
    _embed_case(ctx, torch, rng, n, dim, T, O, rows=37, stride=dim, out_stride=dim, shift=0, scale=1.0)


@pytest.mark.parametrize("T", [F32, F16, BF16])
@pytest.mark.parametrize("O", [F32, F16, BF16])
def test_embed_types_strides_alignment(ctx, torch, T, O):
    rng = np.random.default_rng(T * 3 + O)
    for shift, stride, out_stride, dim in ((0, 72, 80, 64), (1, 65, 67, 64), (3, 100, 99, 33), (5, 1, 1, 1), (2, 4100, 4101, 4099)):
        _embed_case(ctx, torch, rng, 130, dim, T, O, 50, stride, out_stride, shift, scale=45.25)


def _embed_case(ctx, torch, rng, n, dim, T, O, rows, stride, out_stride, shift, scale):
    held, _keep, ptr, _ = _matrix(torch, rng.standard_normal((rows, dim)), T, stride, shift, fill=float("nan"))
    ids = _ids(rng, n, rows)
    d_ids = torch.from_numpy(ids).cuda()
    out = torch.full((shift + (n + 1) * out_stride + 8,), -7.0, dtype=_t(torch, O), device="cuda")
    ctx.embed(d_ids.data_ptr(), n, ptr, T, rows, dim, stride, out.data_ptr() + shift * out.element_size(), O, out_stride, scale)
    got = out.double().cpu().numpy()
    assert (got[:shift] == -7).all() and (got[shift + (n - 1) * out_stride + dim:] == -7).all()
    got = got[shift:shift + n * out_stride].reshape(n, out_stride)
    assert (got[:, dim:] == -7).all()                       # what lies between the rows stays
    want = ref.embed(ids, held, scale)
    tol = np.abs(want) * (U + HALF[O]) * (1 + 2 * U) + STEP0[O] / 2 + 2.0 ** -149
    assert (np.abs(got[:, :dim] - want) <= tol).all()


def test_embed_values_at_the_ends_of_the_types(ctx, torch):
    """Subnormal numbers, the largest ones, infinities and NaN pass through as the type's own conversion has them."""
    v = torch.tensor([0.0, -0.0, 1e-45, 1e-40, 2.0 ** -126, 6e-8, 3e-8, 65504.0, 65520.0, 3.4e38, float("inf"), float("-inf"), float("nan"),
                      1.00390625, 1.01171875, -1.00390625], dtype=torch.float32)
    for T in (F32, F16, BF16):
        table = v.to(_t(torch, T)).cuda().reshape(1, -1)
        for O in (F32, F16, BF16):
            for scale in (1.0, 0.5, 0.0, 3.0):
                out = torch.full((2, v.numel()), -7.0, dtype=_t(torch, O), device="cuda")
                ids = torch.tensor([0, -1], dtype=torch.int32, device="cuda")
                ctx.embed(ids.data_ptr(), 2, table.data_ptr(), T, 1, v.numel(), v.numel(), out.data_ptr(), O, v.numel(), scale)
                want = (table.cpu().float() * scale).to(_t(torch, O))      # both steps are correctly rounded
                assert torch.equal(out[0].cpu().nan_to_num(nan=12345.0), want[0].nan_to_num(nan=12345.0))
                assert torch.equal(torch.isnan(out[0].cpu()), torch.isnan(want[0]))
                assert (out[1] == 0).all()


@pytest.mark.parametrize("count", [0, 1, 99, 100, 101, 2 ** 40])
def test_embed_counts_on_the_device(ctx, torch, count):
    ids = torch.arange(100, dtype=torch.int32, device="cuda") % 7
    table = torch.randn(7, 40, device="cuda")
    out = torch.full((101, 40), -7.0, device="cuda")
    n_dev = torch.tensor([count], dtype=torch.int64, device="cuda")
    ctx.embed(ids.data_ptr(), 100, table.data_ptr(), F32, 7, 40, 40, out.data_ptr(), F32, 40, 1.0, n_dev.data_ptr())
    k = min(count, 100)
    assert torch.equal(out[:k], table[ids.long()][:k]) and (out[k:] == -7).all()


def test_embed_offsets_beyond_32_bits(ctx, torch):
    """Element offsets pass 2^32 in the table and in the output (rows far apart)."""
    rows, dim, stride = 3, 16, (1 << 30) + 8
    table = torch.zeros(2 * stride + dim + (1 << 30) * 2, dtype=torch.float16, device="cuda")     # 8 GiB
    assert 2 * stride * 2 > 2 ** 32
    for r in range(rows):
        table[r * stride:r * stride + dim] = r + 1
    ids = torch.tensor([2, 0, 1], dtype=torch.int32, device="cuda")
    out = torch.full((2 * stride + dim + 8,), -7.0, dtype=torch.float16, device="cuda")
    ctx.embed(ids.data_ptr(), 3, table.data_ptr(), F16, rows, dim, stride, out.data_ptr(), F16, stride, 1.0)
    for t, want in enumerate((3, 1, 2)):
        assert (out[t * stride:t * stride + dim] == want).all()
    assert (out[dim:dim + 64] == -7).all() and (out[stride - 64:stride] == -7).all()


@pytest.mark.parametrize("n, dim, T, O", [(2100, 4096, BF16, BF16), (4097, 1024, F32, F32), (2500, 4001, F16, F32), (33000, 4096, F16, BF16)])
def test_embed_outputs_that_pass_the_caches(ctx, torch, n, dim, T, O):
    """Large outputs take other kernels; the rows and types of the whole output against torch's own conversion."""
    rows = 70
    table = torch.randn(rows, dim, device="cuda").to(_t(torch, T))
    ids = torch.randint(-1, rows + 1, (n,), device="cuda", dtype=torch.int32)
    out = torch.full((n + 1, dim), -7.0, dtype=_t(torch, O), device="cuda")
    ctx.embed(ids.data_ptr(), n, table.data_ptr(), T, rows, dim, dim, out.data_ptr(), O, dim, 0.5)
    there = ((ids >= 0) & (ids < rows))[:, None]
    want = torch.where(there, table[ids.clamp(0, rows - 1).long()].float() * 0.5, torch.zeros(1, device="cuda")).to(_t(torch, O))
    assert torch.equal(out[:n], want) and (out[n] == -7).all()


# ---- gradient -----------------------------------------------------------------------------------------------------
def _grad_case(ctx, torch, rng, ids, dim, G, T, rows, accumulate, scale=1.0, grad_stride=None, table_stride=None, shift=0, n_dev=None, whole=False):
    n = len(ids)
    grad_stride, table_stride = grad_stride or dim, table_stride or dim
    values = rng.integers(-8, 9, (n, dim)).astype(np.float64) if whole else rng.standard_normal((n, dim))
    g, _k1, gp, _ = _matrix(torch, values, G, grad_stride, shift, fill=float("nan"))
    old = rng.integers(-8, 9, (rows, dim)).astype(np.float64) if whole else rng.standard_normal((rows, dim))
    was, buf, tp, view = _matrix(torch, old, T, table_stride, shift, fill=-7.0)
    d_ids = torch.from_numpy(np.asarray(ids, dtype=np.int32)).cuda()
    need = capi.embed_grad_workspace(n, dim)
    work = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    count = torch.tensor([n if n_dev is None else n_dev], dtype=torch.int64, device="cuda")
    ctx.embed_grad(d_ids.data_ptr(), n, gp, G, grad_stride, rows, dim, tp, T, table_stride, work.data_ptr(), need, scale, accumulate,
                   None if n_dev is None else count.data_ptr())
    got = view.double().cpu().numpy()
    used = np.asarray(ids)[:n if n_dev is None else min(n, n_dev)]
    want, size, terms = ref.embed_grad(used, g[:len(used)], rows, scale, was if accumulate else None)
    u = (terms[:, None] + 2) * U
    tol = u * size * (1 + u) + HALF[T] * np.abs(want) + STEP0[T] / 2 + 2.0 ** -149
    tol[terms == 0] = 0.0
    if whole:
        tol[:] = HALF[T] * np.abs(want)                     # whole numbers below 2^24 add up without rounding
    assert (np.abs(got - want) <= tol).all()
    full = buf.double().cpu().numpy()
    assert (full[:shift] == -7).all() and (full[shift + rows * table_stride:] == -7).all()
    if table_stride > dim:
        assert (full[shift:shift + rows * table_stride].reshape(rows, table_stride)[:, dim:] == -7).all()
    assert (work[need:] == 0xAB).all()
    return view.clone()


@pytest.mark.parametrize("n", [1, 2, 7, 8, 9, 64, 300, 1025, 4095, 4096, 4097, 9000])
@pytest.mark.parametrize("accumulate", [False, True])
def test_grad_lengths(ctx, torch, n, accumulate):
    rng = np.random.default_rng(n)
    _grad_case(ctx, torch, rng, _ids(rng, n, 200), 24, BF16, F32, 200, accumulate)


@pytest.mark.parametrize("dim", [1, 3, 8, 65, 129, 1001, 2048, 2056, 4104])
def test_grad_widths(ctx, torch, dim):
    rng = np.random.default_rng(dim)
    for accumulate in (False, True):
        _grad_case(ctx, torch, rng, _ids(rng, 333, 60), dim, F16, F32, 60, accumulate, scale=0.5)


@pytest.mark.parametrize("G", [F32, F16, BF16])
@pytest.mark.parametrize("T", [F32, F16, BF16])
def test_grad_types_strides_alignment(ctx, torch, G, T):
    rng = np.random.default_rng(G * 3 + T)
    for accumulate in (False, True):
        for shift, gs, ts, dim in ((0, 72, 80, 64), (1, 65, 67, 64), (3, 1003, 1001, 999)):
            _grad_case(ctx, torch, rng, _ids(rng, 700, 90), dim, G, T, 90, accumulate, 45.25, gs, ts, shift)


@pytest.mark.parametrize("rows", [1, 2, 255, 511, 512, 513, 128256, 262143, 262144, 262145])
@pytest.mark.parametrize("n", [5000, 9000])
def test_grad_numbers_of_digits(ctx, torch, rows, n):
    """Keys of one to three digits; the first and last rows among them."""
    rng = np.random.default_rng(rows)
    ids = _ids(rng, n, rows)
    ids[:4] = [0, rows - 1, 0, rows - 1]
    _grad_case(ctx, torch, rng, ids, 8, F32, F32, rows, False)
    _grad_case(ctx, torch, rng, ids, 8, F32, F32, rows, True)


@pytest.mark.parametrize("n", [511, 512, 513, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 65536, 65537, 262144, 262145, 300001])
def test_grad_where_the_sort_changes(ctx, torch, n):
    """Every way of bringing equal ids together, next to the sizes at which another begins."""
    rng = np.random.default_rng(n)
    _grad_case(ctx, torch, rng, _ids(rng, n, 3000), 16, BF16, F32, 3000, True, n_dev=n - 5)


@pytest.mark.parametrize("n, rows", [(3000, 11999), (3000, 12000), (8500, 33999), (8500, 34000)])
@pytest.mark.parametrize("dim, T", [(1, F16), (1, F32), (5, F16), (7, BF16), (8, F16), (9, F32), (40, BF16)])
def test_grad_whole_names_few_rows(ctx, torch, n, rows, dim, T):
    """Most rows are zeros; rows of two bytes and more, on any alignment."""
    rng = np.random.default_rng(n + dim)
    _grad_case(ctx, torch, rng, _ids(rng, n, rows), dim, BF16, T, rows, False, 0.5, dim + 2, dim + 3, 1)


@pytest.mark.parametrize("n", [300, 5000, 9000])
def test_grad_of_the_most_rows(ctx, torch, n):
    """2^28 rows: keys of four digits."""
    rows = 2 ** 28
    table = torch.ones(rows, dtype=torch.float16, device="cuda")
    ids = torch.randint(0, rows, (n,), dtype=torch.int32, device="cuda")
    ids[:3] = torch.tensor([0, rows - 1, rows - 1], dtype=torch.int32)
    g = torch.randint(-4, 5, (n, 1), device="cuda").half()
    need = capi.embed_grad_workspace(n, 1)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    want = torch.zeros(rows, device="cuda").index_add_(0, ids.long(), g[:, 0].float())
    for accumulate in (False, True):
        ctx.embed_grad(ids.data_ptr(), n, g.data_ptr(), F16, 1, rows, 1, table.data_ptr(), F16, 1, work.data_ptr(), need, 1.0, accumulate)
        assert torch.equal(table, (want * (2 if accumulate else 1)).half())


@pytest.mark.parametrize("n, dim, G", [(34000, 4001, BF16), (17000, 4097, F32), (33000, 4100, F16)])
def test_grad_larger_than_the_last_cache(ctx, torch, n, dim, G):
    """Gradients that are loaded past the caches; whole numbers, so that torch's own sums are exact."""
    rows = 900
    g = torch.randint(-8, 9, (n, dim), device="cuda").to(_t(torch, G))
    assert g.numel() * g.element_size() > 256 << 20
    ids = torch.randint(-1, rows + 1, (n,), device="cuda", dtype=torch.int32)
    ids[torch.rand(n, device="cuda") < 0.2] = 5
    there = ((ids >= 0) & (ids < rows)).float()[:, None]
    want = torch.zeros(rows, dim, device="cuda").index_add_(0, ids.clamp(0, rows - 1).long(), g.float() * there)
    table = torch.ones(rows, dim, device="cuda")
    need = capi.embed_grad_workspace(n, dim)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    ctx.embed_grad(ids.data_ptr(), n, g.data_ptr(), G, dim, rows, dim, table.data_ptr(), F32, dim, work.data_ptr(), need, 1.0, True)
    assert torch.equal(table, want + 1)
    ctx.embed_grad(ids.data_ptr(), n, g.data_ptr(), G, dim, rows, dim, table.data_ptr(), F32, dim, work.data_ptr(), need, 1.0, False)
    assert torch.equal(table, want)


@pytest.mark.parametrize("n, dim", [(2048, 520), (600, 4096), (257, 8200), (1000, 4090), (3000, 1100), (9000, 1030)])
def test_grad_one_id_in_half_of_the_positions(ctx, torch, n, dim):
    """With and without a sort, over several tiles of columns."""
    rng = np.random.default_rng(dim)
    ids = _ids(rng, n, 50)
    ids[rng.random(n) < 0.5] = 7
    _grad_case(ctx, torch, rng, ids, dim, BF16, F32, 50, True)
    _grad_case(ctx, torch, rng, ids, dim, BF16, BF16, 50, False)


@pytest.mark.parametrize("n", [64, 1000, 8192, 40000])
def test_grad_long_runs(ctx, torch, n):
    """One id throughout, two ids, runs that end on every place of a walker's chunk; whole numbers, so nothing is rounded."""
    rng = np.random.default_rng(n)
    _grad_case(ctx, torch, rng, np.full(n, 3), 40, BF16, F32, 5, True, whole=True)
    _grad_case(ctx, torch, rng, np.arange(n) % 2 + 1, 40, BF16, F32, 5, False, whole=True)
    ids = np.repeat(np.arange(400), np.arange(400) % 131 + 1)[:n]
    rng.shuffle(ids)
    _grad_case(ctx, torch, rng, ids, 40, BF16, F32, 400, False, whole=True)
    _grad_case(ctx, torch, rng, np.full(n, -1), 40, BF16, F32, 5, False, whole=True)      # nobody is named: all rows zero
    _grad_case(ctx, torch, rng, np.full(n, -1), 40, BF16, F32, 5, True, whole=True)


@pytest.mark.parametrize("count", [0, 1, 500, 999, 1000, 2 ** 40])
def test_grad_counts_on_the_device(ctx, torch, count):
    rng = np.random.default_rng(5)
    for accumulate in (False, True):
        _grad_case(ctx, torch, rng, _ids(rng, 1000, 50), 16, F32, F32, 50, accumulate, n_dev=count)


@pytest.mark.parametrize("n", [5, 3000])
def test_grad_offsets_beyond_32_bits(ctx, torch, n):
    """Element offsets pass 2^32 in the gradient and in the table (rows far apart); with and without a sort."""
    dim, rows = 16, 3
    gs, ts = 2 ** 32 // (n - 1) + 3, (1 << 30) + 5
    grad = torch.zeros((n - 1) * gs + dim, dtype=torch.float16, device="cuda")             # 8 GiB
    table = torch.zeros(2 * ts + dim, dtype=torch.float16, device="cuda")                  # 4 GiB
    at = (torch.arange(n, device="cuda")[:, None] * gs + torch.arange(dim, device="cuda")).reshape(-1)
    g = torch.randint(-4, 5, (n, dim), device="cuda").half()
    grad[at] = g.reshape(-1)
    ids = (torch.arange(n, device="cuda") % 3).int()
    need = capi.embed_grad_workspace(n, dim)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    for accumulate in (False, True):
        ctx.embed_grad(ids.data_ptr(), n, grad.data_ptr(), F16, gs, rows, dim, table.data_ptr(), F16, ts, work.data_ptr(), need, 1.0, accumulate)
        for r in range(rows):
            want = g[ids == r].float().sum(0)                                               # whole numbers: exact in 32 bits ...
            want = want.half() if not accumulate else (want.half().float() + want).half()   # ... rounded where they are stored
            assert torch.equal(table[r * ts:r * ts + dim], want)
        assert (table[dim:dim + 64] == 0).all()


def test_grad_without_ids(ctx, torch):
    table = torch.full((50, 33), 5.0, dtype=torch.bfloat16, device="cuda")
    ctx.embed_grad(None, 0, None, F32, 33, 50, 33, table.data_ptr(), BF16, 33, None, 0, 1.0, True)
    assert (table == 5).all()
    ctx.embed_grad(None, 0, None, F32, 33, 50, 33, table.data_ptr(), BF16, 33, None, 0, 1.0, False)
    assert (table == 0).all()


def test_grad_is_the_lookups_gradient(ctx, torch):
    """<G, dW> against differences of <embed(W), dY>, and the same bits from the same ids."""
    rng = np.random.default_rng(11)
    n, rows, dim, scale = 600, 80, 48, 0.5
    ids = _ids(rng, n, rows)
    d_ids = torch.from_numpy(ids).cuda()
    dy = torch.from_numpy(rng.integers(-8, 9, (n, dim))).float().cuda()
    table = torch.from_numpy(rng.integers(-8, 9, (rows, dim))).float().cuda()
    step = torch.from_numpy(rng.integers(-2, 3, (rows, dim))).float().cuda()
    need = capi.embed_grad_workspace(n, dim)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    grad = torch.empty_like(table)
    ctx.embed_grad(d_ids.data_ptr(), n, dy.data_ptr(), F32, dim, rows, dim, grad.data_ptr(), F32, dim, work.data_ptr(), need, scale)

    def loss(w):
        out = torch.empty(n, dim, device="cuda")
        ctx.embed(d_ids.data_ptr(), n, w.data_ptr(), F32, rows, dim, dim, out.data_ptr(), F32, dim, scale)
        return float((out.double() * dy.double()).sum())

    # the lookup is linear and every number here a small multiple of 1/2: the difference is exact
    assert loss(table + step) - loss(table - step) == 2 * float((grad.double() * step.double()).sum())


def test_grad_same_bits(ctx, torch):
    rng = np.random.default_rng(12)
    n, rows, dim = 20000, 300, 264
    d_ids = torch.from_numpy(_ids(rng, n, rows)).cuda()
    dy = torch.randn(n, dim, device="cuda").bfloat16()
    need = capi.embed_grad_workspace(n, dim)
    got = []
    for _ in range(3):
        work = torch.randint(0, 256, (need,), dtype=torch.uint8, device="cuda")
        grad = torch.empty(rows, dim, device="cuda")
        ctx.embed_grad(d_ids.data_ptr(), n, dy.data_ptr(), BF16, dim, rows, dim, grad.data_ptr(), F32, dim, work.data_ptr(), need)
        got.append(grad)
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_grad_batches_of_every_size_on_the_largest_ones_workspace(ctx, torch):
    """One workspace, sized once: the last batches of an epoch are smaller."""
    rng = np.random.default_rng(12)
    rows, dim, most = 700, 2048, 19000
    need = capi.embed_grad_workspace(most, dim)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    dy = torch.from_numpy(rng.integers(-8, 9, (most, dim))).cuda().bfloat16()
    ids = torch.from_numpy(_ids(rng, most, rows)).cuda()
    for n in (most, 18432, 18400, 9217, 9215, 8192, 4600, 2100, 1):
        got = torch.full((rows, dim), -7.0, device="cuda")
        ctx.embed_grad(ids.data_ptr(), n, dy.data_ptr(), BF16, dim, rows, dim, got.data_ptr(), F32, dim, work.data_ptr(), need)
        there = ((ids[:n] >= 0) & (ids[:n] < rows))[:, None]
        want = torch.zeros(rows, dim, device="cuda").index_add_(0, ids[:n].clamp(0, rows - 1).long(), dy[:n].float() * there)
        assert torch.equal(got, want), n                   # (whole numbers below 2^24 add up without rounding)


# ---- paged cache --------------------------------------------------------------------------------------------------
class DeviceCache:
    """A cache's state on the GPU, its calls in place or to other arrays."""

    def __init__(self, torch, state, in_place=True, stride_more=3):
        length, held, table, free, n_free, self.page, self.n_pages, self.max_pages = state
        self.torch, self.n = torch, len(length)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        self.stride = self.max_pages + stride_more
        self.table = torch.full((max(self.n, 1), self.stride), -9, dtype=torch.int32, device="cuda")
        if self.n:
            self.table[:, :self.max_pages] = i32(table)
        self.len, self.held = i32(length), i32(held)
        self.free, self.n_free = i32(free), i32([n_free])
        self.len2, self.held2, self.n_free2 = (self.len, self.held, self.n_free) if in_place else (i32(length) - 99, i32(held) - 99, i32([-99]))
        self.status = torch.full((1,), 77, dtype=torch.int32, device="cuda")
        self.need = capi.cache_workspace(self.n)
        self.work = torch.randint(0, 256, (self.need + 64,), dtype=torch.uint8, device="cuda")
        self.work[self.need:] = 0xAB

    def slots(self, ctx, d_off, slots, pos, cap, stream=None):
        ctx.cache_slots(d_off.data_ptr(), self.n, self.len.data_ptr(), self.held.data_ptr(), self.page, self.n_pages, self.table.data_ptr(),
                        self.stride, self.max_pages, self.free.data_ptr(), self.n_free.data_ptr(), self.len2.data_ptr(), self.held2.data_ptr(),
                        self.n_free2.data_ptr(), slots.data_ptr(), pos.data_ptr(), cap, self.status.data_ptr(), self.work.data_ptr(), self.need,
                        stream)

    def trim(self, ctx, d_keep, stream=None):
        ctx.cache_trim(d_keep.data_ptr(), self.n, self.len.data_ptr(), self.held.data_ptr(), self.page, self.n_pages, self.table.data_ptr(),
                       self.stride, self.max_pages, self.free.data_ptr(), self.n_free.data_ptr(), self.len2.data_ptr(), self.held2.data_ptr(),
                       self.n_free2.data_ptr(), self.status.data_ptr(), self.work.data_ptr(), self.need, stream)

    def state(self):
        assert (self.work[self.need:] == 0xAB).all() and (self.table[:, self.max_pages:] == -9).all()
        return (self.len2.tolist(), self.held2.tolist(), self.table[:self.n, :self.max_pages].tolist(), self.free.tolist(),
                int(self.n_free2[0]))

    def now(self):
        """The state that the last call left is the next call's."""
        self.len, self.held, self.n_free = self.len2, self.held2, self.n_free2


def _cache_round(ctx, torch, rng, n, page, max_pages, n_pages, new, in_place, tight=False, odd=False, more_cap=5):
    import random
    length, held, table, free, n_free = random_cache(random.Random(int(rng.integers(1 << 30))), n, page, max_pages, n_pages)
    if tight:
        n_free = min(n_free, int(sum(new)) // page // 2)
    if odd and n > 2:
        length[1], held[1] = -1, 0
        length[n // 2], held[n // 2] = held[n // 2] * page + 1, held[n // 2]
        free[max(0, n_free - 2)] = n_pages
    off = [0] + np.cumsum(new).tolist()
    cap = off[-1] + more_cap
    state = (length, held, table, free, n_free, page, n_pages, max_pages)
    model, dev = ref.Cache(*state), DeviceCache(torch, state, in_place)
    slots, pos = [-7] * (cap + 1), [-7] * (cap + 1)
    status = model.slots(off, cap, slots, pos)
    d_slots = torch.full((cap + 1,), -7, dtype=torch.int64, device="cuda")
    d_pos = torch.full((cap + 1,), -7, dtype=torch.int32, device="cuda")
    d_off = torch.tensor(off, dtype=torch.int64, device="cuda")
    dev.slots(ctx, d_off, d_slots, d_pos, cap)
    assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free)
    assert d_slots.tolist() == slots and d_pos.tolist() == pos and int(dev.status[0]) == status
    dev.now()
    if not in_place:
        dev.len2, dev.held2, dev.n_free2 = (x.clone() - 50 for x in (dev.len, dev.held, dev.n_free))
    keep = [int(rng.choice([-1, 0, max(0, L), max(0, L - 3), L + 9, max(0, L // 2)])) for L in model.length]
    status = model.trim(keep)
    dev.trim(ctx, torch.tensor(keep, dtype=torch.int32, device="cuda"))
    assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free) and int(dev.status[0]) == status


@pytest.mark.parametrize("n", [1, 2, 63, 64, 255, 256, 257, 1023, 1024, 1025, 2500])
@pytest.mark.parametrize("in_place", [False, True])
def test_cache_requests(ctx, torch, n, in_place):
    rng = np.random.default_rng(n)
    page = [16, 1, 7, 64][n % 4]
    new = rng.choice([0, 1, 1, 5, 40], n)
    _cache_round(ctx, torch, rng, n, page, 12, n * 10 + 20, new, in_place)
    _cache_round(ctx, torch, rng, n, page, 12, n * 10 + 20, new, in_place, tight=True, odd=True, more_cap=0)


@pytest.mark.parametrize("tokens", [0, 1, 255, 256, 257, 1024, 5000, 20000])
def test_cache_one_long_request(ctx, torch, tokens):
    rng = np.random.default_rng(tokens)
    _cache_round(ctx, torch, rng, 1, 16, 1300, 2700, [tokens], True)
    _cache_round(ctx, torch, rng, 3, 16, 1300, 7000, [0, tokens, 0], False)


@pytest.mark.parametrize("n, every", [(1500, 1), (3000, 1), (5000, 7), (70000, 30)])
def test_cache_many_requests_few_tokens(ctx, torch, n, every):
    """More requests than one workgroup plans, most of them without a new token."""
    rng = np.random.default_rng(n)
    new = (np.arange(n) % every == 0).astype(int) * rng.integers(1, 3, n)
    _cache_round(ctx, torch, rng, n, 4, 3, n * 3 + 10, new, True)
    _cache_round(ctx, torch, rng, n, 4, 3, n * 3 + 10, new, False, tight=True, odd=True)


def test_cache_single_tokens_step_after_step(ctx, torch):
    """130 steps of one token each for requests of which some end on the way; pages go round the pool."""
    import random
    rng = random.Random(3)
    n, page, max_pages, n_pages = 70, 8, 24, 600
    state = (*random_cache(rng, n, page, 8, n_pages, full=0.1), page, n_pages, 8)
    state = (state[0], state[1], [r + [-5] * 16 for r in state[2]], state[3], state[4], page, n_pages, max_pages)
    model, dev = ref.Cache(*state), DeviceCache(torch, state)
    d_slots = torch.empty(n, dtype=torch.int64, device="cuda")
    d_pos = torch.empty(n, dtype=torch.int32, device="cuda")
    for step in range(130):
        new = [0 if rng.random() < 0.1 else 1 for _ in range(n)]
        off = [0] + np.cumsum(new).tolist()
        slots, pos = [-7] * n, [-7] * n
        d_slots.fill_(-7)
        d_pos.fill_(-7)
        status = model.slots(off, n, slots, pos)
        dev.slots(ctx, torch.tensor(off, dtype=torch.int64, device="cuda"), d_slots, d_pos, n)
        assert d_slots.tolist() == slots and d_pos.tolist() == pos and int(dev.status[0]) == status
        there = [s for s in slots if s >= 0]
        assert len(set(there)) == len(there)
        keep = [0 if rng.random() < 0.04 else -1 for _ in range(n)]
        status = model.trim(keep)
        dev.trim(ctx, torch.tensor(keep, dtype=torch.int32, device="cuda"))
        assert int(dev.status[0]) == status
        assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free)


def test_cache_offsets_that_cannot_be(ctx, torch):
    """Offsets that descend or end behind cap: those requests keep their state, nothing is written outside the arrays."""
    state = ([5, 0, 3, 0], [1, 0, 1, 0], [[4, -5], [-5, -5], [6, -5], [-5, -5]], list(range(10, 30)) + [-5] * 12, 20, 8, 32, 2)
    for off, cap in (([0, 3, 2, 5, 9], 9), ([0, 2, 4, 6, 100], 8), ([7, 8, 9, 10, 11], 11), ([2 ** 63, 2 ** 63 + 1, 2, 3, 4], 4)):
        dev, model = DeviceCache(torch, state), ref.Cache(*state)
        d_off = torch.from_numpy(np.array(off, np.uint64).view(np.int64)).cuda()
        d_slots = torch.full((cap + 64,), -7, dtype=torch.int64, device="cuda")
        d_pos = torch.full((cap + 64,), -7, dtype=torch.int32, device="cuda")
        dev.slots(ctx, d_off, d_slots, d_pos, cap)
        status = model.slots(off, cap, [-7] * cap, [-7] * cap)
        assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free) and int(dev.status[0]) == status
        assert (d_slots[cap:] == -7).all() and (d_pos[cap:] == -7).all()


# (by one workgroup, by two launches with two tokens a thread, with four)
FIRST_OFFSETS = [(1, 1, 5, 3), (4, 7, 3, 0), (200, 300, 4, 5), (300, 513, 5, 1), (1000, 2049, 2, 0), (5, 5000, 40, 3), (1, 4097, 1, 0), (3, 511, 3000, 0),
                 (2000, 1, 3, 2), (3000, 777, 3, 0), (20000, 1023, 2, 1), (50, (1 << 20) + 13, 30, 7), (2, (1 << 20) - 1023, 2500, 0)]


def _prefilled(torch, cap):
    """Slots and positions that no call writes: (lists, the same on the GPU)"""
    slots, pos = [-1000 - t for t in range(cap)], [-30000000 - t for t in range(cap)]
    return slots, pos, torch.tensor(slots, dtype=torch.int64, device="cuda"), torch.tensor(pos, dtype=torch.int32, device="cuda")


def _holds(torch, buf, values):
    return torch.equal(buf, torch.tensor(values, dtype=buf.dtype, device="cuda"))


@pytest.mark.parametrize("n, first, most, more_cap", FIRST_OFFSETS)
def test_cache_slots_in_front_of_the_first_offset(ctx, torch, n, first, most, more_cap):
    """Offsets that do not begin at 0, as a slice of a larger batch's: what is in front of them is not the call's."""
    import random
    rng = np.random.default_rng(n + first)
    page, max_pages, n_pages = 16, max(4, -(-most // 16) + 2), 3 * n + 400 + n * -(-most // 16)
    state = (*random_cache(random.Random(n), n, page, 2, n_pages, full=0.2), page, n_pages, max_pages)
    state = (state[0], state[1], [r + [-5] * (max_pages - 2) for r in state[2]], *state[3:])
    off = (first + np.append(0, np.cumsum(rng.integers(0, most + 1, n)))).tolist()
    cap = off[-1] + more_cap
    dev, model = DeviceCache(torch, state), ref.Cache(*state)
    slots, pos, d_slots, d_pos = _prefilled(torch, cap)
    status = model.slots(off, cap, slots, pos)
    dev.slots(ctx, torch.tensor(off, dtype=torch.int64, device="cuda"), d_slots, d_pos, cap)
    assert _holds(torch, d_slots, slots) and _holds(torch, d_pos, pos) and int(dev.status[0]) == status
    assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free)


@pytest.mark.parametrize("n, k, most", [(20, 7, 30), (3000, 1200, 5), (40, 11, 60000)])
def test_cache_slots_of_one_batch_in_two_calls(ctx, torch, n, k, most):
    """Two groups of requests, each with a pool of its own, and one array of slots: slices of one batch's offsets, in either order."""
    rng = np.random.default_rng(n)
    page = 16
    off = np.append(0, np.cumsum(rng.integers(0, most + 1, n)))
    cap = int(off[-1])
    d_off = torch.from_numpy(off).cuda()
    for order in ((0, 1), (1, 0)):
        slots, pos, d_slots, d_pos = _prefilled(torch, cap)
        for g in order:
            part = slice(0, k + 1) if g == 0 else slice(k, n + 1)
            m = part.stop - part.start - 1
            most_pages = -(-most // page)
            state = ([0] * m, [0] * m, [[-5] * most_pages] * m, list(range(m * most_pages)), m * most_pages, page, m * most_pages, most_pages)
            dev, model = DeviceCache(torch, state), ref.Cache(*state)
            end = int(off[part.stop - 1])
            assert model.slots(off[part].tolist(), end, slots, pos) == 0
            dev.slots(ctx, d_off[part], d_slots, d_pos, end)
            assert int(dev.status[0]) == 0 and dev.state() == (model.length, model.held, model.table, model.free, model.n_free)
        assert _holds(torch, d_slots, slots) and _holds(torch, d_pos, pos) and min(pos) >= 0


@pytest.mark.parametrize("front", [0, 5000])
def test_cache_slots_where_the_first_offset_is_not_the_smallest(ctx, torch, front):
    """Offsets that descend below the first one: its request is not served, the tokens of those behind it have their slots."""
    state = ([5, 0, 3, 0], [1, 0, 1, 0], [[4, -5], [-5, -5], [6, -5], [-5, -5]], list(range(10, 30)) + [-5] * 12, 20, 8, 32, 2)
    for off in ([5, 2, 4, 4, 6], [9, 1, 1, 3, 4]):
        off = [front + x for x in off]
        cap = off[-1] + 3 if off[0] < off[-1] else off[0]
        dev, model = DeviceCache(torch, state), ref.Cache(*state)
        slots, pos, d_slots, d_pos = _prefilled(torch, cap)
        status = model.slots(off, cap, slots, pos)
        dev.slots(ctx, torch.tensor(off, dtype=torch.int64, device="cuda"), d_slots, d_pos, cap)
        assert status == ref.BAD == int(dev.status[0]) and _holds(torch, d_slots, slots) and _holds(torch, d_pos, pos)
        assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free)


@pytest.mark.parametrize("n_free", [-1, -2 ** 31, 33, 2 ** 31 - 1])
def test_cache_counts_that_cannot_be(ctx, torch, n_free):
    state = ([5, 16], [1, 2], [[4, -5, -5], [6, 7, -5]], list(range(32)), n_free, 8, 32, 3)
    dev, model = DeviceCache(torch, state), ref.Cache(*state)
    off = [0, 1, 2]
    slots, pos = [-7] * 2, [-7] * 2
    d_slots = torch.full((2,), -7, dtype=torch.int64, device="cuda")
    d_pos = torch.full((2,), -7, dtype=torch.int32, device="cuda")
    status = model.slots(off, 2, slots, pos)
    dev.slots(ctx, torch.tensor(off, dtype=torch.int64, device="cuda"), d_slots, d_pos, 2)
    assert int(dev.status[0]) == status == ref.BAD | ref.POOL
    assert d_slots.tolist() == slots and d_pos.tolist() == pos and int(dev.n_free2[0]) == n_free
    status = model.trim([0, 0])
    dev.trim(ctx, torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert int(dev.status[0]) == status and dev.state() == (model.length, model.held, model.table, model.free, model.n_free)


@pytest.mark.parametrize("n", [5, 3000])
def test_cache_trim_leaves_alone_whatever_stands_there(ctx, torch, n):
    """keep < 0: also where length and pages make no sense; nothing is reported, the requests beside it are served."""
    length, held = [(5, -5, 9)[i % 3] for i in range(n)], [(1, -5, 2 ** 31 - 1)[i % 3] for i in range(n)]
    state = (length, held, [[i, -5, -5] for i in range(n)], [-5] * n, 0, 8, n, 3)
    dev, model = DeviceCache(torch, state), ref.Cache(*state)
    keep = [0 if i % 3 == 0 else -1 - i for i in range(n)]
    assert model.trim(keep) == 0
    dev.trim(ctx, torch.tensor(keep, dtype=torch.int32, device="cuda"))
    assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free) and int(dev.status[0]) == 0


@pytest.mark.parametrize("n, every, most", [(20000, 1, 500), (3, 1, 2000000), (2 ** 20, 1, 9), (2 ** 20, 1000, 8500), (16384, 1, 600), (16383, 1, 600)])
def test_cache_of_millions_of_tokens(ctx, torch, n, every, most):
    """Four million tokens and more, of few long requests and of many short ones, some under way, some without a new token."""
    rng = np.random.default_rng(n + every)
    page = 16
    new = np.where(np.arange(n) % every == 0, rng.integers(most // 2, most + 1, n), 0)
    old = np.where(np.arange(n) % 3 == 0, rng.integers(0, 3 * page, n), 0)
    assert new.sum() >= 2 ** 22
    held = -(-old // page)
    need = -(-(old + new) // page) - held
    wide = int((held + need).max())
    n_pages = int(held.sum() + need.sum())
    left = int(need.sum()) - int(need[-1]) if n == 20000 else int(need.sum())      # one page short for the last request
    d = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    off = np.append(0, np.cumsum(new))
    total = int(off[-1])
    table = torch.full((n, wide), -5, dtype=torch.int32, device="cuda")
    first = d(np.cumsum(held) - held, torch.int64)[:, None]
    j = torch.arange(min(wide, 3), device="cuda")
    table[:, :len(j)] = torch.where(j < d(held, torch.int64)[:, None], (first + j).int(), table[:, :len(j)])
    free = torch.arange(int(held.sum()), n_pages, dtype=torch.int32, device="cuda").flip(0).contiguous()[:max(left, 1)].contiguous()
    L, H, N, S = d(old, torch.int32), d(held, torch.int32), d([left], torch.int32), d([77], torch.int32)
    cap = total + 3
    slots, pos = torch.full((cap,), -7, dtype=torch.int64, device="cuda"), torch.full((cap,), -7, dtype=torch.int32, device="cuda")
    room = capi.cache_workspace(n)
    work = torch.empty(room, dtype=torch.uint8, device="cuda")
    d_off = d(off, torch.int64)
    ctx.cache_slots(d_off.data_ptr(), n, L.data_ptr(), H.data_ptr(), page, n_pages, table.data_ptr(), wide, wide, free.data_ptr(), N.data_ptr(), L.data_ptr(),
                    H.data_ptr(), N.data_ptr(), slots.data_ptr(), pos.data_ptr(), cap, S.data_ptr(), work.data_ptr(), room)
    served = np.cumsum(need) <= left
    served |= need == 0
    assert int(S[0]) == (0 if served.all() else ref.POOL) and int(N[0]) == left - int(need[served].sum())
    assert torch.equal(L, d(np.where(served, old + new, old), torch.int32)) and torch.equal(H, d(np.where(served, held + need, held), torch.int32))
    seq = torch.repeat_interleave(torch.arange(n, device="cuda"), d(new, torch.int64))
    t = torch.arange(total, device="cuda")
    ok = d(served, torch.bool)[seq]
    p = d(old, torch.int64)[seq] + t - d_off[seq]
    fresh = p // page - d(held, torch.int64)[seq]
    taken = left - 1 - (d(np.cumsum(need) - need, torch.int64)[seq] + fresh)
    page_of = torch.where(fresh < 0, first[seq, 0] + p // page, free[taken.clamp(0, len(free) - 1)].long())
    assert torch.equal(slots[:total], torch.where(ok, page_of * page + p % page, torch.full_like(p, -1)))
    assert torch.equal(pos[:total], torch.where(ok, p, torch.full_like(p, -1)).int())
    assert (slots[total:] == -7).all() and (pos[total:] == -7).all()
    entry = ok & (p % page == 0) & (fresh >= 0)
    assert torch.equal(table[seq[entry], (p // page)[entry]].long(), page_of[entry])


@pytest.mark.parametrize("n_free", [2 ** 20, 700001, 1024 * 600, 5, 0])
def test_cache_of_the_most_requests(ctx, torch, n_free):
    """2^20 requests of one new token each, on a pool that may run short; then every page back."""
    n, page = 2 ** 20, 16
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    free = torch.arange(n, dtype=torch.int32, device="cuda")
    table, length, held, status = torch.full((n, 1), -5, dtype=torch.int32, device="cuda"), i32(n), i32(n), i32(1)
    left = torch.tensor([n_free], dtype=torch.int32, device="cuda")
    off = torch.arange(n + 1, dtype=torch.int64, device="cuda")
    slots, pos = torch.full((n,), -7, dtype=torch.int64, device="cuda"), torch.full((n,), -7, dtype=torch.int32, device="cuda")
    need = capi.cache_workspace(n)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    p = lambda *a: [x.data_ptr() for x in a]  # noqa: E731
    ctx.cache_slots(off.data_ptr(), n, *p(length, held), page, n, table.data_ptr(), 1, 1, *p(free, left, length, held, left, slots, pos), n, status.data_ptr(),
                    work.data_ptr(), need)
    i = torch.arange(n, device="cuda")
    served = i < n_free
    assert torch.equal(slots, torch.where(served, (n_free - 1 - i) * page, torch.full_like(i, -1)))
    assert torch.equal(pos, torch.where(served, 0, -1).int()) and torch.equal(held, served.int()) and torch.equal(length, served.int())
    assert int(left[0]) == 0 and int(status[0]) == (0 if n_free == n else ref.POOL)
    assert torch.equal(table[:n_free, 0], (n_free - 1 - i[:n_free]).int()) and (table[n_free:] == -5).all()
    ctx.cache_trim(i32(n).data_ptr(), n, *p(length, held), page, n, table.data_ptr(), 1, 1, *p(free, left, length, held, left), status.data_ptr(),
                   work.data_ptr(), need)
    assert int(left[0]) == n_free and int(status[0]) == 0 and not held.any() and not length.any()
    assert torch.equal(free[:n_free], (n_free - 1 - i[:n_free]).int())


def test_cache_slots_beyond_32_bits(ctx, torch):
    """Slots of pages at the end of a pool of 2^42 tokens; one launch and two."""
    page, n_pages = 4096, 2 ** 30
    for n, cap in ((2, 8), (1100, 1100)):
        length, held = [page - 1] + [0] * (n - 1), [1] + [0] * (n - 1)
        table = [[n_pages - 1, -5]] + [[-5, -5]] * (n - 1)
        free = torch.tensor([n_pages - 5, n_pages - 4, n_pages - 3, n_pages - 2], dtype=torch.int32, device="cuda")
        off = [0, 2, 5] + [5] * (n - 2)
        state = (length, held, table, [], 4, page, n_pages, 2)
        dev = DeviceCache(torch, state)
        dev.free = free
        slots = torch.full((cap,), -7, dtype=torch.int64, device="cuda")
        pos = torch.full((cap,), -7, dtype=torch.int32, device="cuda")
        dev.slots(ctx, torch.tensor(off, dtype=torch.int64, device="cuda"), slots, pos, cap)
        P = n_pages * page
        assert slots[:6].tolist() == [P - 1, P - 2 * page, P - 3 * page, P - 3 * page + 1, P - 3 * page + 2, -7]
        assert pos[:6].tolist() == [page - 1, page, 0, 1, 2, -7] and int(dev.n_free[0]) == 2 and int(dev.status[0]) == 0


@pytest.mark.parametrize("n, most", [(3, 1300), (256, 4), (257, 4), (300, 13), (1024, 4), (1024, 128), (1024, 129), (1025, 5)])
def test_cache_trims_of_many_pages(ctx, torch, n, most):
    """Everything given back at once, in one launch and in two; the next step takes the pages again, the last ones first."""
    pages = torch.randperm(n * most)
    state = ([most * 2] * n, [most] * n, pages.view(n, most).tolist(), [-5] * (n * most), 0, 2, n * most, most)
    dev = DeviceCache(torch, state)
    keep = [0 if i % 3 else 3 for i in range(n)]
    dev.trim(ctx, torch.tensor(keep, dtype=torch.int32, device="cuda"))
    model = ref.Cache(*state)
    assert model.trim(keep) == 0 == int(dev.status[0])
    assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free)
    new = [5] * n
    off = [0] + np.cumsum(new).tolist()
    d = torch.full((off[-1],), -7, dtype=torch.int64, device="cuda")
    p = torch.full((off[-1],), -7, dtype=torch.int32, device="cuda")
    slots, pos = [-7] * off[-1], [-7] * off[-1]
    dev.slots(ctx, torch.tensor(off, dtype=torch.int64, device="cuda"), d, p, off[-1])
    assert model.slots(off, off[-1], slots, pos) == int(dev.status[0])
    assert dev.state() == (model.length, model.held, model.table, model.free, model.n_free)
    assert d.tolist() == slots and p.tolist() == pos


@pytest.mark.parametrize("n, most", [(1, 131072), (1, 131073), (1, 1000000), (3, 40001), (3, 333333), (16, 8192), (17, 8191), (256, 512), (300, 436),
                                     (1000, 131), (1023, 128), (7, 130), (5, 131), (2, 2)])
@pytest.mark.parametrize("room", [1.0, 0.6])
def test_cache_trims_of_long_requests(ctx, torch, n, most, room):
    """Few requests with very many pages and the sizes next to the rule's limits: some give all, some a few, some nothing; at 0.6 the
    pool has no room for the later ones."""
    rng = np.random.default_rng(n + most)
    held = rng.integers(most // 2, most + 1, n)
    held[n // 2] = most
    page, n_pages = 2, int(held.sum())
    kind = rng.integers(0, 4, n) if n > 4 else np.arange(n) % 2 * 2
    stay = np.where(kind == 0, 0, np.where(kind == 1, held - 1, np.where(kind == 2, held // 3, held)))
    keep = np.where(kind == 3, -1, stay * page - (stay > 0))
    pages = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n, most), -5, np.int32)
    at = np.append(0, np.cumsum(held))
    for i in range(n):
        table[i, :held[i]] = pages[at[i]:at[i + 1]]
    give = held - stay
    end = np.cumsum(give)
    n_free = n_pages - int(end[-1] * room)
    served = (give == 0) | (n_free + end <= n_pages)
    free = np.arange(-n_pages, 0, dtype=np.int32)
    want = free.copy()
    for i in range(n):
        if served[i] and give[i]:
            want[n_free + end[i] - give[i]:n_free + end[i]] = table[i, stay[i]:held[i]]
    d = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()  # noqa: E731
    L, H, T, F, N, S, K = d(held * page), d(held), d(table), d(free), d([n_free]), d([77]), d(keep)
    need = capi.cache_workspace(n)
    work = torch.full((need,), 0xAB, dtype=torch.uint8, device="cuda")
    ctx.cache_trim(K.data_ptr(), n, L.data_ptr(), H.data_ptr(), page, n_pages, T.data_ptr(), most, most, F.data_ptr(), N.data_ptr(), L.data_ptr(),
                   H.data_ptr(), N.data_ptr(), S.data_ptr(), work.data_ptr(), need)
    assert int(S[0]) == (0 if served.all() else ref.POOL) and int(N[0]) == n_free + int(give[served].sum())
    assert torch.equal(F, d(want)) and torch.equal(T, d(table)) and torch.equal(H, d(np.where(served, stay, held)))
    assert torch.equal(L, d(np.where(served & (kind != 3), np.maximum(keep, 0), held * page)))


def test_cache_without_requests(ctx, torch):
    dev = DeviceCache(torch, ([], [], [], [1, 2, 3, 4], 3, 8, 4, 2))
    z = torch.full((4,), -7, dtype=torch.int64, device="cuda")
    dev.slots(ctx, torch.zeros(1, dtype=torch.int64, device="cuda"), z, z.int(), 4)
    assert int(dev.status[0]) == 0 and int(dev.n_free[0]) == 3 and (z == -7).all()
    dev.status.fill_(9)
    dev.trim(ctx, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert int(dev.status[0]) == 0 and int(dev.n_free[0]) == 3


# ---- verification -------------------------------------------------------------------------------------------------
def _probs(rng, rows, vocab, sharp=3.0):
    x = rng.standard_normal((rows, vocab)) * sharp
    x = np.exp(x - x.max(1, keepdims=True)) if rows else x
    return x / x.sum(1, keepdims=True) if rows else x


def _verify(ctx, torch, draft, off, n_draft, max_draft, target, q, code, vocab, ua, ud, stride, q_stride, shift=0):
    """Runs it and compares with the reference on the values the GPU holds."""
    n = len(off) - 1
    t, _k0, tp, _ = _matrix(torch, target, code, stride, shift, fill=float("nan"))
    qv, qp = None, None
    if q is not None:
        qv, _k1, qp, _ = _matrix(torch, q, code, q_stride, shift, fill=float("nan"))
    dev = lambda a, ty: torch.from_numpy(np.ascontiguousarray(a, dtype=ty)).cuda()  # noqa: E731
    d_draft, d_off = dev(np.append(draft, 0), np.int32), dev(np.asarray(off, dtype=np.uint64).view(np.int64), np.int64)
    d_ua, d_ud = dev(np.append(ua, 0), np.float32), dev(ud, np.float32)
    out = torch.full((n + 1, max_draft + 1), -7, dtype=torch.int32, device="cuda")
    acc = torch.full((n + 1,), -7, dtype=torch.int32, device="cuda")
    need = capi.verify_workspace(n, vocab)
    work = torch.full((need + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    ctx.verify_draft(d_draft.data_ptr(), d_off.data_ptr(), n, n_draft, max_draft, tp, code, stride, qp, q_stride, vocab, d_ua.data_ptr(),
                     d_ud.data_ptr(), out.data_ptr(), acc.data_ptr(), work.data_ptr(), need)
    want, accepted = ref.verify(np.asarray(draft)[:n_draft], off, max_draft, t, qv, vocab, np.asarray(ua, np.float32), np.asarray(ud, np.float32))
    assert acc[:n].tolist() == accepted.tolist()
    assert out[:n].tolist() == want.tolist()
    assert (out[n] == -7).all() and int(acc[n]) == -7 and (work[need:] == 0xAB).all()
    return want, accepted


@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 500, 2047, 2048, 2049, 5001, 128256])
@pytest.mark.parametrize("code", [F32, F16, BF16])
@pytest.mark.parametrize("with_q", [False, True])
def test_verify_vocabularies(ctx, torch, vocab, code, with_q):
    rng = np.random.default_rng(vocab * 6 + code * 2 + with_q)
    n, most = 9, 5
    k = rng.integers(0, most + 1, n)
    k[0], k[1] = most, 0
    off = [0] + np.cumsum(k).tolist()
    total = off[-1]
    target = _probs(rng, total + n, vocab)
    row = np.arange(total) + np.repeat(np.arange(n), k)
    near = target[row] * np.exp(rng.standard_normal((total, vocab)) * 0.5)
    q = near / near.sum(1, keepdims=True)
    draft = np.array([rng.choice(vocab, p=r) for r in q] if with_q else q.argmax(1), dtype=np.int32)
    _verify(ctx, torch, draft, off, total, most, target, q if with_q else None, code, vocab, rng.random(total), rng.random(n),
            vocab + 3, vocab + 1, shift=1)


@pytest.mark.parametrize("n, vocab", [(2047, 4097), (2048, 4097), (2048, 6144), (1536, 6145), (1536, 8193), (700, 20481)])
@pytest.mark.parametrize("code", [F32, BF16])
def test_verify_many_requests(ctx, torch, n, vocab, code):
    """Enough requests that a workgroup has several pieces of a row; rows that end anywhere in them."""
    rng = np.random.default_rng(n + vocab)
    k = rng.integers(0, 2, n)
    off = [0] + np.cumsum(k).tolist()
    total = off[-1]
    target, q = _probs(rng, total + n, vocab), _probs(rng, total, vocab)
    target[rng.random(target.shape) < 0.999] = 0.0      # few entries with weight: wrong by one place is another token
    draft = rng.integers(0, vocab, total).astype(np.int32)
    _verify(ctx, torch, draft, off, total, 1, target, q, code, vocab, rng.random(total), rng.random(n), vocab, vocab)


@pytest.mark.parametrize("k", [1, 2, 63, 64, 65, 130])
def test_verify_many_drafts(ctx, torch, k):
    """Every place at which the first rejection can be, beyond a wave's width; draws at both ends of [0, 1)."""
    rng = np.random.default_rng(k)
    vocab, n = 40, k + 1
    off = [i * k for i in range(n + 1)]
    target = _probs(rng, n * (k + 1), vocab)
    q = _probs(rng, n * k, vocab)
    draft = rng.integers(0, vocab, n * k).astype(np.int32)
    ua = np.zeros((n, k), np.float32)
    for i in range(k):
        ua[i, i] = np.float32(1 - 2 ** -24)
        q[i * k + i, draft[i * k + i]] = 2.0          # with u next to 1 this one is rejected
    ud = np.where(np.arange(n) % 2, 0.0, 1 - 2.0 ** -24).astype(np.float32)
    _, accepted = _verify(ctx, torch, draft, off, n * k, k, target, q, F32, vocab, ua.reshape(-1), ud, vocab, vocab)
    assert accepted.tolist() == list(range(k)) + [k]


def test_verify_borders(ctx, torch):
    """Probabilities and draws whose sums are exact: a draw on a border belongs to the next entry, u q = p is a rejection."""
    vocab = 8
    flat = np.full((17, vocab), 1 / 8)
    off = [0] * 17
    ud = np.arange(16) / 16
    want, _ = _verify(ctx, torch, np.zeros(0, np.int32), off, 0, 0, flat[:16], None, F32, vocab, [], ud, vocab, vocab)
    assert want[:, 0].tolist() == [i // 2 for i in range(16)]
    p, q = np.full((2, vocab), 1 / 8), np.full((1, vocab), 1 / 8)
    q[0, 3], q[0, 4] = 1 / 4, 0
    want, acc = _verify(ctx, torch, np.array([3], np.int32), [0, 1], 1, 1, p, q, F32, vocab, [0.5], [0.0], vocab, vocab)
    assert acc.tolist() == [0] and want.tolist() == [[4, -1]]            # 0.5 * 0.25 = 0.125 is not below it; only 4 is left
    want, acc = _verify(ctx, torch, np.array([3], np.int32), [0, 1], 1, 1, p, q, F32, vocab, [0.49], [0.0], vocab, vocab)
    assert acc.tolist() == [1] and want.tolist() == [[3, 0]]


def test_verify_weights_that_are_none(ctx, torch):
    """Nothing left after the draft: the target itself; no weight at all: -1.  NaN, infinities and negative numbers weigh nothing."""
    vocab, nan, inf = 3000, float("nan"), float("inf")
    p = np.zeros((16, vocab))
    q = np.zeros((8, vocab))
    p[0, [5, 2900]] = 0.5                        # request 0: q covers p, token 7 (p = 0) rejected -> drawn from p
    q[0, [5, 7, 2900]] = 0.5, 1.0, 0.5
    p[2, :] = 0                                  # request 1: no weight anywhere
    q[1, 9] = 1.0
    p[4, [1, 2, 3, 2500]] = nan, inf, -1.0, 0.25  # request 2: only 2500 weighs
    q[2, [1, 2500]] = 1.0, nan                   # ... and q = NaN there: nothing is left, drawn from p
    p[6, [0, 1]] = 0.5, 0.5                      # request 3: a drafted token that is none
    q[3, 1] = 0.5
    off = [0, 1, 2, 3, 4]
    want, acc = _verify(ctx, torch, np.array([7, 9, 1, -1], np.int32), off, 4, 1, p[:8], q[:4], F32, vocab, [0.5] * 4, [0.6] * 4, vocab, vocab)
    assert acc.tolist() == [0, 0, 0, 0] and want[:, 0].tolist() == [2900, -1, 2500, 0]
    # certain drafts: the rejected token is left out, whatever it weighs; one outside the vocabulary leaves all
    p2 = np.zeros((6, 4))
    p2[0, [0, 2]] = 0.5
    p2[2, 1] = 0.25
    p2[4, 3] = 1.0
    want, acc = _verify(ctx, torch, np.array([2, 1, 4], np.int32), [0, 1, 2, 3], 3, 1, p2, None, F32, 4, [0.9, 0.5, 0.0], [0.9, 0.9, 0.0], 4, 4)
    assert acc.tolist() == [0, 0, 0] and want[:, 0].tolist() == [0, 1, 3]


def test_verify_offsets_that_cannot_be(ctx, torch):
    vocab = 16
    p, q = np.full((12, vocab), 1 / 16), np.full((8, vocab), 1 / 16)
    off = [0, 2, 1, 4, 8, 9, 2 ** 62]            # descends, holds more than max_draft, passes n_draft
    want, acc = _verify(ctx, torch, np.arange(8, dtype=np.int32), off, 8, 3, p, q, F32, vocab, [0.5] * 8, [0.5] * 6, vocab, vocab)
    assert acc.tolist() == [2, -1, 3, -1, -1, -1]
    assert (want[[1, 3, 4, 5]] == -1).all()


def test_verify_offsets_beyond_32_bits(ctx, torch):
    """Rows of probabilities so far apart that element offsets pass 2^32."""
    vocab, stride = 16, 2 ** 30 + 7
    target = torch.zeros(4 * stride + vocab, dtype=torch.float16, device="cuda")            # 8 GiB
    q = torch.zeros(3 * stride + vocab, dtype=torch.float16, device="cuda")                 # 6 GiB
    for r, v in enumerate((3, 5, 7, 9, 11)):
        target[r * stride + v] = 1.0
        if r < 4:
            q[r * stride + v] = 1.0
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    off = torch.tensor([0, 4], dtype=torch.int64, device="cuda")
    u, out, acc = torch.full((4,), 0.5, device="cuda"), i32([[-7] * 5]), i32([-7])
    need = capi.verify_workspace(1, vocab)
    work = torch.empty(need, dtype=torch.uint8, device="cuda")
    for draft, want, k in (([3, 5, 7, 9], [3, 5, 7, 9, 11], 4), ([3, 5, 7, 8], [3, 5, 7, 9, -1], 3)):
        ctx.verify_draft(i32(draft).data_ptr(), off.data_ptr(), 1, 4, 4, target.data_ptr(), F16, stride, q.data_ptr(), stride, vocab, u.data_ptr(),
                         u.data_ptr(), out.data_ptr(), acc.data_ptr(), work.data_ptr(), need)
        assert out.tolist() == [want] and int(acc[0]) == k


def test_verify_draws_what_the_target_says(ctx, torch):
    """20,000 requests of one drafted token: what comes out is distributed as the target, for each token within five standard
    deviations of a share of 20,000 (a sound draw misses that once in a million tokens)."""
    rng = np.random.default_rng(77)
    vocab, n = 12, 20000
    p1, q1, p2 = _probs(rng, 1, vocab, 1.0)[0], _probs(rng, 1, vocab, 1.0)[0], _probs(rng, 1, vocab, 1.0)[0]
    target = np.empty((2 * n, vocab))
    target[0::2], target[1::2] = p1, p2
    q = np.tile(q1, (n, 1))
    draft = rng.choice(vocab, n, p=q1).astype(np.int32)
    want, acc = _verify(ctx, torch, draft, list(range(n + 1)), n, 1, target, q, F32, vocab, rng.random(n), rng.random(n), vocab, vocab)
    share = np.bincount(want[:, 0], minlength=vocab) / n
    assert (np.abs(share - p1) <= 5 * np.sqrt(p1 * (1 - p1) / n)).all()
    second = want[acc == 1, 1]
    share = np.bincount(second, minlength=vocab) / len(second)
    assert (np.abs(share - p2) <= 5 * np.sqrt(p2 * (1 - p2) / len(second))).all()


# ---- streams, graphs, threads -------------------------------------------------------------------------------------
def test_calls_follow_their_stream(ctx, torch):
    """Inputs that are still being made on the stream, and the null stream for torch's default stream."""
    ids = torch.zeros(4096, dtype=torch.int32, device="cuda")
    table = torch.randn(100, 256, device="cuda")
    out = torch.zeros(4096, 256, device="cuda")
    big = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for stream in (torch.cuda.Stream(), None):
        with torch.cuda.stream(stream) if stream else torch.cuda.stream(torch.cuda.default_stream()):
            x = big
            for _ in range(8):
                x = x @ big * 1e-2
            ids.copy_((torch.arange(4096, device="cuda") % 100).int() + (x[0, 0] * 0).int())
            ctx.embed(ids.data_ptr(), 4096, table.data_ptr(), F32, 100, 256, 256, out.data_ptr(), F32, 256, 1.0, None,
                      torch.cuda.current_stream().cuda_stream)
            got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, table[(torch.arange(4096) % 100).cuda()])
        ids.zero_()
        out.zero_()
        torch.cuda.synchronize()


def test_captured_and_replayed(ctx, torch):
    """All operators in two captured graphs, each replayed several times with new inputs and eager work between, against eager calls."""
    rng = np.random.default_rng(4)
    n, rows, dim, seqs, vocab, most = 600, 500, 136, 20, 3001, 3

    def buffers():
        import random
        b = dict(ids=torch.zeros(n, dtype=torch.int32, device="cuda"), table=torch.randn(rows, dim, device="cuda").bfloat16(),
                 out=torch.zeros(n, dim, device="cuda"), dy=torch.randn(n, dim, device="cuda"), grad=torch.zeros(rows, dim, device="cuda"),
                 whole=torch.zeros(rows, dim, device="cuda"), work=torch.empty(capi.embed_grad_workspace(n, dim), dtype=torch.uint8, device="cuda"),
                 off=torch.zeros(seqs + 1, dtype=torch.int64, device="cuda"), slots=torch.zeros(n, dtype=torch.int64, device="cuda"),
                 pos=torch.zeros(n, dtype=torch.int32, device="cuda"), keep=torch.zeros(seqs, dtype=torch.int32, device="cuda"))
        b["cache"] = DeviceCache(torch, (*random_cache(random.Random(1), seqs, 8, 40, 2000, full=0.03), 8, 2000, 40))
        k = np.arange(seqs) % (most + 1)
        total = int(k.sum())
        b["voff"] = torch.from_numpy(np.append(0, np.cumsum(k))).cuda()
        b["draft"] = torch.zeros(total, dtype=torch.int32, device="cuda")
        b["target"] = torch.softmax(torch.randn(total + seqs, vocab, device="cuda"), -1)
        b["q"] = torch.softmax(torch.randn(total, vocab, device="cuda"), -1)
        b["ua"], b["ud"] = torch.zeros(total, device="cuda"), torch.zeros(seqs, device="cuda")
        b["vout"], b["acc"] = torch.zeros(seqs, most + 1, dtype=torch.int32, device="cuda"), torch.zeros(seqs, dtype=torch.int32, device="cuda")
        b["vwork"] = torch.empty(capi.verify_workspace(seqs, vocab), dtype=torch.uint8, device="cuda")
        return b

    def run(b):
        s = torch.cuda.current_stream().cuda_stream
        ctx.embed(b["ids"].data_ptr(), n, b["table"].data_ptr(), BF16, rows, dim, dim, b["out"].data_ptr(), F32, dim, 2.0, b["off"].data_ptr() + 8 * seqs, s)
        for t, acc in ((b["grad"], True), (b["whole"], False)):
            ctx.embed_grad(b["ids"].data_ptr(), n, b["dy"].data_ptr(), F32, dim, rows, dim, t.data_ptr(), F32, dim, b["work"].data_ptr(),
                           b["work"].numel(), 1.0, acc, b["off"].data_ptr() + 8 * seqs, s)
        b["cache"].slots(ctx, b["off"], b["slots"], b["pos"], n, s)
        b["cache"].trim(ctx, b["keep"], s)
        ctx.verify_draft(b["draft"].data_ptr(), b["voff"].data_ptr(), seqs, b["draft"].numel(), most, b["target"].data_ptr(), F32, vocab,
                         b["q"].data_ptr(), vocab, vocab, b["ua"].data_ptr(), b["ud"].data_ptr(), b["vout"].data_ptr(), b["acc"].data_ptr(),
                         b["vwork"].data_ptr(), b["vwork"].numel(), s)

    def inputs(bs, rng):
        new = rng.integers(0, 25, seqs)
        off = np.minimum(np.append(0, np.cumsum(new)), n)
        ids = _ids(rng, n, rows)
        keep = rng.choice([-1, 0, 30, 1000], seqs).astype(np.int32)
        total = bs[0]["draft"].numel()
        draft, ua, ud = rng.integers(0, vocab, total).astype(np.int32), rng.random(total).astype(np.float32), rng.random(seqs).astype(np.float32)
        for b in bs:
            for k, v in (("off", off), ("ids", ids), ("keep", keep), ("draft", draft), ("ua", ua), ("ud", ud)):
                b[k].copy_(torch.from_numpy(v))

    pairs = []
    for _ in range(2):
        torch.manual_seed(5)
        a = buffers()
        torch.manual_seed(5)
        b = buffers()
        inputs((a, b), rng)
        g = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            run(a)
        pairs.append((g, a, b))
    for turn in range(4):
        for g, a, b in pairs:
            inputs((a, b), rng)
            g.replay()
            run(b)
            torch.cuda.synchronize()
            for k in ("out", "grad", "whole", "slots", "pos", "vout", "acc"):
                assert torch.equal(a[k], b[k]), (turn, k)
            assert a["cache"].state() == b["cache"].state() and int(a["cache"].status[0]) == int(b["cache"].status[0])


# ids that are ranked / sorted by digits, requests of two launches
@pytest.mark.parametrize("n, dim, seqs", [(3000, 1100, 1100), (9000, 136, 1500)])
def test_captured_and_replayed_on_their_workspaces(ctx, torch, n, dim, seqs):
    """The calls of several launches that hand their work on through a workspace, in two captured graphs with a workspace each, replayed
    with new inputs, at the same time on two streams, with eager work between, against eager calls.  Within a graph the two gradients
    share one workspace, and so do slots and trim."""
    import random
    rng = np.random.default_rng(n)
    rows, vocab, most, page, max_pages = 500, 5001, 2, 8, 12
    n_pages = seqs * max_pages
    k = np.arange(seqs) % (most + 1)
    total = int(k.sum())
    start = random_cache(random.Random(1), seqs, page, max_pages, n_pages, full=0.03)

    def buffers(seed):
        torch.manual_seed(seed)
        b = dict(ids=torch.zeros(n, dtype=torch.int32, device="cuda"), dy=torch.randn(n, dim, device="cuda").bfloat16(),
                 grad=torch.zeros(rows, dim, device="cuda"), whole=torch.zeros(rows, dim, device="cuda"),
                 work=torch.randint(0, 256, (capi.embed_grad_workspace(n, dim),), dtype=torch.uint8, device="cuda"),
                 off=torch.zeros(seqs + 1, dtype=torch.int64, device="cuda"), slots=torch.zeros(n, dtype=torch.int64, device="cuda"),
                 pos=torch.zeros(n, dtype=torch.int32, device="cuda"), keep=torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                 voff=torch.from_numpy(np.append(0, np.cumsum(k))).cuda(), draft=torch.zeros(total, dtype=torch.int32, device="cuda"),
                 target=torch.softmax(torch.randn(total + seqs, vocab, device="cuda"), -1), q=torch.softmax(torch.randn(total, vocab, device="cuda"), -1),
                 ua=torch.zeros(total, device="cuda"), ud=torch.zeros(seqs, device="cuda"),
                 vout=torch.zeros(seqs, most + 1, dtype=torch.int32, device="cuda"), acc=torch.zeros(seqs, dtype=torch.int32, device="cuda"),
                 vwork=torch.randint(0, 256, (capi.verify_workspace(seqs, vocab),), dtype=torch.uint8, device="cuda"))
        b["cache"] = DeviceCache(torch, (*start, page, n_pages, max_pages))
        return b

    def run(b):
        s = torch.cuda.current_stream().cuda_stream
        for t, acc in ((b["grad"], True), (b["whole"], False)):
            ctx.embed_grad(b["ids"].data_ptr(), n, b["dy"].data_ptr(), BF16, dim, rows, dim, t.data_ptr(), F32, dim, b["work"].data_ptr(),
                           b["work"].numel(), 1.0, acc, b["off"].data_ptr() + 8 * seqs, s)
        b["cache"].slots(ctx, b["off"], b["slots"], b["pos"], n, s)
        b["cache"].trim(ctx, b["keep"], s)
        ctx.verify_draft(b["draft"].data_ptr(), b["voff"].data_ptr(), seqs, total, most, b["target"].data_ptr(), F32, vocab, b["q"].data_ptr(), vocab,
                         vocab, b["ua"].data_ptr(), b["ud"].data_ptr(), b["vout"].data_ptr(), b["acc"].data_ptr(), b["vwork"].data_ptr(),
                         b["vwork"].numel(), s)

    def inputs(bs):
        off = np.minimum(np.append(0, np.cumsum(rng.integers(0, 2 * n // seqs + 1, seqs))), n)
        keep = rng.choice([-1, 0, 30, 1000], seqs).astype(np.int32)
        draft, ua, ud = rng.integers(0, vocab, total).astype(np.int32), rng.random(total).astype(np.float32), rng.random(seqs).astype(np.float32)
        for b in bs:
            for name, v in (("off", off), ("ids", _ids(np.random.default_rng(int(off[-1])), n, rows)), ("keep", keep), ("draft", draft), ("ua", ua), ("ud", ud)):
                b[name].copy_(torch.from_numpy(v))

    pairs = []
    for seed in range(2):
        a, b = buffers(seed), buffers(seed)
        inputs((a, b))
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            run(a)
        pairs.append((g, s, a, b))
    for turn in range(4):
        for _, _, a, b in pairs:
            inputs((a, b))
        torch.cuda.synchronize()
        for g, s, _, _ in pairs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, _, a, b in pairs:
            run(b)
            torch.cuda.synchronize()
            for name in ("grad", "whole", "slots", "pos", "vout", "acc"):
                assert torch.equal(a[name], b[name]), (turn, name)
            assert a["cache"].state() == b["cache"].state() and int(a["cache"].status[0]) == int(b["cache"].status[0])
            # (and the eager calls are right: the sums of whole gradients, the positions)
            count = int(b["off"][seqs])
            ids = b["ids"][:count].long()
            there = (ids >= 0) & (ids < rows)
            want = torch.zeros(rows, dim, device="cuda", dtype=torch.float64).index_add_(0, ids[there], b["dy"][:count][there].double())
            size = torch.zeros(rows, dim, device="cuda", dtype=torch.float64).index_add_(0, ids[there], b["dy"][:count][there].double().abs())
            m = torch.bincount(ids[there], minlength=rows).double()[:, None]
            assert ((b["whole"].double() - want).abs() <= (m + 2) * U * size * (1 + (m + 2) * U) + U * want.abs() + 2.0 ** -149).all()


def test_two_threads(ctx, torch):
    """Calls on one context from two threads, each on a stream and workspace of its own."""
    import threading
    rng = np.random.default_rng(6)
    n, rows, dim = 3000, 400, 72
    jobs, errors = [], []
    for _ in range(2):
        ids = torch.from_numpy(_ids(rng, n, rows)).cuda()
        dy = torch.from_numpy(rng.integers(-8, 9, (n, dim))).float().cuda()
        there = ((ids >= 0) & (ids < rows)).float()[:, None]
        want = torch.zeros(rows, dim, device="cuda").index_add_(0, ids.clamp(0, rows - 1).long(), dy * there)
        jobs.append((ids, dy, want, torch.empty(rows, dim, device="cuda"), torch.empty(capi.embed_grad_workspace(n, dim), dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()

    def go(ids, dy, want, got, work):
        try:
            s = torch.cuda.Stream()
            for _ in range(50):
                ctx.embed_grad(ids.data_ptr(), n, dy.data_ptr(), F32, dim, rows, dim, got.data_ptr(), F32, dim, work.data_ptr(), work.numel(), 1.0,
                               False, None, s.cuda_stream)
                s.synchronize()
                assert torch.equal(got, want)
        except Exception as e:   # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=go, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors


def test_two_contexts_and_the_current_device(ctx, torch):
    """Two contexts on one GPU take turns on one stream; the current device stays what it was."""
    other = capi.Context(device=0)
    try:
        table = torch.randn(9, 24, device="cuda")
        ids = torch.tensor([8, 0, 3], dtype=torch.int32, device="cuda")
        mid, out = torch.zeros(3, 24, device="cuda"), torch.zeros(3, 24, device="cuda")
        again = torch.tensor([2, 1, 0], dtype=torch.int32, device="cuda")
        for _ in range(20):
            ctx.embed(ids.data_ptr(), 3, table.data_ptr(), F32, 9, 24, 24, mid.data_ptr(), F32, 24)
            other.embed(again.data_ptr(), 3, mid.data_ptr(), F32, 3, 24, 24, out.data_ptr(), F32, 24)
        assert torch.equal(out, table[[3, 0, 8]]) and torch.cuda.current_device() == 0
    finally:
        other.close()


def test_refusals_leave_the_context_usable(ctx, torch):
    table = torch.randn(4, 8, device="cuda")
    out = torch.full((2, 8), -7.0, device="cuda")
    ids = torch.tensor([1, 3], dtype=torch.int32, device="cuda")
    with pytest.raises(capi.L3Error) as e:
        ctx.embed(ids.data_ptr(), 2, table.data_ptr(), 9, 4, 8, 8, out.data_ptr(), F32, 8)
    assert e.value.code == capi.L3_E_INVALID_ARG and "type" in str(e.value)
    with pytest.raises(capi.L3Error) as e:
        ctx.embed_grad(ids.data_ptr(), 2, out.data_ptr(), F32, 8, 4, 8, table.data_ptr(), F32, 8, table.data_ptr(), 16)
    assert "l3_embed_grad_workspace" in str(e.value)
    assert (out == -7).all()
    ctx.embed(ids.data_ptr(), 2, table.data_ptr(), F32, 4, 8, 8, out.data_ptr(), F32, 8)
    assert torch.equal(out, table[ids.long()])


def test_refusals_on_two_threads_have_their_own_texts(ctx, torch):
    import threading
    at = torch.zeros(64, device="cuda").data_ptr()
    wrong = []

    def go(dim, rows, word):
        for _ in range(3000):
            try:
                ctx.embed(at, 1, at, F32, rows, dim, dim, at, F32, dim)
                wrong.append("taken")
            except capi.L3Error as e:
                if e.code != capi.L3_E_INVALID_ARG or word not in str(e):
                    wrong.append(str(e))

    threads = [threading.Thread(target=go, args=a) for a in ((0, 1, "dim"), (1, 0, "n_rows"), (1, 2 ** 40, "n_rows"))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]


def test_refusals_do_not_wait_for_a_batch(ctx, torch):
    """An encode call of another thread holds the context while its batch runs; a refused operator returns meanwhile.  With a
    batch of tens of milliseconds and refusals of some ten microseconds there is room for thousands; where each waits there are two
    for a batch at most."""
    import threading
    text = np.frombuffer(b"some words, 123 of them\n" * (1 << 21), dtype=np.uint8)      # 48 MiB
    off = np.arange(0, len(text) + 1, 1 << 16, dtype=np.uint64)
    off[-1] = len(text)
    ctx.encode_batch(text, off)
    at = torch.zeros(64, device="cuda").data_ptr()
    batches = 6
    side = threading.Thread(target=lambda: [ctx.encode_batch(text, off) for _ in range(batches)])
    side.start()
    refused = 0
    while side.is_alive():
        with pytest.raises(capi.L3Error):
            ctx.embed(at, 1, at, 9, 1, 1, 1, at, F32, 1)
        refused += 1
    side.join()
    assert refused > 10 * batches, refused


# ---- together -----------------------------------------------------------------------------------------------------
def test_from_text_to_text(ctx, torch, oracle):
    """Prompts are encoded, take pages, are looked up; drafts are verified, what was not accepted is trimmed, the answers decoded; and
    the lookup's gradient comes back.  The ids never leave the GPU before decode."""
    import random
    rng = random.Random(8)
    docs = [b"Hello, world!", b"", "don't 12345 café\n\n".encode()] + [corpus.random_doc(rng, max_pieces=12) for _ in range(29)]
    text, off = capi.pack_docs(docs)
    n, vocab, dim, most, page = len(docs), ctx.vocab_size(), 64, 4, 16
    cap = int(text.size) * 3 + 2 * n
    d_text = torch.from_numpy(text.copy()).cuda()
    d_doc = torch.from_numpy(off.astype(np.int64)).cuda()
    ids = torch.full((cap,), -1, dtype=torch.int32, device="cuda")
    d_off = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    torch.cuda.synchronize()
    rc, total = ctx.encode_batch_device(d_text.data_ptr(), int(text.size), d_doc.data_ptr(), n, capi.L3_BOS, ids.data_ptr(), cap, d_off.data_ptr())
    assert rc == capi.L3_OK
    want_ids, want_off = oracle.encode_batch(text, off, True, False, threads=2)
    lens = np.diff(want_off.astype(np.int64))

    max_pages = int(-(-(lens.max() + most + 1) // page))
    state = ([0] * n, [0] * n, [[-5] * max_pages] * n, list(range(n * max_pages)), n * max_pages, page, n * max_pages, max_pages)
    cache = DeviceCache(torch, state)
    slots = torch.full((cap,), -7, dtype=torch.int64, device="cuda")
    pos = torch.full((cap,), -7, dtype=torch.int32, device="cuda")
    cache.slots(ctx, d_off, slots, pos, cap)
    model = ref.Cache(*state)
    m_slots, m_pos = [-7] * cap, [-7] * cap
    assert model.slots(want_off.astype(int).tolist(), cap, m_slots, m_pos) == 0 == int(cache.status[0])
    assert slots.tolist() == m_slots and pos.tolist() == m_pos

    table = torch.randn(vocab, dim, device="cuda").bfloat16()
    hidden = torch.full((cap, dim), -7.0, dtype=torch.bfloat16, device="cuda")
    ctx.embed(ids.data_ptr(), cap, table.data_ptr(), BF16, vocab, dim, dim, hidden.data_ptr(), BF16, dim, 1.0, d_off.data_ptr() + 8 * n)
    assert torch.equal(hidden[:total], table[torch.from_numpy(want_ids.astype(np.int64)).cuda()]) and (hidden[total:] == -7).all()

    # a model that is certain: it continues every prompt with its own first four tokens; the draft has every third one wrong
    k = np.minimum(lens, most)
    voff = np.append(0, np.cumsum(k))
    first = [want_ids[int(want_off[i]):int(want_off[i]) + k[i]] for i in range(n)]
    draft = np.concatenate(first).astype(np.int32)
    target = torch.zeros(int(voff[-1]) + n, vocab, device="cuda")
    for i in range(n):
        for j in range(k[i] + 1):
            target[voff[i] + i + j, int(first[i][j]) if j < k[i] else 128001] = 1.0
    wrong = np.arange(len(draft)) % 3 == 2
    d_draft = torch.from_numpy(np.where(wrong, (draft + 1) % 1000, draft).astype(np.int32)).cuda()
    d_voff = torch.from_numpy(voff).cuda()
    ua, ud = torch.rand(len(draft), device="cuda"), torch.rand(n, device="cuda")
    out = torch.empty(n, most + 1, dtype=torch.int32, device="cuda")
    acc = torch.empty(n, dtype=torch.int32, device="cuda")
    vwork = torch.empty(capi.verify_workspace(n, vocab), dtype=torch.uint8, device="cuda")
    # the step's tokens (the last one of the prompt is in the cache already): the k drafted ones
    s2, p2 = torch.full((len(draft),), -7, dtype=torch.int64, device="cuda"), torch.full((len(draft),), -7, dtype=torch.int32, device="cuda")
    cache.slots(ctx, d_voff, s2, p2, len(draft))
    assert int(cache.status[0]) == 0 and int(s2.min()) >= 0
    ctx.verify_draft(d_draft.data_ptr(), d_voff.data_ptr(), n, len(draft), most, target.data_ptr(), F32, vocab, None, 0, vocab, ua.data_ptr(),
                     ud.data_ptr(), out.data_ptr(), acc.data_ptr(), vwork.data_ptr(), vwork.numel())
    keep = (torch.from_numpy(lens).cuda() + acc).int()
    cache.trim(ctx, keep)
    assert int(cache.status[0]) == 0 and cache.len.tolist() == keep.tolist()
    accepted, answers = acc.tolist(), out.cpu().numpy()
    for i in range(n):
        good = next((j for j in range(k[i]) if wrong[voff[i] + j] and int(d_draft[voff[i] + j]) != int(draft[voff[i] + j])), k[i])
        assert accepted[i] == good
        line = [int(x) for x in first[i][:good + 1]] + ([128001] if good == k[i] else [])
        assert answers[i].tolist() == line + [-1] * (most + 1 - len(line))
    got, goff = ctx.decode_batch(answers.reshape(-1), np.arange(n + 1, dtype=np.uint64) * (most + 1))
    for i in range(n):
        assert got[int(goff[i]):int(goff[i + 1])].tobytes() == oracle.decode([t for t in answers[i].tolist() if t >= 0])

    grad = torch.empty(vocab, dim, device="cuda")
    dy = torch.ones(cap, dim, dtype=torch.bfloat16, device="cuda")
    work = torch.empty(capi.embed_grad_workspace(cap, dim), dtype=torch.uint8, device="cuda")
    ctx.embed_grad(ids.data_ptr(), cap, dy.data_ptr(), BF16, dim, vocab, dim, grad.data_ptr(), F32, dim, work.data_ptr(), work.numel(), 1.0, False,
                   d_off.data_ptr() + 8 * n)
    count = np.bincount(want_ids, minlength=vocab)
    assert torch.equal(grad.cpu(), torch.from_numpy(np.repeat(count[:, None], dim, 1)).float())
