"""The operators that learn node classifiers (stag_amd.train, include/stag_train.h) against plain 64-bit implementations."""
import math
import os

import numpy as np
import pytest
import torch

from stag_amd import train

if os.path.exists("/dev/kfd"):
    torch.cuda.is_available()      # torch's copy of the HIP runtime has to be the first in a process

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -23                     # a 32-bit operation is off by at most half of this, whichever way it rounds by at most this


def packed(rng, n, n_features, density=0.2, garbage=True):
    """Random packed rows; the bits behind the last feature hold garbage, which has to be ignored."""
    words = -(-n_features // 128) * 4
    x = rng.random((n, words * 32)) < density
    if not garbage:
        x[:, n_features:] = False
    bits = np.packbits(x, axis=1, bitorder="little").view(np.int32).reshape(n, words)
    return torch.from_numpy(bits.copy()).to(DEV), x[:, :n_features].astype(np.float64)


def picked(x, rows):
    """The batch's rows of x, and which of them are no padding."""
    if rows is None:
        return x, np.ones(len(x), bool)
    real = (rows >= 0) & (rows < len(x))
    return x[np.where(real, rows, 0)] * real[:, None], real


def half_step(t, dtype):
    """Half a step of dtype at |t| (values below the smallest normal ones: half of the smallest step)."""
    info = torch.finfo(dtype)
    return np.maximum(np.abs(t), info.smallest_normal) * info.eps / 2


def near(got, want, tol, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), "%s: %d of %d off; worst %g over its tolerance at %s" % (
        what, bad.sum(), bad.size, np.nanmax((np.abs(got - want) / np.maximum(tol, 1e-300))[bad]), np.argwhere(bad)[0])


# n rows held, batch (None: all rows in order), features, classifiers
SHAPES = [
    (1, None, 1, 1), (1, None, 145, 2), (2, None, 31, 3), (3, None, 32, 8), (5, 7, 33, 1), (16, None, 127, 31), (17, 1, 128, 32), (20, 40, 129, 33),
    (31, None, 145, 7), (32, None, 640, 64), (33, 65, 643, 65), (64, None, 750, 13), (65, 63, 750, 100), (100, 129, 1000, 257), (300, None, 2100, 5),
    (200, 300, 5250, 4), (1, None, 7500, 8), (4, 4, 7500, 1000), (1000, 1025, 300, 40), (700, 513, 1500, 96), (2000, 3001, 145, 10), (40, None, 20000, 12),
    (600, 1100, 700, 300), (2100, 2100, 2600, 400), (5, None, 40000, 9), (400, 513, 33000, 33),
]


def batch(rng, n, m):
    if m is None:
        return None, None
    rows = rng.integers(0, n, m).astype(np.int32)
    rows[rng.random(m) < 0.1] = -1
    if m > 2:
        rows[[0, m - 1]] = [n, 2**31 - 1]      # past the end is padding too
    return rows, torch.from_numpy(rows).to(DEV)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, m, n_features, k", SHAPES)
def test_scores(n, m, n_features, k, dtype):
    rng = np.random.default_rng(n + 7 * n_features + k)
    bits, x = packed(rng, n, n_features)
    rows, d_rows = batch(rng, n, m)
    table = torch.from_numpy(rng.normal(size=(n_features, k)).astype(np.float32)).to(DEV).to(dtype)
    bias = torch.from_numpy(rng.normal(size=k).astype(np.float32)).to(DEV)
    scale = 0.37
    got = train.row_scores(bits, table, bias, scale=scale, rows=d_rows)
    assert got.dtype == F32
    xb, real = picked(x, rows)
    t, b = table.double().cpu().numpy(), bias.double().cpu().numpy()
    want = np.where(real[:, None], scale * (xb @ t) + b, 0.0)
    # a sum of N terms in 32 bits, in any order, is off by at most N U sum|terms|; the rounding of scale, product and bias: 4 more
    tol = (xb.sum(1)[:, None] + 4) * U * (scale * (xb @ np.abs(t)) + np.abs(b)) * real[:, None]
    near(got.cpu(), want, tol)
    assert torch.equal(got, train.row_scores(bits, table, bias, scale=scale, rows=d_rows))
    near(train.row_scores(bits, table, scale=scale, rows=d_rows).cpu(), np.where(real[:, None], scale * (xb @ t), 0.0), tol)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, m, n_features, k", SHAPES)
def test_grad(n, m, n_features, k, dtype):
    rng = np.random.default_rng(n + 7 * n_features + k)
    bits, x = packed(rng, n, n_features)
    rows, d_rows = batch(rng, n, m)
    xb, real = picked(x, rows)
    grad = torch.from_numpy(rng.normal(size=(len(xb), k)).astype(np.float32)).to(DEV).to(dtype)
    g = np.where(real[:, None], grad.double().cpu().numpy(), 0.0)
    grad[torch.from_numpy(~real).to(DEV)] = math.nan         # padding rows hold anything
    scale = 0.37
    table_grad, bias_grad = train.row_scores_grad(bits, grad, n_features, scale=scale, rows=d_rows)
    assert table_grad.dtype == bias_grad.dtype == F32
    near(table_grad.cpu(), scale * (xb.T @ g), (xb.sum(0)[:, None] + 4) * U * scale * (xb.T @ np.abs(g)), "table")
    near(bias_grad.cpu(), g.sum(0), (real.sum() + 4) * U * np.abs(g).sum(0), "bias")
    again = train.row_scores_grad(bits, grad, n_features, scale=scale, rows=d_rows)
    assert torch.equal(table_grad, again[0]) and torch.equal(bias_grad, again[1])


@pytest.mark.parametrize("n, k, n_features", [(4, 3, 900), (80, 8, 900), (700, 24, 900), (2500, 200, 900), (2100, 400, 2500)])
def test_32_bit_values_keep_their_24_bits(n, k, n_features):
    """One token a row, so that nothing hides the rounding of a value: what comes back is the value."""
    rng = np.random.default_rng(n)
    words = -(-n_features // 128) * 4
    f = rng.permutation(np.arange(n) % n_features)
    bits = np.zeros((n, words), np.uint32)
    bits[np.arange(n), f >> 5] = np.uint32(1) << (f & 31).astype(np.uint32)
    bits = torch.from_numpy(bits.view(np.int32)).to(DEV)
    table = torch.from_numpy((rng.normal(size=(n_features, k)) * 10.0 ** rng.uniform(-12, 12, size=(n_features, k))).astype(np.float32)).to(DEV)
    got = train.row_scores(bits, table).cpu().numpy()
    want = table.cpu().numpy()[f]
    near(got, want, 2 * U * np.abs(want))
    grad = torch.from_numpy((rng.normal(size=(n, k)) * 10.0 ** rng.uniform(-12, 12, size=(n, k))).astype(np.float32)).to(DEV)
    table_grad = train.row_scores_grad(bits, grad, n_features)[0].cpu().numpy()
    want, size = np.zeros((n_features, k)), np.zeros((n_features, k))
    np.add.at(want, f, grad.double().cpu().numpy())
    np.add.at(size, f, grad.double().abs().cpu().numpy())
    near(table_grad, want, (2 + n // n_features + 1) * U * size)


@pytest.mark.parametrize("n, k, n_features", [(1, 4, 333), (40, 5, 333), (600, 70, 333), (1500, 200, 333), (2100, 400, 2500), (700, 20, 333)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_infinities_reach_only_the_rows_that_have_the_token(n, k, n_features, dtype):
    rng = np.random.default_rng(9)
    bits, x = packed(rng, n, n_features)
    table = torch.from_numpy(rng.normal(size=(n_features, k)).astype(np.float32)).to(DEV).to(dtype)
    table[17, 0], table[200, k - 1], table[201, k // 2] = math.inf, math.nan, -math.inf
    got = train.row_scores(bits, table).cpu().numpy()
    t = table.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = np.stack([t[r > 0].sum(0) for r in x])
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)])
    near(got[fine], want[fine], n_features * U * np.abs(t[np.isfinite(t)]).max() * n_features)
    grad = torch.from_numpy(rng.normal(size=(n, k)).astype(np.float32)).to(DEV).to(dtype)
    grad[n // 2, 0], grad[n - 1, k - 1] = math.inf, math.nan
    got = train.row_scores_grad(bits, grad, n_features)
    g = grad.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = np.stack([g[c > 0].sum(0) for c in x.T])
        near_bias = g.sum(0)
    assert np.array_equal(np.isnan(got[0].cpu().numpy()), np.isnan(want)) and np.array_equal(np.isinf(got[0].cpu().numpy()), np.isinf(want))
    assert np.array_equal(np.isnan(got[1].cpu().numpy()), np.isnan(near_bias)) and np.array_equal(np.isinf(got[1].cpu().numpy()), np.isinf(near_bias))


def with_special(finite, has, special):
    """finite + the infinities and NaN of `special` [terms, k] that each sum has: has [sums, terms] of 0 and 1."""
    up, down, nan = (has @ x.astype(np.float64) > 0 for x in (special == np.inf, special == -np.inf, np.isnan(special)))
    return np.where(nan | (up & down), np.nan, np.where(up, np.inf, np.where(down, -np.inf, finite)))


@pytest.mark.parametrize("share", [0.002, 0.2, 1.0])
@pytest.mark.parametrize("n, k, n_features", [(3, 5, 700), (700, 20, 333), (900, 40, 700), (600, 70, 700), (4300, 129, 600), (2100, 400, 2500)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_many_infinities_and_nan(n, k, n_features, dtype, share):
    """A share of all values, up to each, are infinities of both signs and NaN; a few rows and features have nothing; some of the batch is padding."""
    rng = np.random.default_rng(n + k)
    bits, x = packed(rng, n, n_features, density=0.03)
    bits[5::100] = 0
    x[5::100] = 0
    rows, d_rows = batch(rng, n, n)
    xb, real = picked(x, rows)

    def values(shape):
        v = rng.normal(size=shape).astype(np.float32)
        kind = rng.random(shape)
        special = (rng.random(shape) < share) & (rng.random(shape[1]) < 0.7)          # some columns have none
        v[special] = np.where(kind < 0.45, np.inf, np.where(kind < 0.9, -np.inf, np.nan))[special]
        t = torch.from_numpy(v).to(DEV).to(dtype)
        v = t.double().cpu().numpy()
        return t, np.where(np.isfinite(v), v, 0.0), np.where(np.isfinite(v), 0.0, v)

    def check(got, want, tol):
        got = got.double().cpu().numpy()
        fine = np.isfinite(want)
        assert ((got == want) | (np.isnan(got) & np.isnan(want)))[~fine].all()
        near(got[fine], want[fine], tol[fine])

    table, finite, special = values((n_features, k))
    bias = torch.from_numpy(rng.normal(size=k).astype(np.float32)).to(DEV)
    b = bias.double().cpu().numpy()
    want = np.where(real[:, None], with_special(0.37 * (xb @ finite) + b, xb, special), 0.0)
    check(train.row_scores(bits, table, bias, scale=0.37, rows=d_rows), want, (xb.sum(1)[:, None] + 4) * U * (0.37 * (xb @ np.abs(finite)) + np.abs(b)))
    grad, finite, special = values((n, k))
    table_grad, bias_grad = train.row_scores_grad(bits, grad, n_features, scale=0.37, rows=d_rows)
    check(table_grad, with_special(0.37 * (xb.T @ finite), xb.T, special), (xb.sum(0)[:, None] + 4) * U * 0.37 * (xb.T @ np.abs(finite)))
    r = real[None].astype(np.float64)
    check(bias_grad[None], with_special(r @ finite, r, special), (real.sum() + 4) * U * (r @ np.abs(finite)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_scores_of_a_long_sum_with_nan_all_along_it(dtype):
    """One column has a NaN in each 256 features of a sum that one workgroup adds up; others have single infinities near its end."""
    rng = np.random.default_rng(31)
    n, m, n_features, k = 40, 131_072, 270_000, 64
    assert train._workspace("stag_row_scores_workspace", m, n_features, k, train._TYPES[dtype]) == 0        # not cut into parts
    x = rng.random((n, n_features)) < 0.02
    nan_at = np.arange(200, n_features, 256)
    x[:, nan_at] = False
    x[3, nan_at[1]] = True
    x[4, nan_at[-1]] = True
    x[[7, 8], [269_990, 269_990]] = True
    bits = torch.from_numpy(np.packbits(np.pad(x, ((0, 0), (0, -n_features % 128))), axis=1, bitorder="little").view(np.int32).reshape(n, -1).copy()).to(DEV)
    table = torch.randn((n_features, k), generator=torch.Generator(device=DEV).manual_seed(1), device=DEV)
    table[torch.from_numpy(nan_at).to(DEV), 0] = math.nan
    table[269_990, 7], table[269_000, 40], table[268_001, 40] = math.inf, -math.inf, math.inf
    table = table.to(dtype)
    rows = rng.integers(0, n, m).astype(np.int32)
    rows[rng.random(m) < 0.05] = -1
    got = train.row_scores(bits, table, rows=torch.from_numpy(rows).to(DEV)).cpu().numpy()
    t = table.double().cpu().numpy()
    has, finite = x.astype(np.float64), np.where(np.isfinite(t), t, 0.0)
    want = with_special(has @ finite, has, np.where(np.isfinite(t), 0.0, t))
    tol = (has.sum(1)[:, None] + 4) * U * (has @ np.abs(finite))
    for r in range(n):
        mine = got[rows == r]
        assert (mine == mine[0]).all() or np.array_equal(mine, np.broadcast_to(mine[0], mine.shape), equal_nan=True)
        fine = np.isfinite(want[r])
        assert np.array_equal(mine[0][~fine], want[r][~fine], equal_nan=True), r
        near(mine[0][fine], want[r][fine], tol[r][fine])
    assert np.isinf(want[7, 7]) and np.isnan(want[3, 0]) and np.isfinite(want[5, 0]) and (got[rows < 0] == 0).all()


@pytest.mark.parametrize("n_features, k, m, dtype", [(61_440, 128, 140_000, F32), (61_440, 128, 140_000, F16), (7_500, 1000, 270_000, BF16)])
def test_grad_of_a_long_batch_with_nan_all_along_it(n_features, k, m, dtype):
    """The same for a batch that one workgroup adds up: NaN in one column every 100 rows, single infinities near the end."""
    rng = np.random.default_rng(32)
    n = 50
    bits, x = packed(rng, n, n_features, density=0.05)
    rows = rng.integers(0, n, m)
    nan_at = np.arange(50, m, 100)
    rows[nan_at] = 3
    x[3, :] = 0                                                     # the row that NaN goes with has few features
    x[3, [5, 77, n_features - 1]] = 1
    bits[3] = torch.from_numpy(np.packbits(np.pad(x[3].astype(bool), (0, bits.shape[1] * 32 - n_features)), bitorder="little").view(np.int32)).to(DEV)
    rows[rng.random(m) < 0.05] = -1
    rows[[m - 40, m - 30, m - 20, m - 10]] = 7, 8, 7, -1
    d_rows = torch.from_numpy(rows.astype(np.int32)).to(DEV)
    grad = torch.randn((m, k), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    grad[torch.from_numpy(nan_at).to(DEV), 0] = math.nan
    grad[m - 40, 7], grad[m - 30, 100], grad[m - 20, 100], grad[m - 10, 50] = math.inf, math.inf, -math.inf, math.nan          # the last is padding
    grad = grad.to(dtype)
    table_grad, bias_grad = (t.double().cpu().numpy() for t in train.row_scores_grad(bits, grad, n_features, rows=d_rows))
    # what each held row is picked for, summed in 64 bits
    real, at = d_rows >= 0, d_rows.clamp(min=0).long()
    g = torch.where(real[:, None], grad.double(), 0.0)
    fine, special = torch.where(torch.isfinite(g), g, 0.0), torch.where(torch.isfinite(g), 0.0, g)
    per_row, size = (torch.zeros((n, k), dtype=torch.float64, device=DEV).index_add_(0, at, y).cpu().numpy() for y in (fine, fine.abs()))
    marks = torch.zeros((n, k), dtype=torch.float64, device=DEV).index_add_(0, at, special).cpu().numpy()
    count = np.bincount(rows[rows >= 0], minlength=n)
    want = with_special(x.T @ per_row, x.T, marks)
    tol = ((x.T @ count)[:, None] + 4) * U * (x.T @ size)
    fine = np.isfinite(want)
    assert np.array_equal(table_grad[~fine], want[~fine], equal_nan=True) and (~fine[:, 7]).any() and (~fine[:, 100]).any() and fine[:, 50].all() and fine[1, 0]
    near(table_grad[fine], want[fine], tol[fine])
    one = np.ones((1, n))
    want = with_special(one @ per_row, one, marks)[0]
    fine = np.isfinite(want)
    assert np.array_equal(bias_grad[~fine], want[~fine], equal_nan=True) and (~fine).sum() == 3
    near(bias_grad[fine], want[fine], ((rows >= 0).sum() + 4) * U * size.sum(0)[fine])


def test_infinities_in_sums_of_millions_of_terms():
    """Sums that one workgroup adds up in more than 32,768 groups of terms: 8.6 million features, 4.3 million rows."""
    rng = np.random.default_rng(33)
    m, f, k = 131_072, 8_600_000, 64
    assert train._workspace("stag_row_scores_workspace", m, f, k, 1) == 0
    table = torch.randn((f, k), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(BF16)
    bits = np.zeros((4, -(-f // 128) * 4), np.uint32)
    token = [np.unique(rng.integers(0, f - 100, 20_000)) for _ in range(4)]
    for r, t in enumerate(token):
        token[r] = np.append(t, f - 1 - r)
        np.bitwise_or.at(bits[r], token[r] >> 5, np.uint32(1) << (token[r] & 31).astype(np.uint32))
    table[f - 1, 3], table[f - 2, 40], table[int(token[2][10]), 5], table[int(token[2][10_000]), 5], table[f - 90, 6] = math.inf, -math.inf, math.inf, -math.inf, math.nan
    rows = torch.arange(m, device=DEV, dtype=torch.int32) % 4
    got = train.row_scores(torch.from_numpy(bits.view(np.int32)).to(DEV), table, rows=rows)
    for r in range(4):
        mine, terms = got[r::4], table[torch.from_numpy(token[r]).to(DEV)].double()
        want, size = terms.sum(0).cpu().numpy(), terms.abs().sum(0).cpu().numpy()
        assert torch.equal(mine.nan_to_num(7e30), mine[:1].expand_as(mine).nan_to_num(7e30))
        fine = np.isfinite(want)
        assert (~fine).sum() == (1 if r < 3 else 0) and np.array_equal(mine[0].cpu().numpy()[~fine], want[~fine], equal_nan=True)
        near(mine[0].cpu().numpy()[fine], want[fine], (len(token[r]) + 4) * U * size[fine])
    del table, got
    n, m, f, k = 50, 4_300_000, 61_440, 128
    bits, x = packed(rng, n, f, density=0.05)
    rows = rng.integers(0, n, m).astype(np.int32)
    rows[[m - 1, m - 2, 5]] = 7, 8, 9
    d_rows = torch.from_numpy(rows).to(DEV)
    grad = torch.randn((m, k), generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).to(BF16)
    grad[m - 1, 3], grad[m - 2, 40], grad[5, 40] = math.inf, math.inf, math.nan
    got = train.row_scores_grad(bits, grad, f, rows=d_rows)[0].double().cpu().numpy()
    g = grad.double()
    sums = [torch.zeros((n, k), dtype=torch.float64, device=DEV).index_add_(0, d_rows.long(), y).cpu().numpy()
            for y in (torch.where(torch.isfinite(g), g, 0.0), torch.where(torch.isfinite(g), g.abs(), 0.0), torch.where(torch.isfinite(g), 0.0, g))]
    want = with_special(x.T @ sums[0], x.T, sums[2])
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine], equal_nan=True) and (~fine).any(0).nonzero()[0].tolist() == [3, 40]
    terms = (x.T @ np.bincount(rows, minlength=n))[:, None]
    near(got[fine], want[fine], ((terms + 4) * U * (x.T @ sums[1]))[fine])


@pytest.mark.parametrize("n, k, n_features", [(1, 4, 333), (40, 5, 333), (600, 70, 333), (1500, 200, 333), (2100, 400, 2500), (700, 20, 333)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_sums_near_the_largest_number_beside_infinities(n, k, n_features, dtype):
    """2^127 fits 32 bits, its double does not; an infinity or NaN elsewhere in the batch changes nothing about it."""
    rng = np.random.default_rng(2)
    bits, x = packed(rng, n, n_features)
    table = torch.from_numpy(rng.integers(-4, 5, (n_features, k)).astype(np.float32)).to(DEV).to(dtype)
    table[33, 0] = table[34, k // 2] = 2.0 ** 127
    table[17, 0], table[18, k - 1] = math.inf, math.nan
    got = train.row_scores(bits, table, scale=0.5).double().cpu().numpy()
    t = table.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = 0.5 * np.stack([t[r > 0].sum(0) for r in x])
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    near(got[fine], want[fine], U * np.abs(want[fine]))            # whole numbers: sums of small ones are exact, beside 2^127 they are nothing
    grad = torch.from_numpy(rng.integers(-4, 5, (n, k)).astype(np.float32)).to(DEV).to(dtype)
    grad[n // 3, 0], grad[n // 2, k - 1], grad[n - 1, 1] = 2.0 ** 127, 2.0 ** 127, math.inf
    got = train.row_scores_grad(bits, grad, n_features)[0].double().cpu().numpy()
    g = grad.double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        want = np.stack([g[c > 0].sum(0) for c in x.T])
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fine = np.isfinite(want)
    near(got[fine], want[fine], U * np.abs(want[fine]))


@pytest.mark.parametrize("dtype, smallest", [(F16, 2.0 ** -24), (BF16, 2.0 ** -133), (F32, 2.0 ** -149)])
@pytest.mark.parametrize("n, k", [(6, 8), (700, 24)])
def test_values_below_the_normal_ones(n, k, dtype, smallest):
    """Subnormal coefficients and gradients count.  16-bit ones exactly; the pieces of a 32-bit one are at least 2^-133 apart."""
    rng = np.random.default_rng(n)
    n_features = 300
    words = -(-n_features // 128) * 4
    f = np.arange(n) % n_features
    bits = np.zeros((n, words), np.uint32)
    bits[np.arange(n), f >> 5] = np.uint32(1) << (f & 31).astype(np.uint32)
    bits = torch.from_numpy(bits.view(np.int32)).to(DEV)
    table = torch.from_numpy(rng.integers(-60, 60, (n_features, k)) * smallest).to(dtype).to(DEV)
    slack = 2.0 ** -133 if dtype == F32 else 0.0
    near(train.row_scores(bits, table).double().cpu(), table.double().cpu().numpy()[f], slack)
    grad = torch.from_numpy(rng.integers(-60, 60, (n, k)) * smallest).to(dtype).to(DEV)
    want = np.zeros((n_features, k))
    np.add.at(want, f, grad.double().cpu().numpy())
    near(train.row_scores_grad(bits, grad, n_features)[0].double().cpu(), want, 3 * slack)


def test_offsets_beyond_32_bits():
    """Scores, a table, its gradient and packed rows of more than 2^32 bytes each, looked at where an offset of 32 bits would go astray."""
    rng = np.random.default_rng(0)
    n_features, k, m = 100, 1000, 2_200_000                      # 2.2e9 scores
    base, x = packed(rng, 64, n_features)
    rows = torch.arange(m, device=DEV, dtype=torch.int32) % 64
    rows[-1] = -1
    table = torch.from_numpy(rng.normal(size=(n_features, k)).astype(np.float32)).to(DEV)
    scores = train.row_scores(base, table, rows=rows)
    want = x @ table.double().cpu().numpy()
    for i in (0, 1, 1_073_741, 1_073_742, 2_147_483, 2_147_484, m - 2):
        near(scores[i].cpu(), want[i % 64], (n_features + 4) * U * (x @ np.abs(table.double().cpu().numpy()))[i % 64])
    assert (scores[-1] == 0).all()
    label = (rows % k).to(torch.int32)
    loss, grad = train.sibling_loss(scores, label, scale=1.0, grad_dtype=F16)
    z = scores[m - 2].double().cpu().numpy()
    g = 1 / (1 + np.exp(-z)) - (np.arange(k) == int(label[m - 2]))
    near(grad[m - 2].double().cpu(), g, 8 * U * np.abs(g) + half_step(g, F16) * (1 + 8 * U))
    counts = np.bincount(rows[:-1].cpu().numpy(), minlength=64)
    del scores
    table_grad, bias_grad = train.row_scores_grad(base, grad, n_features, rows=rows)
    per = grad[:64].double().cpu().numpy()                       # rows repeat with a period of 64, and so do their labels
    near(table_grad.double().cpu(), x.T @ (per * counts[:, None]), (m + 4) * U * (x.T @ np.abs(per * counts[:, None])))
    del grad, table_grad
    f, k = 70_000, 32_768                                        # 2.3e9 coefficients in 16 bits, gradients in 32
    bits, x = packed(rng, 3, f)
    table = torch.randn((f, k), device=DEV, dtype=BF16)
    near(train.row_scores(bits, table)[:, -40:].cpu(), x @ table[:, -40:].double().cpu().numpy(), (x.sum(1)[:, None] + 4) * U * (x @ np.abs(table[:, -40:].double().cpu().numpy())))
    grad = torch.from_numpy(rng.normal(size=(3, k)).astype(np.float32)).to(DEV)
    got = train.row_scores_grad(bits, grad, f)[0]
    near(got[-50:].cpu(), x.T[-50:] @ grad.double().cpu().numpy(), 7 * U * (x.T[-50:] @ np.abs(grad.double().cpu().numpy())))
    del table, got
    n, f = 2_400_000, 16_000                                     # 4.8 GB of packed rows
    rows = torch.tensor([0, 1_073_741, 2_147_483, 2_147_484, n - 1, n], dtype=torch.int32, device=DEV)
    bits = torch.zeros((n, 500), dtype=torch.int32, device=DEV)
    small, x = packed(rng, 5, f, garbage=False)
    bits[rows[:5].long()] = small
    table = torch.from_numpy(rng.normal(size=(f, 3)).astype(np.float32)).to(DEV)
    got = train.row_scores(bits, table, rows=rows)
    t = table.double().cpu().numpy()
    near(got[:5].cpu(), x @ t, (x.sum(1)[:, None] + 4) * U * (x @ np.abs(t)))
    assert (got[5] == 0).all()
    grad = torch.from_numpy(rng.normal(size=(6, 3)).astype(np.float32)).to(DEV)
    g = grad[:5].double().cpu().numpy()
    near(train.row_scores_grad(bits, grad, f, rows=rows)[0].cpu(), x.T @ g, 9 * U * (x.T @ np.abs(g)))


@pytest.mark.parametrize("n, k", [(3, 5), (50, 40), (700, 130)])
def test_strided_tables_and_outputs(n, k):
    """Tables, gradients and outputs inside larger buffers at odd places, with what lies between the rows left as it was."""
    rng = np.random.default_rng(5)
    n_features = 777
    words = -(-n_features // 128) * 4
    wide = torch.randint(-2**31, 2**31 - 1, (n, words + 8), device=DEV, dtype=torch.int32)
    bits, x = packed(rng, n, n_features)
    wide[:, 4:4 + words] = bits
    inside = wide[:, 4:4 + words]
    big = torch.from_numpy(rng.normal(size=(n_features, k + 5)).astype(np.float32)).to(DEV)
    table = big[:, 3:3 + k]
    out = torch.full((n, k + 7), 7.0, device=DEV)
    got = train.row_scores(inside, table, out=out[:, 1:1 + k])
    assert got.data_ptr() == out[:, 1:].data_ptr()
    t = table.double().cpu().numpy()
    near(got.cpu(), x @ t, (x.sum(1)[:, None] + 4) * U * (x @ np.abs(t)))
    assert (out[:, 0] == 7).all() and (out[:, 1 + k:] == 7).all()
    near(train.row_scores(bits, table.t().contiguous().t()).cpu(), x @ t, (x.sum(1)[:, None] + 4) * U * (x @ np.abs(t)))   # columns apart: copied
    grad = torch.from_numpy(rng.normal(size=(n, k + 3)).astype(np.float32)).to(DEV)[:, 2:2 + k]
    into = torch.full((n_features + 2, k + 1), 7.0, device=DEV)
    bias = torch.full((k + 2,), 7.0, device=DEV)
    train.row_scores_grad(inside, grad, n_features, out=(into[:n_features, 1:], bias[1:1 + k]))
    g = grad.double().cpu().numpy()
    near(into[:n_features, 1:].cpu(), x.T @ g, (x.sum(0)[:, None] + 4) * U * (x.T @ np.abs(g)))
    assert (into[n_features:] == 7).all() and (into[:, 0] == 7).all() and bias[0] == 7 and bias[-1] == 7
    one = torch.from_numpy(rng.normal(size=(1, k)).astype(np.float32)).to(DEV).expand(n, k)      # a broadcast gradient
    near(train.row_scores_grad(bits, one, n_features)[0].cpu(), x.T @ one.double().cpu().numpy(), (x.sum(0)[:, None] + 4) * U * x.sum(0)[:, None] * 5)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n, k, n_features", [(530, 66, 400), (600, 129, 300), (4200, 197, 2200)])
@pytest.mark.parametrize("left, right", [(4, 4), (0, 0), (1, 2), (8, 5)])
def test_values_between_the_rows_are_not_read(n, k, n_features, left, right, dtype):
    """Tables and gradients inside larger buffers of NaN, at columns that fit wide loads and at others, with widths that end inside one; an infinity of
    their own in the last column goes where it belongs."""
    rng = np.random.default_rng(k)
    width = -(-(left + k) // 4) * 4 + (right if right else 0) if right != 0 else left + k
    bits, x = packed(rng, n, n_features)

    def inside(rows):
        big = torch.full((rows + 1, width), math.nan, device=DEV).to(dtype)
        big[:rows, left:left + k] = torch.from_numpy(rng.normal(size=(rows, k)).astype(np.float32))
        return big[:rows, left:left + k]

    table, grad = inside(n_features), inside(n)
    t, g = table.double().cpu().numpy(), grad.double().cpu().numpy()
    near(train.row_scores(bits, table).cpu(), x @ t, (x.sum(1)[:, None] + 4) * U * (x @ np.abs(t)))
    table_grad, bias_grad = train.row_scores_grad(bits, grad, n_features)
    near(table_grad.cpu(), x.T @ g, (x.sum(0)[:, None] + 4) * U * (x.T @ np.abs(g)))
    near(bias_grad.cpu(), g.sum(0), (n + 4) * U * np.abs(g).sum(0))
    table[n_features - 1, k - 1] = math.inf
    has = x[:, n_features - 1] > 0
    got = train.row_scores(bits, table).double().cpu().numpy()
    assert np.isinf(got[has, k - 1]).all()
    t[n_features - 1, k - 1] = 0.0
    got[has, k - 1] = (x @ t)[has, k - 1]
    near(got, x @ t, (x.sum(1)[:, None] + 4) * U * (x @ np.abs(t)))


def test_empty_batches():
    bits, _ = packed(np.random.default_rng(0), 5, 40)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    table = torch.ones(40, 3, device=DEV)
    assert train.row_scores(bits, table, rows=none).shape == (0, 3)
    assert train.row_scores(bits[:0], table).shape == (0, 3)
    into = (torch.full((40, 3), 7.0, device=DEV), torch.full((3,), 7.0, device=DEV))
    train.row_scores_grad(bits, torch.empty(0, 3, device=DEV), 40, rows=none, out=into)
    assert (into[0] == 0).all() and (into[1] == 0).all()
    padding = torch.full((70,), -1, dtype=torch.int32, device=DEV)
    assert (train.row_scores(bits, table, torch.ones(3, device=DEV), rows=padding) == 0).all()
    assert (train.row_scores(bits[:0], table, torch.ones(3, device=DEV), rows=torch.zeros_like(padding)) == 0).all()
    got = train.row_scores_grad(bits, torch.full((70, 3), math.nan, device=DEV), 40, rows=padding)
    assert (got[0] == 0).all() and (got[1] == 0).all()
    loss, grad = train.sibling_loss(torch.empty(0, 3, device=DEV), none)
    assert (loss == 0).all() and grad.shape == (0, 3)


# ---------------------------------------------------------------------------------------------------------------- loss
def plain_loss(z, label, lo, hi, w, scale):
    m, k = z.shape
    c = np.arange(k)[None, :]
    inside = (c >= lo[:, None]) & (c < hi[:, None])
    y = c == label[:, None]
    with np.errstate(invalid="ignore", over="ignore"):
        s = np.where(y, -z, z)
        loss = np.where(s < 0, 0.0, s) + np.log1p(np.exp(-np.abs(s)))
        p = 1.0 / (1.0 + np.exp(-s))
    loss = np.where(inside, loss, 0.0) * w[:, None] * scale
    return loss.sum(0), np.where(inside, np.where(y, -p, p), 0.0) * w[:, None] * scale, np.abs(loss).sum(0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("siblings", [False, True])
@pytest.mark.parametrize("m, k", [(1, 1), (2, 3), (7, 4), (33, 8), (300, 13), (257, 257), (64, 1000), (5000, 12), (4099, 37), (100, 1025), (3, 4100), (20000, 1)])
def test_loss(m, k, siblings, dtype):
    rng = np.random.default_rng(m + k)
    z = (rng.normal(size=(m, k)) * 5).astype(np.float32)
    lo, hi = np.zeros(m, np.int64), np.full(m, k)
    if siblings:
        lo = rng.integers(0, k, m)
        hi = np.minimum(lo + rng.integers(0, 9, m), k)            # some rows train nothing
        z[(np.arange(k) < lo[:, None]) | (np.arange(k) >= hi[:, None])] = np.nan      # never read
    label = rng.integers(-1, k, m)
    label = np.where(rng.random(m) < 0.7, np.clip(lo + rng.integers(0, 9, m), 0, k + 1), label)
    w = rng.random(m).astype(np.float32) + 0.1
    scale = 2.0 / m
    sib = torch.from_numpy(np.stack([lo, hi], 1).astype(np.int32)).to(DEV) if siblings else None
    loss, grad = train.sibling_loss(torch.from_numpy(z).to(DEV), torch.from_numpy(label.astype(np.int32)).to(DEV), siblings=sib,
                                    weight=torch.from_numpy(w).to(DEV), scale=scale, grad_dtype=dtype)
    assert grad.dtype == dtype
    want_loss, want_grad, size = plain_loss(z.astype(np.float64), label, lo, hi, w.astype(np.float64), np.float64(np.float32(scale)))
    # exp and log1p within 2 U of their values, a handful of other operations: 8 U a term, m additions
    near(loss.cpu(), want_loss, (m + 8) * U * size, "loss")
    # the same for the sigmoid: 8 U, then the rounding to the type
    near(grad.float().cpu(), want_grad, 8 * U * np.abs(want_grad) + half_step(want_grad, dtype) * (1 + 8 * U), "grad")
    again = train.sibling_loss(torch.from_numpy(z).to(DEV), torch.from_numpy(label.astype(np.int32)).to(DEV), siblings=sib,
                               weight=torch.from_numpy(w).to(DEV), scale=scale, grad_dtype=dtype)
    assert torch.equal(loss, again[0]) and torch.equal(grad, again[1])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m, k, widest", [(700, 300, 300), (700, 301, 40), (1200, 40, 40), (1200, 41, 9), (5, 9000, 9000), (3000, 2048, 33)])
def test_loss_of_wide_ranges(m, k, widest, dtype):
    rng = np.random.default_rng(m + k)
    z = (rng.normal(size=(m, k)) * 5).astype(np.float32)
    lo = rng.integers(-3, k, m)
    hi = lo + rng.integers(0, widest + 1, m)
    inside = (np.arange(k) >= lo[:, None]) & (np.arange(k) < hi[:, None])
    z[~inside] = np.nan
    label = np.clip(lo + rng.integers(-1, widest + 1, m), -2**31, 2**31 - 1)
    sib = torch.from_numpy(np.stack([lo, hi], 1).astype(np.int32)).to(DEV)
    loss, grad = train.sibling_loss(torch.from_numpy(z).to(DEV), torch.from_numpy(label.astype(np.int32)).to(DEV), siblings=sib, grad_dtype=dtype)
    want_loss, want_grad, size = plain_loss(z.astype(np.float64), label, lo, hi, np.ones(m), 1.0)
    near(loss.cpu(), want_loss, (m + 8) * U * size, "loss")
    near(grad.float().cpu(), want_grad, 8 * U * np.abs(want_grad) + half_step(want_grad, dtype) * (1 + 8 * U), "grad")
    extreme = torch.tensor([[-2**31, 2**31 - 1], [2**31 - 1, -2**31], [2**31 - 1, 2**31 - 1], [-2**31, -2**31], [k, k + 5]], dtype=torch.int32, device=DEV)
    z = torch.from_numpy(rng.normal(size=(2000, k)).astype(np.float32)).to(DEV)
    whole = train.sibling_loss(z, torch.zeros(2000, dtype=torch.int32, device=DEV))
    sib = extreme[torch.arange(2000, device=DEV) % 5]
    part = train.sibling_loss(z, torch.zeros(2000, dtype=torch.int32, device=DEV), siblings=sib)
    assert torch.equal(part[1][::5], whole[1][::5]) and (part[1].view(400, 5, k)[:, 1:] == 0).all()


def test_loss_at_the_ends():
    """Scores far out: no overflow, and the small side keeps its digits; sibling ranges reaching outside are cut."""
    z = torch.tensor([[-math.inf, -200.0, -90.0, 0.0, 90.0, 200.0, math.inf, 3.0]], device=DEV)
    for label in (-1, 0, 3, 6, 99):
        loss, grad = train.sibling_loss(z, torch.tensor([label], dtype=torch.int32, device=DEV), siblings=torch.tensor([[-5, 100]], dtype=torch.int32, device=DEV))
        want = plain_loss(z.double().cpu().numpy(), np.array([label]), np.array([0]), np.array([8]), np.ones(1), 1.0)
        fine = np.isfinite(want[0])
        assert np.array_equal(np.isinf(loss.cpu().numpy()), ~fine)
        near(loss.cpu().numpy()[fine], want[0][fine], 16 * U * np.abs(want[0][fine]) + 2.0 ** -149)
        near(grad.cpu(), want[1], 16 * U * np.abs(want[1]) + 2.0 ** -126)
    empty = torch.tensor([[5, 2]], dtype=torch.int32, device=DEV)
    loss, grad = train.sibling_loss(torch.full((1, 8), math.nan, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), siblings=empty)
    assert (loss == 0).all() and (grad == 0).all()


@pytest.mark.parametrize("k", [12, 13])
def test_loss_strided(k):
    rng = np.random.default_rng(k)
    m = 50
    z = torch.from_numpy(rng.normal(size=(m, k + 3)).astype(np.float32)).to(DEV)
    label = torch.from_numpy(rng.integers(0, k, m).astype(np.int32)).to(DEV)
    out = (torch.full((k,), 7.0, device=DEV), torch.full((m, k + 2), 7.0, device=DEV, dtype=BF16))
    train.sibling_loss(z[:, 2:2 + k], label, out=(out[0], out[1][:, 1:1 + k]))
    want = train.sibling_loss(z[:, 2:2 + k].contiguous(), label, grad_dtype=BF16)
    assert torch.equal(out[1][:, 1:1 + k], want[1]) and (out[1][:, 0] == 7).all() and (out[1][:, -1] == 7).all()
    near(out[0].cpu(), want[0].double().cpu(), 60 * U * want[0].double().cpu().numpy())


# --------------------------------------------------------------------------------------------------------------- adamw
def plain_step(p, g, m, v, t, lr, betas, eps, decay, l1):
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    d = np.sqrt(v / (1 - betas[1] ** t)) + eps
    move = lr * m / ((1 - betas[0] ** t) * d)
    p = p * (1 - lr * decay) - move
    size = np.abs(p) + np.abs(move)
    return np.sign(p) * np.maximum(np.abs(p) - lr * l1 / d, 0), m, v, size + lr * l1 / d


SETS = [
    [((7500, 8), F32, F32), ((8,), F32, F32)],
    [((1,), F32, F32)],
    [((255,), F32, F32), ((256,), F32, F32), ((257,), F32, F32), ((1023,), F32, F32), ((1024,), F32, F32), ((1025,), F32, F32)],
    [((145, 3), BF16, F32), ((3,), F32, F32), ((33, 7), F16, F16), ((0, 4), F32, F32), ((100, 100), BF16, BF16), ((5,), F32, BF16)],
    [((301, 3 + j % 5), [F32, BF16, F16][j % 3], [F32, F32, F16, BF16][j % 4]) for j in range(300)],
]


@pytest.mark.parametrize("t", [0, 1, 99, 100000])
@pytest.mark.parametrize("which", range(len(SETS)))
def test_adamw_32(which, t):
    rng = np.random.default_rng(which)
    params, grads, values, decay, l1 = [], [], [], [], []
    for j, (shape, kind, grad_kind) in enumerate(SETS[which]):
        params.append(torch.from_numpy(rng.normal(size=shape).astype(np.float32)).to(DEV).to(kind))
        grads.append(torch.from_numpy((rng.normal(size=shape) * 0.01).astype(np.float32)).to(DEV).to(grad_kind))
        decay.append(0.1 * (j % 3))
        l1.append(0.001 * (j % 2))
    opt = train.AdamW(params, grads, lr=0.01, weight_decay=decay, l1=l1)
    m = torch.from_numpy((rng.normal(size=opt.m.shape) * 0.01).astype(np.float32)).to(DEV)
    v = torch.from_numpy((rng.random(size=opt.m.shape) * 1e-4).astype(np.float32)).to(DEV)
    if t == 0:
        m.zero_(), v.zero_()
    opt.load_state(t, m, v)
    before = [p.double().cpu().numpy() for p in params]
    opt.step()
    assert opt.steps == t + 1
    for j, p in enumerate(params):
        n, a = p.numel(), opt.state_at[j]
        g = grads[j].double().cpu().numpy().ravel()
        mj, vj = m[a:a + n].double().cpu().numpy(), v[a:a + n].double().cpu().numpy()
        want, wm, wv, size = plain_step(before[j].ravel(), g, mj, vj, t + 1, 0.01, (0.9, 0.999), 1e-8, decay[j], l1[j])
        near(opt.m[a:a + n].cpu(), wm, 3 * U * (np.abs(mj) + np.abs(g)), "m of %d" % j)
        near(opt.v[a:a + n].cpu(), wv, 4 * U * (vj + g * g), "v of %d" % j)
        # m is the difference of what may cancel: its error against the root, times lr, joins the 24 U of the update's own operations
        slack = 0.01 * 3 * U * (np.abs(mj) + np.abs(g)) / ((1 - 0.9 ** (t + 1)) * (np.sqrt(wv / (1 - 0.999 ** (t + 1))) + 1e-8))
        near(p.double().cpu().numpy().ravel(), want, 24 * U * size + slack + half_step(want, p.dtype) * (1 + 1e-4), "p of %d" % j)


def restated_rounding(x, scale, chance):
    y = (x / scale).astype(np.float32)
    a = np.abs(y)
    up = np.where(a < 2.0 ** -6, np.float32(2.0 ** -6), np.float32(0))       # below 2^-6 codes are as far apart as above it, and what is
    a = np.where(a < 2.0 ** -6, np.floor(a * np.float32(2.0 ** 29)) * np.float32(2.0 ** -29), a)      # below 2^-29 is dropped
    bits = ((a + up).view(np.uint32) + (chance << 4 | 8).astype(np.uint32)) & np.uint32(0xfff00000)
    return np.copysign(bits.view(np.float32) - up, y)


def restated_scale(x):
    top = np.maximum(np.abs(x).reshape(-1, 256).max(1), 2.0 ** -117)
    mant, exp = np.frexp(top)
    return np.ldexp(np.float32(1), exp - 9 + (mant > 0.875)).astype(np.float32)


@pytest.mark.parametrize("kind, grad_kind", [(F32, F32), (BF16, BF16), (F16, F32)])
def test_adamw_8(kind, grad_kind):
    """The codes are a function of the inputs: a 32-bit restatement gives the same ones, over several steps."""
    rng = np.random.default_rng(3)
    shapes = [(300, 7), (5,), (256,), (1024, 3), (1, 1), (1023,)]
    params = [torch.from_numpy(rng.normal(size=s).astype(np.float32)).to(DEV).to(kind) for s in shapes]
    grads = [torch.empty(s, device=DEV, dtype=grad_kind) for s in shapes]
    betas, lr = (0.9, 0.99), 0.01
    opt = train.AdamW(params, grads, lr=lr, betas=betas, state_bits=8)
    f32 = np.float32
    total = opt.state_values
    codes_m, codes_v = np.zeros(total, f32), np.zeros(total, f32)
    scale_m, scale_v = np.ones(total // 256, f32), np.ones(total // 256, f32)
    for t in range(1, 6):
        flat = np.zeros(total, f32)
        for j, g in enumerate(grads):
            g.copy_(torch.from_numpy((rng.normal(size=shapes[j]) * np.exp(3 * rng.normal(size=shapes[j]))).astype(f32)))
            flat[opt.state_at[j]:opt.state_at[j] + g.numel()] = g.float().cpu().numpy().ravel()
        before = [p.double().cpu().numpy().ravel() for p in params]
        opt.step()
        m = codes_m * np.repeat(scale_m, 256)
        v = codes_v * np.repeat(scale_v, 256)
        v = v * v
        m = m * f32(betas[0]) + flat * f32(1 - betas[0])
        v = v * f32(betas[1]) + (flat * flat) * f32(1 - betas[1])
        root = np.sqrt(v)
        scale_m, scale_v = restated_scale(m), restated_scale(root)
        x = (np.arange(total, dtype=np.uint64) ^ np.uint64(t * 0x9E3779B9 & 0xffffffff)) & np.uint64(0xffffffff)
        x = (x ^ x >> np.uint64(16)) * np.uint64(0x7FEB352D) & np.uint64(0xffffffff)
        x = (x ^ x >> np.uint64(15)) * np.uint64(0x846CA68B) & np.uint64(0xffffffff)
        x = (x ^ x >> np.uint64(16)).astype(np.uint32)
        codes_m = restated_rounding(m, np.repeat(scale_m, 256), x >> np.uint32(16))
        codes_v = restated_rounding(root, np.repeat(scale_v, 256), x & np.uint32(0xffff))
        codes_v = np.where((root > 0) & (codes_v == 0), f32(2.0 ** -9), codes_v).astype(f32)
        assert np.array_equal(opt.m_scale.cpu().numpy(), scale_m) and np.array_equal(opt.v_scale.cpu().numpy(), scale_v), t
        assert np.array_equal(opt.m.float().cpu().numpy(), codes_m), t
        assert np.array_equal(opt.v.float().cpu().numpy(), codes_v), t
        # a code is at most one step from what it stands for: 1/8 of the value, or 2^-9 of the scale
        deq = codes_v * np.repeat(scale_v, 256)
        assert (np.abs(deq - root) <= np.maximum(root / 8, np.repeat(scale_v, 256) * 2.0 ** -9) * 1.0001).all()
        for j, p in enumerate(params):
            a, n = opt.state_at[j], p.numel()
            d = root[a:a + n] / math.sqrt(1 - betas[1] ** t) + 1e-8
            move = lr * m[a:a + n].astype(np.float64) / ((1 - betas[0] ** t) * d)
            want = before[j] - move
            near(p.double().cpu().numpy().ravel(), want, 24 * U * (np.abs(want) + np.abs(move)) + half_step(want, kind) * (1 + 1e-4), "p of %d" % j)


def test_adamw_8_moves_on_the_mean():
    """Without gradients the root of the second moment decays by sqrt(beta2) a step on the mean, although every step is far below half a code."""
    n = 1 << 18
    p, g = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    opt = train.AdamW([p], [g], state_bits=8)
    root = 100.0 + 100.0 * torch.rand(n, device=DEV)
    opt.load_state(0, torch.zeros(n, device=DEV).to(torch.float8_e4m3fn), root.to(torch.float8_e4m3fn), torch.ones(n // 256, device=DEV), torch.ones(n // 256, device=DEV))
    start = (opt.v.float() * opt.v_scale.repeat_interleave(256)).double()
    steps = 100
    for _ in range(steps):
        opt.step()
    end = (opt.v.float() * opt.v_scale.repeat_interleave(256)).double()
    want = 0.999 ** (steps / 2)
    # the sum of `steps` roundings of one value, each at most one step of 2^-3, is a bounded walk: a value strays by less than
    # sqrt(steps) / 8 of itself (one deviation), the mean of n of them by sqrt(n) less; five deviations
    assert abs(float(end.mean() / start.mean()) - want) < 5 * math.sqrt(steps) / 8 / math.sqrt(n)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_takes_nan_and_infinities_one_by_one(bits):
    n = 2000
    p, g = torch.zeros(n, device=DEV), torch.ones(n, device=DEV)
    g[700], g[1300], g[1999] = math.nan, math.inf, 0.0
    opt = train.AdamW([p], [g], lr=0.1, state_bits=bits)
    opt.step()
    opt.step()
    bad = ~torch.isfinite(p)
    assert bad.nonzero().flatten().tolist() == [700, 1300] and p[1999] == 0
    # 8 bits: m and the root are off by 1/8 of themselves at most in the second step
    near(p[:700].cpu(), np.full(700, -0.2), 1e-3 if bits == 32 else 0.1 * (9 / 7 - 1) + 1e-3)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_where_the_second_moment_overflows(bits):
    """A finite gradient whose square is not: the value stands still with 32 bits, and is NaN from the second step on with 8."""
    p, g = torch.ones(300, device=DEV), torch.ones(300, device=DEV)
    g[7] = 1e30
    opt = train.AdamW([p], [g], lr=0.125, state_bits=bits)
    opt.step()
    assert torch.isfinite(p).all() and p[7] == 1
    opt.step()
    assert p[7] == 1 if bits == 32 else torch.isnan(p[7])
    assert torch.isfinite(p[:7]).all() and torch.isfinite(p[8:]).all() and torch.isinf(opt.v[7]) if bits == 32 else torch.isnan(opt.v.float()[7])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("gradient", [1e30, math.inf, math.nan])
def test_what_overflows_leaves_its_neighbours_alone(gradient, bits):
    """The 255 values that share scales with one whose moments are infinite or NaN, and those of other blocks, stay finite; so do their states."""
    p, g = torch.ones(600, device=DEV), torch.ones(600, device=DEV)
    g[300] = gradient
    opt = train.AdamW([p], [g], lr=0.125, state_bits=bits)
    others = torch.arange(600, device=DEV) != 300
    for _ in range(3):
        opt.step()
        assert torch.isfinite(p[others]).all() and torch.isfinite(opt.m[:600].float()[others]).all() and torch.isfinite(opt.v[:600].float()[others]).all()
        assert not torch.isfinite(opt.v[300].float())
        if bits == 8:
            assert torch.isfinite(opt.m_scale).all() and torch.isfinite(opt.v_scale).all()
    # A block of its own moves by lr a step.  8 bits: a code is off by 1/8 of itself at most, so m enters the second step with 0.9 * 0.1 / 8 of 0.19 = 6 %
    # and the third with 0.9 * 0.19 * (1.06 * 1.125 - 1) of 0.271 = 12 %, the root with -6.0 to 6.4 and -11.5 to 13.5 %: steps off by 13 and 27 % at most
    near(p[:256].cpu(), np.full(256, 1 - 3 * 0.125), 1e-5 if bits == 32 else 0.125 * (0.13 + 0.27))


def small_gradients(rng, n_blocks=14):
    """Blocks of 256 gradients of about 1e-23, 3e-23 .. 3e-17, and one block of all of these sizes."""
    size = np.repeat(10.0 ** (-23 + 0.5 * np.arange(n_blocks - 1)), 256)
    size = np.concatenate([size, rng.permutation(size)[:256]])
    return (size * rng.uniform(0.3, 1, size.size) * rng.choice([-1.0, 1.0], size.size)).astype(np.float32)


def root_range(v, operations):
    """Between what the root lies of v made in 32 bits by this many operations: each is off by U of v, or by 2^-150 where it has less than 24 bits."""
    off = operations * (U * v + 2.0 ** -150)
    return np.sqrt(np.maximum(v - off, 0)) * (1 - 2 * U), np.sqrt(v + off) * (1 + 2 * U)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_where_the_second_moment_is_below_the_normal_numbers(bits):
    """Second moments of 1e-49 to 1e-37, where numbers of 32 bits end at 1.4e-45 and have all their bits from 1.2e-38 on: two steps."""
    rng = np.random.default_rng(23)
    g = small_gradients(rng)
    d_g, p = torch.from_numpy(g).to(DEV), torch.zeros(g.size, device=DEV)
    opt = train.AdamW([p], [d_g], lr=0.1, eps=1e-8, state_bits=bits)

    def held():
        if bits == 32:
            return opt.m.double().cpu().numpy(), opt.v.double().sqrt().cpu().numpy()
        return tuple((x.double().view(-1, 256) * s.double().unsqueeze(1)).flatten().cpu().numpy() for x, s in ((opt.m, opt.m_scale), (opt.v, opt.v_scale)))

    g = g.astype(np.float64)
    for t in (1, 2):
        before, start = held(), p.double().cpu().numpy()
        opt.step()
        if t == 1:
            d_g.mul_(0.5)
        m, v = before[0] * 0.9 + g * 0.1, before[1] ** 2 * 0.999 + g * g * 0.001
        lo, hi = root_range(v, 6)
        # roots are off by sqrt(6 * 2^-150) = 7e-23 at most, which makes 2e-13 of d; 16 operations and constants of 32 bits
        want = start - 0.1 * m / ((1 - 0.9 ** t) * (np.sqrt(v / (1 - 0.999 ** t)) + 1e-8))
        near(p.cpu(), want, 16 * U * (np.abs(start) + np.abs(want - start)) + 1e-12 * np.abs(want - start))
        after = held()
        if bits == 32:
            near(after[0], m, 4 * U * (np.abs(before[0]) + np.abs(g)))
            assert (after[1] >= lo).all() and (after[1] <= hi).all()
        else:      # a code is off by less than one step of its own: 2^-3 of it, 2^-9 scales at least
            for got, low, high, scale in ((np.abs(after[0]), np.abs(m) * (1 - 4 * U), np.abs(m) * (1 + 4 * U), opt.m_scale), (after[1], lo, hi, opt.v_scale)):
                s = np.repeat(scale.double().cpu().numpy(), 256)
                assert (got >= low - np.maximum(low / 8, s / 512)).all() and (got <= high + np.maximum(high / 8, s / 512)).all()
        g = g * 0.5


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_steps_by_lr_where_the_second_moment_is_below_the_normal_numbers(bits):
    """A first step without eps moves a value by lr, however small its gradient."""
    rng = np.random.default_rng(24)
    g = (10.0 ** rng.uniform(-20, -17, 3000) * rng.choice([-1.0, 1.0], 3000)).astype(np.float32)
    p = torch.zeros(3000, device=DEV)
    train.AdamW([p], [torch.from_numpy(g).to(DEV)], lr=0.125, eps=0.0, state_bits=bits).step()
    v = g.astype(np.float64) ** 2 * 0.001
    lo, hi = root_range(v, 4)
    near(p.cpu(), -0.125 * np.sign(g), 0.125 * (np.maximum(np.sqrt(v) / lo, hi / np.sqrt(v)) - 1 + 16 * U))


def test_a_fit_with_8_bit_states_stays_finite():
    """Rows scored far from 0 leave tokens that they meet first with gradients of 1e-21 to 1e-18."""
    rng = np.random.default_rng(25)
    bits, _, label = problem(rng, n=1024, ncol=1500, k=8)
    for steps, k, batch in ((8, 8, 256), (40, 4, 64)):
        assert np.isfinite(train.fit_siblings(bits, label, k, 7500, steps=steps, batch=batch, l1=1e-4, state_bits=8)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_at_odd_addresses(bits):
    """Tensors at addresses that no vector load may use, and what lies around them."""
    rng = np.random.default_rng(1)
    for kind in (F32, BF16, F16):
        buffers = [torch.full((3000,), 7.0, device=DEV).to(kind) for _ in range(2)]
        p, g = buffers[0][1:2002], buffers[1][3:2004]
        p.copy_(torch.from_numpy(rng.normal(size=2001).astype(np.float32)))
        g.copy_(torch.from_numpy(rng.normal(size=2001).astype(np.float32)))
        q, h = p.clone(), g.clone()
        a, b = (train.AdamW([x], [y], lr=0.01, l1=0.1, state_bits=bits) for x, y in ((p, g), (q, h)))
        for _ in range(2):
            a.step()
            b.step()
        assert torch.equal(p, q) and torch.equal(a.m.view(torch.uint8), b.m.view(torch.uint8)) and torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))
        assert buffers[0][0] == 7 and (buffers[0][2002:] == 7).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_counts_a_step_of_nothing(bits):
    empty, one = torch.zeros((0, 5), device=DEV), torch.tensor(1.0, device=DEV)
    opt = train.AdamW([empty], [empty.clone()], state_bits=bits)
    opt.step(), opt.step()
    assert opt.steps == 2
    opt = train.AdamW([empty, one], [empty.clone(), torch.tensor(2.0, device=DEV)], lr=0.25, state_bits=bits)      # a tensor of no dimensions has one value
    opt.step(), opt.step()
    assert opt.steps == 2 and abs(float(one) - 0.5) < (1e-5 if bits == 32 else 0.25 / 4)      # the moments are off by 1/8 at most in the second step


def test_parameters_and_unsigned_words():
    """Parameters that require gradients are tensors like others (nothing is recorded), and so are rows of uint32 words."""
    rng = np.random.default_rng(8)
    for n in (1, 700):
        bits, _ = packed(rng, n, 300)
        table = torch.from_numpy(rng.normal(size=(300, 40)).astype(np.float32)).to(DEV)
        bias = torch.ones(40, device=DEV)
        want = train.row_scores(bits, table, bias)
        got = train.row_scores(bits.view(torch.uint32), torch.nn.Parameter(table), torch.nn.Parameter(bias))
        assert torch.equal(got, want) and not got.requires_grad
        assert torch.equal(train.row_scores_grad(bits.view(torch.uint32), want, 300)[0], train.row_scores_grad(bits, want, 300)[0])
    p = torch.nn.Parameter(torch.ones(10, device=DEV))
    train.AdamW([p], [torch.ones(10, device=DEV)], lr=0.5).step()
    assert (p - 0.5).abs().max() < 1e-5


def test_adamw_refuses_shared_memory():
    x, y = torch.zeros(100, device=DEV), torch.zeros(100, device=DEV)
    with pytest.raises(ValueError, match=r"params\[0\] and params\[1\] share memory"):
        train.AdamW([x[:60], x[50:]], [y[:60], y[50:]])
    with pytest.raises(ValueError, match="share memory"):
        train.AdamW([x[:50]], [x[20:70]])
    train.AdamW([x[:50], x[50:]], [y[:50], y[:50]])          # gradients may be shared
    opt = train.AdamW([x], [y])
    with pytest.raises(ValueError, match="states of 32 bits have none"):
        opt.load_state(0, opt.m, opt.v, opt.m, opt.v)
    with pytest.raises(ValueError, match="values: 256 are wanted"):
        opt.load_state(0, opt.m[:100], opt.v)


def test_an_empty_batch_of_a_large_table():
    """More values than a launch has threads: a gradient of nothing is zeros everywhere."""
    bits = torch.zeros((0, 2188), dtype=torch.int32, device=DEV)
    out = torch.empty((70_000, 65_536), device=DEV).fill_(7.0), torch.full((65_536,), 7.0, device=DEV)
    train.row_scores_grad(bits, torch.zeros((0, 65_536), device=DEV), 70_000, out=out)
    assert not any(bool(out[0][i:i + 7_000].any()) for i in range(0, 70_000, 7_000)) and not out[1].any()


def test_more_features_than_32_bits_count_are_refused():
    """2^32 + 5 features, which is 5 in 32 bits."""
    bits = torch.zeros((1, 2**27 + 4), dtype=torch.int32, device=DEV)
    held = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="sizes of 2"):
        train.row_scores_grad(bits, torch.ones((1, 1), device=DEV), 2**32 + 5)
    assert torch.cuda.memory_allocated() < held + 2**20


def test_contiguous_rows_at_odd_addresses_are_refused():
    """With the same error as rows that are not contiguous."""
    flat = torch.zeros(41, dtype=torch.int32, device=DEV)
    for bits in (flat[1:].view(10, 4), flat[1:33].view(4, 8)[:, :4]):
        with pytest.raises(ValueError, match="aligned 16-byte units"):
            train.row_scores(bits, torch.ones((100, 3), device=DEV))
        with pytest.raises(ValueError, match="aligned 16-byte units"):
            train.row_scores_grad(bits, torch.ones((bits.shape[0], 3), device=DEV), 100)


def test_outputs_over_inputs_are_refused():
    bits, _ = packed(np.random.default_rng(0), 50, 300)
    buffer = torch.zeros(400, 40, device=DEV)
    label = torch.zeros(50, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="out and table share memory"):
        train.row_scores(bits, buffer[:300, :8], out=buffer[:50, 4:12])
    with pytest.raises(ValueError, match=r"out\[1\] and scores share memory"):
        train.sibling_loss(buffer[:50, :8], label, out=(torch.zeros(8, device=DEV), buffer[:50, :8]))
    with pytest.raises(ValueError, match=r"out\[0\] and grad share memory"):
        train.row_scores_grad(bits, buffer[:50, :8], 300, out=(buffer[:300, :8], torch.zeros(8, device=DEV)))
    buffer[:, :8] = 1
    scores = train.row_scores(bits, buffer[:300, :8], out=buffer[:50, 8:16])         # columns beside one another
    assert torch.equal(scores, train.row_scores(bits, torch.ones(300, 8, device=DEV))) and (buffer[:, :8] == 1).all() and (buffer[:, 16:] == 0).all()


def test_an_optimizer_keeps_its_tensors():
    """Its addresses stay valid whatever the caller does to the lists it was made from."""
    params, grads = [torch.ones(1000, device=DEV)], [torch.ones(1000, device=DEV)]
    opt = train.AdamW(params, grads, lr=0.25)
    del params[0], grads[0]
    opt.step()
    assert isinstance(opt.params, tuple) and (opt.params[0] - 0.75).abs().max() < 1e-6


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("move", [
    lambda x: setattr(x, "data", torch.ones(1000, device=DEV)), lambda x: x.set_(torch.ones(1000, device=DEV)), lambda x: x.resize_(100_000),
    lambda x: x.untyped_storage().resize_(0), lambda x: setattr(x, "data", x.data.to(BF16))])
def test_an_optimizer_whose_tensors_moved_does_not_step(move, bits):
    """Memory that was given back may be another tensor's."""
    for which in range(4):
        params, grads = [torch.ones(1000, device=DEV) for _ in range(2)], [torch.ones(1000, device=DEV) for _ in range(2)]
        opt = train.AdamW(params, grads, lr=0.25, state_bits=bits)
        opt.step()
        steps = opt.steps
        move((params + grads)[which])
        with pytest.raises(ValueError, match=r"%s\[%d\] has other memory" % ("params" if which < 2 else "grads", which % 2)):
            opt.step()
        assert opt.steps == steps


@pytest.mark.parametrize("bits", [32, 8])
def test_states_are_not_taken_away(bits):
    p, q = torch.ones(1000, device=DEV), torch.ones(1000, device=DEV)
    opt, other = (train.AdamW([x], [torch.ones(1000, device=DEV)], lr=0.25, state_bits=bits) for x in (p, q))
    for name in ("m", "v") + (("m_scale", "v_scale") if bits == 8 else ()):
        with pytest.raises(RuntimeError, match="not resizable"):
            getattr(opt, name).untyped_storage().resize_(0)
    opt.step(), other.step()
    assert all(torch.equal(getattr(opt, x).view(torch.uint8), getattr(other, x).view(torch.uint8)) for x in ("m", "v"))
    assert (opt.m[:1000].float() != 0).all()
    opt.m.data = zeros = torch.zeros_like(opt.m)
    opt.step(), other.step()
    assert torch.equal(p, q) and not zeros.float().any()


def test_an_optimizer_keeps_the_memory_of_views():
    """A view that is given other memory is not followed; the memory it had stays the optimizer's while that lives."""
    flat, grad = torch.ones(2000, device=DEV), torch.ones(2000, device=DEV)
    views = [flat[:1000], flat[1000:]]
    opt = train.AdamW(views, [grad[:1000], grad[1000:]], lr=0.25)
    at = flat.data_ptr()
    views[1].data = new = torch.ones(1000, device=DEV)
    del flat
    others = [torch.ones(2000, device=DEV) for _ in range(50)]
    opt.step()
    assert views[0].data_ptr() == at and (views[0] - 0.75).abs().max() < 1e-6
    assert (new == 1).all() and all(x.data_ptr() != at and (x == 1).all() for x in others)


# ------------------------------------------------------------------------------------------------------ used together
def problem(rng, n=400, ncol=60, k=6):
    consensus = rng.integers(1, 5, (k, ncol))
    label = rng.integers(0, k, n).astype(np.int32)
    sym = np.where(rng.random((n, ncol)) < 0.1, rng.integers(0, 5, (n, ncol)), consensus[label])
    words = -(-5 * ncol // 128) * 4
    x = np.zeros((n, words * 32), bool)
    x[np.arange(n)[:, None], 5 * np.arange(ncol) + sym] = True
    bits = np.packbits(x, axis=1, bitorder="little").view(np.int32).reshape(n, words)
    return torch.from_numpy(bits.copy()).to(DEV), x[:, :5 * ncol].astype(np.float64), label


def test_steps_equal_the_formulas():
    """Three steps of scores, loss, gradient and AdamW on a padded batch against the same in 64 bits; the gradient also against differences."""
    rng = np.random.default_rng(11)
    bits, x, label = problem(rng)
    n, (f, k) = len(x), (x.shape[1], 6)
    rows = np.concatenate([rng.permutation(n)[:250], np.full(6, -1)]).astype(np.int32)
    y = label[np.where(rows < 0, 0, rows)]
    sib = np.stack([np.where(rows < 0, 0, 0), np.where(rows < 0, 0, k)], 1).astype(np.int32)       # padding trains nothing
    table, bias = torch.from_numpy(rng.normal(size=(f, k)).astype(np.float32) * 0.1).to(DEV), torch.zeros(k, device=DEV)
    grads = (torch.empty_like(table), torch.empty_like(bias))
    opt = train.AdamW([table, bias], grads, lr=0.05, eps=1e-3, weight_decay=[0.01, 0.0], l1=[1e-4, 0.0])
    xb, real = picked(x, rows)
    T, b = table.double().cpu().numpy(), bias.double().cpu().numpy()
    state = [[np.zeros_like(T), np.zeros_like(T)], [np.zeros_like(b), np.zeros_like(b)]]
    d = [torch.from_numpy(a).to(DEV) for a in (rows, y.astype(np.int32), sib)]

    def total(T, b):
        return plain_loss(np.where(real[:, None], xb @ T + b, 0.0), y, sib[:, 0], sib[:, 1], np.ones(len(rows)), 1 / 250)[0].sum()

    for t in range(1, 4):
        scores = train.row_scores(bits, table, bias, rows=d[0])
        loss, g = train.sibling_loss(scores, d[1], siblings=d[2], scale=1 / 250)
        train.row_scores_grad(bits, g, f, rows=d[0], out=grads)
        z = np.where(real[:, None], xb @ T + b, 0.0)
        want_loss, want_g, _ = plain_loss(z, y, sib[:, 0], sib[:, 1], np.ones(len(rows)), 1 / 250)
        # after a step the tables differ by the errors of the steps before, which an eps of 1e-3 keeps below 1e-5 of the update
        near(loss.cpu(), want_loss, 1e-4 * want_loss)
        gT, gb = xb.T @ want_g, want_g.sum(0)
        near(grads[0].cpu(), gT, 1e-5 + 1e-4 * np.abs(gT))
        near(grads[1].cpu(), gb, 1e-5 + 1e-4 * np.abs(gb))
        if t == 1:
            for _ in range(3):
                D, e, h = rng.normal(size=T.shape), rng.normal(size=b.shape), 1e-5
                slope = (total(T + h * D, b + h * e) - total(T - h * D, b - h * e)) / (2 * h)
                mine = (grads[0].double().cpu().numpy() * D).sum() + (grads[1].double().cpu().numpy() * e).sum()
                assert abs(mine - slope) <= 1e-5 * (np.abs(gT * D).sum() + np.abs(gb * e).sum())
        opt.step()
        T, *state[0] = plain_step(T, gT, *state[0], t, 0.05, (0.9, 0.999), 1e-3, 0.01, 1e-4)[:3]
        b, *state[1] = plain_step(b, gb, *state[1], t, 0.05, (0.9, 0.999), 1e-3, 0.0, 0.0)[:3]
        near(table.cpu(), T, 1e-4)
        near(bias.cpu(), b, 1e-4)


@pytest.mark.parametrize("bits_", [32, 8])
def test_a_captured_training_step_counts_on(bits_):
    """A whole step recorded into a HIP graph and replayed, with eager work of the same kind between the replays: each replay is the eager step."""
    rng = np.random.default_rng(2)
    bits, x, label = problem(rng, n=700, ncol=150, k=9)
    f, k = x.shape[1], 9
    start = torch.from_numpy(rng.normal(size=(f, k)).astype(np.float32) * 0.1).to(DEV)

    def program():
        table, bias = start.clone(), torch.zeros(k, device=DEV)
        grads = (torch.empty_like(table), torch.empty_like(bias))
        rows, lab = torch.zeros(600, dtype=torch.int32, device=DEV), torch.zeros(600, dtype=torch.int32, device=DEV)
        opt = train.AdamW([table, bias], grads, lr=0.01, state_bits=bits_)

        def step():
            scores = train.row_scores(bits, table, bias, rows=rows)
            loss, g = train.sibling_loss(scores, lab, scale=1 / 600, grad_dtype=BF16)
            train.row_scores_grad(bits, g, f, rows=rows, out=grads)
            opt.step()
            return loss, scores

        return table, bias, rows, lab, opt, step

    eager, graphed, other = program(), program(), program()
    program()[5]()                                           # the first call of a kernel loads its code
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    for prog in (graphed, other):                            # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = prog[5]()
        graphs.append((graph, out))
    torch.cuda.synchronize()
    for t in range(5):
        pick = rng.integers(0, 700, 600).astype(np.int32)
        for prog in (eager, graphed, other):
            prog[2].copy_(torch.from_numpy(pick))
            prog[3].copy_(torch.from_numpy(label[pick]))
        loss, scores = eager[5]()
        graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize()
        for prog, (_, out) in zip((graphed, other), graphs):
            assert torch.equal(out[0], loss) and torch.equal(out[1], scores), t
            assert torch.equal(prog[0], eager[0]) and torch.equal(prog[1], eager[1]), t
            assert torch.equal(prog[4].m.view(torch.uint8), eager[4].m.view(torch.uint8)) and prog[4].steps == t + 1


def test_on_two_streams_at_once():
    rng = np.random.default_rng(8)
    bits, x = packed(rng, 900, 1500)
    tables = [torch.from_numpy(rng.normal(size=(1500, k)).astype(np.float32)).to(DEV) for k in (9, 150)]
    grads = [torch.from_numpy(rng.normal(size=(900, k)).astype(np.float32)).to(DEV) for k in (9, 150)]
    want = [(train.row_scores(bits, t), train.row_scores_grad(bits, g, 1500)[0]) for t, g in zip(tables, grads)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in tables]
    got = [[], []]
    for _ in range(10):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append((train.row_scores(bits, tables[j]), train.row_scores_grad(bits, grads[j], 1500)[0]))
    torch.cuda.synchronize()
    for j in range(2):
        for a, b in got[j]:
            assert torch.equal(a, want[j][0]) and torch.equal(b, want[j][1])


def test_labels_of_64_bits():
    """A label that is no sibling stays none, also where 32 bits of it would be one; so is a row of uint32 words a tensor."""
    bits, _, label = problem(np.random.default_rng(6))
    label = label.astype(np.int64)
    out = np.where(np.arange(400) % 3 == 0, label + 2**32, label)
    want = train.fit_siblings(bits, np.where(np.arange(400) % 3 == 0, -1, label), 6, 300, steps=3)
    assert np.array_equal(train.fit_siblings(bits, out, 6, 300, steps=3), want)
    assert np.array_equal(train.fit_siblings(bits.cpu().numpy().view(np.uint32), out, 6, 300, steps=3, batch=1000), want)


def test_fit_siblings_feeds_the_walk():
    """fit_siblings on rows of the package's own encoder gives coefficients that its database takes and classifies with; its first step is the formula's."""
    from stag_amd.engine import Database
    rng = np.random.default_rng(4)
    ncol, k, n = 60, 4, 240
    consensus = rng.integers(0, 4, (k, ncol))
    label = rng.integers(0, k, n)
    sym = np.where(rng.random((n, ncol)) < 0.05, rng.integers(0, 4, (n, ncol)), consensus[label])
    reads = ["".join(r) for r in np.array(list("ACGT"))[sym]]
    names = ["a", "b", "c", "d"]
    taxonomy = {"tree_root": names, **{x: [] for x in names}}
    rank = {"0": np.array([0.0, 1.0])}
    with Database.from_dicts(taxonomy, rank, {x: np.zeros(1 + 5 * ncol) for x in names}, n_features=5 * ncol) as db:
        bits = db.encode_a2m(reads)[0]
    x = np.unpackbits(bits.view(np.uint8), axis=1, bitorder="little")[:, :5 * ncol].astype(np.float64)
    one = train.fit_siblings(bits, label, k, 5 * ncol, steps=1, lr=0.1)
    g = (0.5 - (label[:, None] == np.arange(k))) / n
    full = np.concatenate([g.sum(0)[:, None], (x.T @ g).T], 1)
    assert one.shape == (k, 1 + 5 * ncol) and one.dtype == np.float64
    # the first step moves by lr g / (|g| + eps); a token that no row or every class has alike has a gradient of 0, or one that is rounding
    sure = np.abs(full) > 1e-6
    near(one[sure], (-0.1 * full / (np.abs(full) + 1e-8))[sure], 1e-3)
    for options in (dict(steps=30, lr=0.05, l1=1e-3), dict(steps=30, batch=64, table_dtype=BF16, state_bits=8, weight=np.ones(n, np.float32))):
        coefficients = train.fit_siblings(bits, label, k, 5 * ncol, **options)
        assert np.isfinite(coefficients).all()
        with Database.from_dicts(taxonomy, rank, dict(zip(names, coefficients)), n_features=5 * ncol) as db:
            res = db.classify_a2m(reads)
        scores = x @ coefficients[:, 1:].T + coefficients[:, 0]
        assert (res.status == 0).all()
        got = np.array([names.index(db.names[j]) for j in res.path_node[:, 0]])
        assert np.array_equal(got, scores.argmax(1))           # the walk answers with what was learned
