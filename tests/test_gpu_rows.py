"""The operators over rows of scores (accb_top_rows, accb_sample_rows, accb_distill_rows[_backward]) against their
definitions in 64 bits (rows_reference.py).

Tolerances.  Values and indices are exact.  A log-sum-exp is m / T + log(sum): the sum's terms carry the error of a
32-bit exponential (exponent |y| <= 150 rounded to 2^-24 of itself and a base-2 exponential good to 2 units in the last place), which
is at most 150 * ln 2 * 2^-24 + 2^-22 < 1e-5 for one term; terms that far down weigh nothing, and for the terms that
count (|y| <= 20) it is 20 * ln 2 * 2^-24 + 2^-22 + 64 * 2^-24 (a thread's running sum of at most 128 terms, each
addition half a step) < 6e-6.  The result is rounded once, 2^-24 of itself.  A loss of weight w inherits sum p = 1
times that.  A gradient entry is w / T times (sum p + r) q - p or (sum p + r - r / q_r) q: q and 1 / q_r are within the
same 6e-6 of themselves plus 2^-22, the rest is computed in 64 bits and rounded once; so every part is off by at most
twice 6e-6 of itself, and the whole is rounded to the element type."""
import os
import subprocess
import sys
import threading

import numpy as np
import pytest

from rows_reference import clean, distill, sample, top

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

TYPES = ["float32", "float16", "bfloat16"]
EPS = {"float32": 2.0**-24, "float16": 2.0**-11, "bfloat16": 2.0**-8}
SUM_ERROR = 6e-6


def scores(torch, rng, rows, cols, kind, pitch=None, offset=0, spread=2.0, peaks=True):
    """Rows of scores in memory of their own: `pitch` elements apart, the first one `offset` elements into it."""
    x = rng.normal(0, spread, (rows, cols)).astype(np.float32)
    if peaks and cols > 4:
        for r in range(rows):
            at = rng.choice(cols, min(8, cols), replace=False)
            x[r, at] = rng.uniform(4, 14, at.size)
    return place(torch, x, kind, pitch, offset)


def place(torch, x, kind, pitch=None, offset=0):
    rows, cols = x.shape
    pitch = pitch or cols
    memory = torch.full((offset + rows * pitch + 64,), 77.0, dtype=getattr(torch, kind), device="cuda")
    view = memory[offset:].as_strided((rows, cols), (pitch, 1), storage_offset=offset)
    view.copy_(torch.from_numpy(x))
    return view


def numbers(t):
    return t.double().cpu().numpy()


# ------------------------------------------------------------------ top
def run_top(ctx, torch, x, k, temperature=1.0, lse=True):
    rows = x.shape[0]
    values = torch.full((rows, k), 7.0, dtype=x.dtype, device="cuda")
    index = torch.full((rows, k), -7, dtype=torch.int32, device="cuda")
    out = torch.full((rows,), 7.0, device="cuda") if lse else None
    ctx.top_rows(x, values, index, lse=out, temperature=temperature)
    ctx.sync()
    return numbers(values), index.cpu().numpy(), numbers(out) if lse else None


def check_top(ctx, torch, x, k, temperature=1.0, every=1):
    values, index, lse = run_top(ctx, torch, x, k, temperature)
    for r in range(0, x.shape[0], every):
        row = numbers(x[r])
        v, i, s = top(row, k, temperature)
        assert np.array_equal(values[r], v), (r, values[r], v)
        assert np.array_equal(index[r], i), (r, index[r], i)
        assert lse[r] == s or abs(lse[r] - s) <= SUM_ERROR + 2.0**-24 * abs(s), (r, lse[r], s)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (2, 33, 33), (4, 1000, 50), (2, 1024, 1024), (3, 4099, 1000),
                                         (2, 32768, 64), (5, 50257, 20), (1, 131072, 1024), (2, 151001, 7)])
def test_top(ctx, torch_cuda, rng, kind, rows, cols, k):
    check_top(ctx, torch_cuda, scores(torch_cuda, rng, rows, cols, kind), k, 1.0 if k % 2 else 2.5)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("offset,pitch", [(1, 1013), (3, 1001), (7, 1024), (8, 1009), (0, 1003)])
def test_top_of_rows_anywhere(ctx, torch_cuda, rng, kind, offset, pitch):
    check_top(ctx, torch_cuda, scores(torch_cuda, rng, 9, 1001, kind, pitch, offset), 17)


def test_top_of_rows_too_long_for_shared_memory(ctx, torch_cuda, rng):
    check_top(ctx, torch_cuda, scores(torch_cuda, rng, 2, (1 << 20) - 3, "float32", (1 << 20) + 5, 1), 300)


@pytest.mark.parametrize("kind", TYPES)
def test_top_settles_ties_by_index(ctx, torch_cuda, rng, kind):
    t = torch_cuda
    x = rng.integers(-3, 4, (6, 5000)).astype(np.float32)
    x[0] = 0.0
    x[1] = np.where(rng.random(5000) < 0.5, 0.0, -0.0)  # equal values
    x[2, ::3] = -0.0
    for k in (1, 2, 100, 1024):
        check_top(ctx, t, place(t, x, kind), k)


@pytest.mark.parametrize("kind", TYPES)
def test_top_of_rows_with_little_in_them(ctx, torch_cuda, rng, kind):
    t = torch_cuda
    x = rng.normal(0, 1, (8, 3000)).astype(np.float32)
    x[0] = -np.inf
    x[1, 5:] = -np.inf
    x[2] = np.nan
    x[3, ::2] = np.nan
    x[4] = np.finfo(np.float32).min if kind == "float32" else float(t.finfo(getattr(t, kind)).min)
    x[5, 7] = np.inf
    x[6, 1:] = -np.inf
    x[7] = np.nan
    x[7, 2999] = -1.0
    values, index, lse = run_top(ctx, t, place(t, x, kind), 40)
    for r, row in enumerate(numbers(place(t, x, kind))):
        v, i, s = top(row, 40, 1.0)
        assert np.array_equal(values[r], v) and np.array_equal(index[r], i), r
        if r != 5:  # an infinite score: inf - inf in the reference's formula
            assert lse[r] == s or abs(lse[r] - s) <= SUM_ERROR + 2.0**-24 * abs(s)
    assert lse[5] == np.inf


@pytest.mark.parametrize("kind,cols", [("bfloat16", 150000), ("float16", 149993), ("float32", 75000)])
@pytest.mark.parametrize("k", [600, 1000, 1024])
def test_top_of_rows_held_by_five_blocks(ctx, torch_cuda, rng, kind, cols, k):
    """A list in parts of odd length, and so many large entries at the row's start that they do not fit a part."""
    x = rng.normal(0, 2, (60, cols)).astype(np.float32)
    x[:, :1500] = rng.uniform(8, 12, (60, 1500))
    x[:, :4] = rng.uniform(13, 14, (60, 4))
    check_top(ctx, torch_cuda, place(torch_cuda, x, kind), k, every=29)


@pytest.mark.parametrize("rows,cols,k", [(1500, 3001, 30), (1300, 1000, 200)])
def test_top_many_rows(ctx, torch_cuda, rng, rows, cols, k):
    """More rows than the GPU holds at a time, rows whose candidates fit a list and others side by side."""
    x = rng.normal(0, 2, (rows, cols)).astype(np.float32)
    x[::3] = np.round(x[::3])  # ties
    x[5::7, :cols // 2] += 9.0
    x[4] = -np.inf
    x[9, 3:] = np.nan
    check_top(ctx, torch_cuda, place(torch_cuda, x, "bfloat16", cols + 1, 1), k)


# --------------------------------------------------------------- sampling
def settings(torch, rows, **values):
    kinds = dict(temperature=torch.float32, top_p=torch.float32, min_p=torch.float32, top_k=torch.int32, uniform=torch.float32)
    return {k: torch.as_tensor(np.broadcast_to(np.asarray(v), (rows,)).copy()).to(kinds[k]).cuda() for k, v in values.items() if v is not None}


def bits_of(torch, allowed):
    rows, cols = allowed.shape
    padded = np.zeros((rows, (cols + 31) // 32 * 32), bool)
    padded[:, :cols] = allowed
    words = np.packbits(padded.reshape(rows, -1, 32), axis=2, bitorder="little").view(np.uint32)[:, :, 0]
    return torch.from_numpy(words.view(np.int32).copy()).cuda()


def run_sample(ctx, torch, x, allowed=None, **s):
    rows = x.shape[0]
    token = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    logprob = torch.full((rows,), 7.0, device="cuda")
    ctx.sample_rows(x, s.pop("uniform"), token, logprob=logprob, allowed=allowed, **s)
    ctx.sync()
    return token.cpu().numpy(), numbers(logprob)


def check_sample(ctx, torch, x, allowed=None, every=1, **values):
    rows = x.shape[0]
    s = settings(torch, rows, **values)
    host = {k: v.double().cpu().numpy() for k, v in s.items()}
    token, logprob = run_sample(ctx, torch, x, bits_of(torch, allowed) if allowed is not None else None, **s)
    for r in range(0, rows, every):
        row = numbers(x[r])
        want, log_share, distance = sample(row, allowed=None if allowed is None else allowed[r], **{k: v[r] for k, v in host.items()})
        # a weight is off by half a unit of 2^-43 (of a total of at least one) and by the cubic polynomial, less than
        # (ln 2 / 128)^4 / 24 < 2^-34.6 of itself; both of two sums may be, so a share is off by less than
        weight_error = 2.0**-33.6 + row.size * 2.0**-43
        assert token[r] == want or distance < weight_error, (r, token[r], want, distance)
        if token[r] == want:
            # computed in 64 bits from such sums and rounded once
            assert logprob[r] == log_share or abs(logprob[r] - log_share) <= 2.0**-24 * abs(log_share) + weight_error


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [1, 2, 31, 33, 1000, 4099, 32768, 50257, 131072, 151001])
def test_sample_without_cuts(ctx, torch_cuda, rng, kind, cols):
    check_sample(ctx, torch_cuda, scores(torch_cuda, rng, 4, cols, kind), uniform=rng.random(4), temperature=[1.0, 0.5, 3.0, 100.0])


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cuts", [dict(top_k=1), dict(top_k=5), dict(top_k=300), dict(top_k=3000), dict(top_p=0.5), dict(top_p=0.9),
                                  dict(top_p=0.999), dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0), dict(min_p=7.0),
                                  dict(top_k=50, top_p=0.9), dict(top_k=50, top_p=0.9, min_p=0.05), dict(top_k=4000, min_p=0.01),
                                  dict(top_p=0.99999994), dict(top_k=10**9), dict(top_k=-3), dict(top_p=1.5, min_p=-1.0)])
@pytest.mark.parametrize("cols,temperature", [(4099, 0.7), (40000, 1.0), (100003, 2.0)])
def test_sample_with_cuts(ctx, torch_cuda, rng, kind, cols, temperature, cuts):
    check_sample(ctx, torch_cuda, scores(torch_cuda, rng, 6, cols, kind), uniform=rng.random(6), temperature=temperature, **cuts)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols", [(1500, 700), (1200, 5003)])
def test_sample_many_rows(ctx, torch_cuda, rng, kind, rows, cols):
    """More rows than the GPU holds at a time, so that a cluster of blocks takes one after the other."""
    t = torch_cuda
    x = scores(t, rng, rows, cols, kind, cols + 3, 1)
    x[::4] = scores(t, rng, (rows + 3) // 4, cols, kind, spread=0.05, peaks=False)
    x[7] = -float("inf")
    x[8, 1:] = float("nan")
    temperature = rng.choice([0.5, 1.0, 1.0, 2.0], rows)
    temperature[16] = 0.0
    temperature[17] = 1e-35
    temperature[18] = np.inf
    check_sample(ctx, t, x, uniform=rng.random(rows), temperature=temperature)
    check_sample(ctx, t, x, uniform=rng.random(rows), min_p=0.02)
    top_k = np.where(np.arange(rows) % 3 == 0, 20, 0)  # rows with and without cuts side by side
    check_sample(ctx, t, x, uniform=rng.random(rows), temperature=temperature, top_k=top_k)
    u = np.where(np.arange(rows) % 2 == 0, 0.0, 1.0 - 2.0**-24)
    check_sample(ctx, t, x, uniform=u, temperature=temperature)


@pytest.mark.parametrize("kind", TYPES)
def test_sample_flat_rows(ctx, torch_cuda, rng, kind):
    """Rows without a peak: every entry is near the border, and there are many ties in 16 bits."""
    x = scores(torch_cuda, rng, 8, 70001, kind, spread=0.3, peaks=False)
    for cuts in (dict(top_p=0.9), dict(top_k=1000), dict(top_k=40000, top_p=0.7), dict(min_p=0.5), dict()):
        check_sample(ctx, torch_cuda, x, uniform=rng.random(8), **cuts)


@pytest.mark.parametrize("kind", TYPES)
def test_sample_equal_scores(ctx, torch_cuda, kind):
    """All scores equal: the weights are exact in the reference too, so that borders can be met exactly."""
    t = torch_cuda
    x = place(t, np.full((9, 4096), 1.5, np.float32), kind)
    u = np.arange(9) / 8 * 0.9999999
    u[:8] = np.arange(8) / 8
    check_sample(ctx, t, x, uniform=u)
    check_sample(ctx, t, x, uniform=u, top_p=0.5)
    check_sample(ctx, t, x, uniform=u, top_k=8)
    check_sample(ctx, t, x, uniform=u, top_k=1000, top_p=0.25)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("offset,pitch", [(1, 5003), (5, 5001), (8, 5008)])
def test_sample_allowed(ctx, torch_cuda, rng, kind, offset, pitch):
    t = torch_cuda
    x = scores(t, rng, 12, 5001, kind, pitch, offset)
    allowed = rng.random((12, 5001)) < 0.3
    allowed[0] = False
    allowed[1] = False
    allowed[1, 5000] = True
    allowed[2] = False
    allowed[2, 0] = True
    allowed[3] = True
    host = numbers(x)
    host[~allowed] = rng.choice([np.nan, np.inf, -np.inf, 60000.0], (~allowed).sum())  # whatever a masked place holds
    x.copy_(t.from_numpy(host))
    check_sample(ctx, t, x, allowed, uniform=rng.random(12))
    check_sample(ctx, t, x, allowed, uniform=rng.random(12), temperature=0.8, top_k=40, top_p=0.9, min_p=0.01)


def test_sample_every_row_with_settings_of_its_own(ctx, torch_cuda, rng):
    n = 200
    check_sample(ctx, torch_cuda, scores(torch_cuda, rng, n, 3001, "bfloat16"), uniform=rng.random(n),
                 temperature=rng.choice([0.0, -1.0, np.nan, 0.3, 1.0, 2.0], n), top_k=rng.choice([0, 1, 2, 30, 3001, 5000], n),
                 top_p=rng.choice([1.0, 0.3, 0.9, np.nan], n), min_p=rng.choice([0.0, 0.1, np.nan], n))


@pytest.mark.parametrize("kind", TYPES)
def test_sample_rows_with_little_in_them(ctx, torch_cuda, rng, kind):
    t = torch_cuda
    x = rng.normal(0, 1, (8, 3000)).astype(np.float32)
    x[0] = -np.inf
    x[1, 5:] = -np.inf
    x[2] = np.nan
    x[3, ::2] = np.nan
    x[4] = np.finfo(np.float32).min if kind == "float32" else float(t.finfo(getattr(t, kind)).min)
    x[5, 7] = x[5, 1234] = np.inf
    x[6, 1:] = -np.inf
    x[7] = np.nan
    x[7, 2999] = -1.0
    for cuts in (dict(), dict(top_k=20), dict(top_p=0.9), dict(min_p=0.1), dict(top_k=20, top_p=0.5), dict(temperature=0.0),
                 dict(temperature=1e-30), dict(temperature=np.inf), dict(temperature=np.inf, top_p=0.5)):
        check_sample(ctx, t, place(t, x, kind), uniform=rng.random(8), **cuts)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [300, 9001, 100003])
def test_sample_infinite_scores_among_others(ctx, torch_cuda, rng, kind, cols):
    """Rows whose best scores are +inf, a few in one place or one in most threads' vectors: what the staged scores are
    replaced by is listed by other lanes of the warp than the ones that replaced it."""
    rows, every = 40, 1 if cols < 5000 else 3 if cols < 50000 else 7
    x = rng.normal(0, 2, (rows, cols)).astype(np.float32)
    for r in range(rows):
        n = (1, 2, 3, 20, 150)[r % 5]
        at = rng.choice(cols, n, replace=False) if r % 2 else rng.integers(0, cols - n + 1) + np.arange(n)
        x[r, at] = np.inf
    x = place(torch_cuda, x, kind, cols + 1, 1)
    allowed = rng.random((rows, cols)) < 0.7
    for cuts in (dict(top_k=1), dict(top_k=2), dict(top_k=30), dict(top_k=190), dict(top_k=400), dict(top_k=5, top_p=0.7), dict(top_p=0.5),
                 dict(top_k=9, temperature=0.0), dict(top_k=50, min_p=0.5), dict(top_k=50, temperature=1e5)):
        check_sample(ctx, torch_cuda, x, uniform=rng.random(rows), every=every, **cuts)
        check_sample(ctx, torch_cuda, x, allowed, uniform=rng.random(rows), every=every, **cuts)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("top_p", [-0.02, -1.0, -1e30, -np.inf, -0.0])
def test_sample_a_negative_share_takes_the_first(ctx, torch_cuda, rng, kind, top_p):
    """As 0 does, however negative: of rows of one entry, of equal ones, of any at a great temperature."""
    t = torch_cuda
    for cols in (1, 5, 4096, 100003):
        x = rng.normal(0, 2, (6, cols)).astype(np.float32)
        x[:2] = 1.5
        x[2] = np.round(x[2])
        for rest in (dict(), dict(temperature=np.inf), dict(temperature=0.01), dict(min_p=0.1), dict(min_p=1e-3, temperature=1e6), dict(top_k=3),
                     dict(top_k=1000)):
            check_sample(ctx, t, place(t, x, kind), uniform=rng.random(6), top_p=top_p, **rest)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("top", [1000.0, 30.0, 2.0, 1.0, -1.0, -20.0])
@pytest.mark.parametrize("min_p", [0.0, 1e-6])
def test_sample_shares_of_cold_rows_with_many_best(ctx, torch_cuda, rng, kind, top, min_p):
    """Hundreds of entries with each of the few best values, so that no list holds them, and temperatures at which the
    values next to one another weigh very differently: what a bin may weigh at most is not taken from scores above the
    row's largest."""
    t = torch_cuda
    rows, cols = 48, 20011
    step = abs(top) * {"float32": 1e-5, "float16": 2.0**-9, "bfloat16": 2.0**-6}[kind]
    x = rng.normal(top - 40 * step, 5 * step, (rows, cols)).astype(np.float32)
    x = np.minimum(x, np.float32(top - 20 * step))
    for r in range(rows):
        at = rng.permutation(cols)
        for i, v in enumerate((top, top - step * rng.uniform(0.5, 3), top - step * rng.uniform(3, 6))):
            x[r, at[700 * i:700 * i + 600]] = v
    x = place(t, x, kind)
    temperature = step * 10.0 ** rng.uniform(-1.5, 1.5, rows)
    check_sample(ctx, t, x, uniform=rng.choice([0.0, 0.5, 0.999], rows), temperature=temperature, top_p=rng.uniform(0.05, 0.95, rows),
                 min_p=np.full(rows, min_p))


def test_sample_a_share_of_equal_scores_above_others(ctx, torch_cuda):
    """600 scores of 1000 and 600 just below, cold: a share of 0.3 keeps 187 of the first."""
    t = torch_cuda
    x = np.zeros((1, 4096), np.float32)
    x[0, :600], x[0, 600:1200] = 1000.0, 999.99
    for u in (0.0, 0.5, 0.999):
        check_sample(ctx, t, place(t, x, "float32"), uniform=u, temperature=0.003, top_p=0.3)


@pytest.mark.parametrize("kind", TYPES)
def test_sample_the_only_entry_has_log_probability_zero(ctx, torch_cuda, rng, kind):
    """Exactly, whatever its score and the temperature, and no token's is above zero."""
    t = torch_cuda
    rows, cols = 64, 3001
    x = rng.normal(0, 3, (rows, cols)).astype(np.float32)
    x[::4] *= 1e-3
    x[np.arange(rows), rng.integers(0, cols, rows)] = x.max(axis=1) * rng.uniform(1.1, 1.5, rows)
    x = place(t, x, kind)
    one = np.zeros((rows, cols), bool)
    one[np.arange(rows), rng.integers(0, cols, rows)] = True
    temperature = (10.0 ** rng.uniform(-2, 2, rows)).astype(np.float32)
    for allowed, cuts in ((None, dict(top_k=1)), (None, dict(top_p=0.0)), (None, dict(min_p=1.0)), (one, dict()), (one, dict(top_k=40)),
                          (one, dict(top_p=0.9)), (one, dict(min_p=0.1)), (None, dict(top_k=1, top_p=0.5, min_p=0.5))):
        _, logprob = run_sample(ctx, t, x, None if allowed is None else bits_of(t, allowed),
                                **settings(t, rows, uniform=rng.random(rows), temperature=temperature, **cuts))
        assert (logprob == 0).all(), (cuts, logprob[logprob != 0])
    for cuts in (dict(), dict(top_k=2), dict(top_p=0.9), dict(top_k=400), dict(min_p=0.5)):
        _, logprob = run_sample(ctx, t, x, **settings(t, rows, uniform=rng.random(rows), temperature=temperature / 50, **cuts))
        assert (logprob <= 0).all(), (cuts, logprob[logprob > 0])


def test_sample_random_numbers_at_the_ends(ctx, torch_cuda, rng):
    t = torch_cuda
    x = scores(t, rng, 6, 5000, "float32")
    for u in (0.0, 1.0 - 2.0**-24, 1.0, 2.0):
        check_sample(ctx, t, x, uniform=u)
    token, _ = run_sample(ctx, t, x, **settings(t, 6, uniform=np.nan))
    assert ((token >= 0) & (token < 5000)).all()


def test_sample_of_rows_too_long_for_shared_memory(ctx, torch_cuda, rng):
    n = (1 << 20) - 1
    x = scores(torch_cuda, rng, 2, n, "float32", n + 2, 3)
    allowed = rng.random((2, n)) < 0.5
    for cuts in (dict(), dict(top_k=100, top_p=0.9), dict(top_p=0.8, min_p=1e-4)):
        check_sample(ctx, torch_cuda, x, uniform=rng.random(2), **cuts)
        check_sample(ctx, torch_cuda, x, allowed, uniform=rng.random(2), **cuts)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("near_zero", [False, True])
def test_sample_close_to_the_borders(ctx, torch_cuda, rng, kind, near_zero):
    """Random numbers next to the border between two tokens (as near as 32 bits come); also where the scores are so much
    smaller than the largest that their difference from it takes more than 32 bits."""
    t = torch_cuda
    rows, cols = 120, 20011
    x = scores(t, rng, rows, cols, kind)
    temperature = np.full(rows, 0.9, np.float32)
    if near_zero:
        top = 2.0 ** rng.integers(4, 8, rows)
        x.copy_(t.from_numpy((rng.uniform(0, 2.0**-25, (rows, cols)) * top[:, None]).astype(np.float32)))
        x[t.arange(rows), t.from_numpy(rng.choice(cols, rows))] = t.from_numpy(top).to(x.dtype).cuda()
        temperature = (top / rng.uniform(9, 11, rows)).astype(np.float32)
    u = np.empty(rows, np.float32)
    for r, row in enumerate(numbers(x)):
        share = np.cumsum(np.exp((row - row.max()) / float(temperature[r])))
        u[r] = (share / share[-1])[rng.integers(0, cols - 1)]
    check_sample(ctx, t, x, uniform=u, temperature=temperature)
    check_sample(ctx, t, x, uniform=u, temperature=temperature, top_p=0.99999)


def test_sample_draws_by_the_shares(ctx, torch_cuda):
    """4096 evenly spaced random numbers over one row draw every index as often as its share says, give or take one."""
    t = torch_cuda
    n = 4096
    row = t.linspace(-3, 3, 50, device="cuda")
    x = row.expand(n, 50).contiguous()
    u = (t.arange(n, device="cuda") + 0.5) / n
    token = t.empty(n, dtype=t.int32, device="cuda")
    ctx.sample_rows(x, u, token)
    ctx.sync()
    share = t.softmax(row.double(), 0).cpu().numpy()
    assert np.abs(np.bincount(token.cpu().numpy(), minlength=50) - n * share).max() <= 1.0


# ----------------------------------------------------------- distillation
def teacher_of(torch, rng, x, k, kind, temperature, rest):
    """A teacher's k best scores of rows like the student's, some entries missing."""
    rows, cols = x.shape
    z = np.nan_to_num(numbers(x), nan=0.0, posinf=5.0, neginf=-5.0) + rng.normal(0, 0.7, (rows, cols))
    at = np.stack([rng.permutation(np.argsort(-row)[:k]) for row in z])
    values = np.take_along_axis(z, at, 1)
    lse = np.array([np.log(np.exp(row / temperature - (row / temperature).max()).sum()) + (row / temperature).max() for row in z])
    at = at.astype(np.int32)
    if k > 3:
        at[::3, k // 2] = -1
        at[1::3, 0] = cols
        values[2::3, 1] = -np.inf
    return (torch.from_numpy(values).to(getattr(torch, kind)).cuda(), torch.from_numpy(at).cuda(),
            torch.from_numpy(lse).float().cuda() if rest else None)


def check_gradient(got, x, teacher, index, lse, weight, upstream, temperature, kind):
    t, i = numbers(teacher), index.cpu().numpy()
    for r, row in enumerate(numbers(x)):
        _, d, parts = distill(row, t[r], i[r], None if lse is None else float(lse[r]), float(weight[r]), temperature)
        d = d * upstream[r]
        # (sum p + r) q - p, (sum p + r - r / q_r) q: every part is off by its own share, however small the difference
        parts = parts * abs(upstream[r])
        small = 2.0**-24 if kind == "float16" else 2.0**-126  # half a step of subnormal numbers
        bad = ~(np.abs(got[r] - d) <= EPS[kind] * np.abs(d) + 2 * SUM_ERROR * parts + small)
        assert not bad.any(), (r, np.nonzero(bad)[0][:5], got[r][bad][:5], d[bad][:5])


def check_distill(ctx, torch, rng, x, k, temperature=1.0, rest=False, teacher_kind="float32", in_place=False, weight=None, teacher=None,
                  grad_pitch=None, grad_offset=0):
    rows, cols = x.shape
    kind = str(x.dtype)[6:]
    tv, ti, lse = teacher or teacher_of(torch, rng, x, k, teacher_kind, temperature, rest)
    if weight is None:
        weight = rng.uniform(0.1, 2, rows).astype(np.float32)
        weight[rows // 2:rows // 2 + 1] = 0.0 if rows > 2 else weight[0]
    w = torch.from_numpy(weight).cuda()
    host = x.clone()
    want = [distill(row, numbers(tv)[r], ti.cpu().numpy()[r], None if lse is None else float(lse[r]), float(weight[r]), temperature)[0]
            for r, row in enumerate(numbers(host))]
    new = lambda *shape: torch.full(shape, 7.0, device="cuda")  # noqa: E731
    loss, stats = new(rows), new(rows, 4)
    ctx.distill_rows(x, tv, ti, loss, stats=stats, teacher_lse=lse, weight=w, temperature=temperature)
    ctx.sync()
    allowance = np.abs(weight) * SUM_ERROR * 2 + 2.0**-23 * np.abs(want)
    assert (np.abs(numbers(loss) - want) <= allowance).all(), (numbers(loss), want)
    # backward from the statistics
    upstream = rng.uniform(-2, 2, rows).astype(np.float32)
    fresh = lambda: place(torch, np.zeros((rows, cols), np.float32), kind, grad_pitch, grad_offset)  # noqa: E731
    grad = fresh()
    ctx.distill_rows_backward(x, tv, ti, stats, torch.from_numpy(upstream).cuda(), grad, teacher_lse=lse, weight=w, temperature=temperature)
    ctx.sync()
    check_gradient(numbers(grad), host, tv, ti, lse, weight, upstream, temperature, kind)
    # both in one pass
    both, grad = new(rows), x if in_place else fresh()
    ctx.distill_rows(x, tv, ti, both, grad=grad, teacher_lse=lse, weight=w, temperature=temperature)
    ctx.sync()
    assert torch.equal(both, loss)
    check_gradient(numbers(grad), host, tv, ti, lse, weight, np.ones(rows), temperature, kind)
    if in_place:
        x.copy_(host)
        ctx.distill_rows_backward(x, tv, ti, stats, None, x, teacher_lse=lse, weight=w, temperature=temperature)
        ctx.sync()
        check_gradient(numbers(x), host, tv, ti, lse, weight, np.ones(rows), temperature, kind)
        x.copy_(host)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (3, 2, 1), (5, 7, 7), (2, 33, 5), (4, 1000, 50), (2, 1024, 1024), (3, 4099, 300),
                                         (2, 32768, 64), (5, 50257, 20), (2, 131072, 100), (2, 151001, 7)])
def test_distill(ctx, torch_cuda, rng, kind, rows, cols, k, rest):
    check_distill(ctx, torch_cuda, rng, scores(torch_cuda, rng, rows, cols, kind), k, 1.0 if cols % 2 else 2.0, rest)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("teacher_kind", TYPES)
def test_distill_types_of_the_teacher(ctx, torch_cuda, rng, kind, teacher_kind):
    check_distill(ctx, torch_cuda, rng, scores(torch_cuda, rng, 3, 3001, kind), 20, 0.7, True, teacher_kind)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("offset,pitch,grad_offset,grad_pitch", [(1, 1013, 1, 1013), (3, 1001, 0, 1008), (0, 1008, 5, 1003), (7, 1003, 7, 1011)])
def test_distill_of_rows_anywhere(ctx, torch_cuda, rng, kind, offset, pitch, grad_offset, grad_pitch):
    x = scores(torch_cuda, rng, 6, 1001, kind, pitch, offset)
    check_distill(ctx, torch_cuda, rng, x, 12, rest=True, grad_pitch=grad_pitch, grad_offset=grad_offset)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols", [1001, 100003])
def test_distill_in_place(ctx, torch_cuda, rng, kind, cols):
    check_distill(ctx, torch_cuda, rng, scores(torch_cuda, rng, 4, cols, kind, cols + 2, 1), 16, rest=True, in_place=True)


@pytest.mark.parametrize("rest", [False, True])
def test_distill_of_rows_too_long_for_shared_memory(ctx, torch_cuda, rng, rest):
    n = (1 << 20) - 5
    check_distill(ctx, torch_cuda, rng, scores(torch_cuda, rng, 2, n, "float32", n + 2, 1), 40, rest=rest, in_place=True)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("kind", TYPES)
def test_distill_an_index_named_twice(ctx, torch_cuda, rng, kind, rest):
    t = torch_cuda
    x = scores(t, rng, 3, 2000, kind)
    tv, ti, lse = teacher_of(t, rng, x, 300, "float32", 1.0, rest)
    ti[0, 5] = ti[0, 299] = ti[0, 100]
    ti[1, :] = 17
    ti[2, 290] = ti[2, 0]
    if rest:
        lse = lse + 1.5  # what is named twice must not add up to more than there is
        lse[1] += 5.0
    check_distill(ctx, t, rng, x, 300, teacher=(tv, ti, lse))


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("kind", TYPES)
def test_distill_rows_that_do_not_count(ctx, torch_cuda, rng, kind, rest):
    t = torch_cuda
    x = scores(t, rng, 6, 3001, kind)
    tv, ti, lse = teacher_of(t, rng, x, 9, "float32", 1.0, rest)
    x[0] = float("nan")           # weight 0
    x[1] = -float("inf")          # a student that excludes everything
    ti[2] = -1                    # a teacher that names nothing
    tv[3] = -float("inf")
    x[4, 5::2] = -float("inf")    # a student that excludes half
    ti[4] = t.arange(0, 18, 2, dtype=t.int32, device="cuda")
    weight = np.array([0, 1, 1, 1, 1, 1], np.float32)
    check_distill(ctx, t, rng, x, 9, weight=weight, teacher=(tv, ti, lse), in_place=True)


def test_distill_the_rest_alone_far_below(ctx, torch_cuda, rng):
    """The student leaves the unnamed entries less than 32 bits can hold next to the named ones."""
    t = torch_cuda
    x = rng.normal(0, 1, (2, 2000)).astype(np.float32)
    x[:, :4] += 150.0
    tv = t.tensor([[1.0, 0.5, 0.2, 0.1]] * 2, device="cuda")
    ti = t.arange(4, dtype=t.int32, device="cuda").repeat(2, 1)
    lse = t.tensor([2.0, 3.0], device="cuda")
    loss = t.empty(2, device="cuda")
    ctx.distill_rows(place(t, x, "float32"), tv, ti, loss, teacher_lse=lse)
    ctx.sync()
    want = [distill(x[r], tv[r].cpu().numpy(), ti[r].cpu().numpy(), float(lse[r]), 1.0, 1.0)[0] for r in range(2)]
    assert np.abs(numbers(loss) - want).max() <= 2.0**-23 * max(want) + 2 * SUM_ERROR


@pytest.mark.parametrize("kind,cols", [("float32", 2000), ("bfloat16", 40000), ("float16", 3001), ("float32", (1 << 20) - 7)])
@pytest.mark.parametrize("temperature", [1.0, 0.05])
def test_distill_gradient_of_the_rest_far_below(ctx, torch_cuda, rng, kind, cols, temperature):
    """Entries that are not named and so unlikely that their probability has no 32-bit value: the share of the rest that
    an entry has still moves it.  From nearly as likely as the named ones to e^-600."""
    t = torch_cuda
    apart = np.array([0.0, 10.0, 20.0, 24.0, 40.0, 70.0, 100.0, 200.0, 600.0], np.float32) * temperature
    if cols > 1 << 19:
        apart = apart[5:7]
    rows = apart.size
    x = rng.normal(0, 2 * temperature, (rows, cols)).astype(np.float32)
    at = np.stack([rng.choice(cols, 4, replace=False) for _ in range(rows)]).astype(np.int32)
    np.put_along_axis(x, at, rng.normal(0, temperature, (rows, 4)).astype(np.float32) + 9 * temperature + apart[:, None], 1)
    tv = t.tensor([[1.0, 0.5, 0.2, 0.1]] * rows, device="cuda") * temperature
    lse = t.full((rows,), 2.0, device="cuda")
    lse[1::3] = 4.0
    check_distill(ctx, t, rng, place(t, x, kind, cols + 1, 1), 4, temperature, teacher=(tv, t.from_numpy(at).cuda(), lse), in_place=True)


@pytest.mark.parametrize("rest", [False, True])
def test_distill_infinities_in_a_row_that_counts(ctx, torch_cuda, rng, rest):
    """+inf has no share of a softmax: loss and gradient are NaN, of that row alone."""
    t = torch_cuda
    x = scores(t, rng, 4, 1000, "bfloat16")
    tv, ti, lse = teacher_of(t, rng, x, 3, "float32", 1.0, rest)
    x[0, 999] = float("inf")
    x[1, int(ti[1, 2])] = float("inf")
    tv[2, 1] = float("inf")
    loss, grad = t.zeros(4, device="cuda"), t.zeros_like(x)
    ctx.distill_rows(x, tv, ti, loss, grad=grad, teacher_lse=lse)
    ctx.sync()
    if not rest:
        assert loss.isnan().tolist() == [True, True, True, False]
    assert not loss[:3].isfinite().any() and loss[3].isfinite()
    assert not grad[3].isnan().any()


def test_distill_nan_in_a_row_that_counts(ctx, torch_cuda, rng):
    t = torch_cuda
    for rest in (False, True):
        x = scores(t, rng, 3, 1000, "bfloat16")
        tv, ti, lse = teacher_of(t, rng, x, 5, "float32", 1.0, rest)
        x[0, 999] = float("nan")
        x[1, int(ti[1, 4])] = float("nan")
        loss, stats, grad = t.zeros(3, device="cuda"), t.zeros(3, 4, device="cuda"), t.zeros_like(x)
        ctx.distill_rows(x, tv, ti, loss, stats=stats, grad=grad, teacher_lse=lse)
        ctx.sync()
        assert loss.isnan().tolist() == [True, True, False]
        assert grad[:2].isnan().all() and not grad[2].isnan().any()
        grad.zero_()
        ctx.distill_rows_backward(x, tv, ti, stats, None, grad, teacher_lse=lse)
        ctx.sync()
        assert grad[:2].isnan().all() and not grad[2].isnan().any()


def test_distill_a_teacher_whose_weight_is_all_elsewhere(ctx, torch_cuda, rng):
    """teacher_lse of +inf, or far above the scores: the named entries have no probability and the rest has it all."""
    t = torch_cuda
    x = scores(t, rng, 3, 1000, "float32")
    tv, ti, lse = teacher_of(t, rng, x, 5, "float32", 1.0, True)
    lse[0], lse[1] = float("inf"), 1e30
    check_distill(ctx, t, rng, x, 5, teacher=(tv, ti, lse), weight=np.ones(3, np.float32))


@pytest.mark.parametrize("cols", [3000, 131072])
def test_distill_of_entries_named_twice_is_the_same_every_time(ctx, torch_cuda, rng, cols):
    """Whichever thread meets an index first, the sums are taken in one order."""
    t = torch_cuda
    rows, k = 600, 768
    x = scores(t, rng, rows, cols, "float32" if cols < 5000 else "bfloat16")
    ti = t.from_numpy(rng.integers(0, min(cols, 300), (rows, k)).astype(np.int32)).cuda()
    x[:, :300] += t.from_numpy(rng.uniform(5, 30, (rows, 300)).astype(np.float32)).cuda()  # what is named has most of the weight
    tv, lse = t.randn(rows, k, device="cuda"), t.full((rows,), 9.0, device="cuda")
    new = lambda: (t.empty(rows, device="cuda"), t.empty_like(x), t.empty(rows, 4, device="cuda"))  # noqa: E731
    want, got = new(), new()
    for i in range(40):
        loss, grad, stats = got if i else want
        ctx.distill_rows(x, tv, ti, loss, grad=grad, stats=stats, teacher_lse=lse)
        assert all(t.equal(a, b) for a, b in zip(got, want)) if i else True


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("cols,temperature", [(3001, 1.0), (32768, 0.7), (131072, 1.0)])
def test_distill_a_loss_near_agreement(ctx, torch_cuda, rng, kind, cols, temperature):
    """A student that is nearly its teacher, so that the loss is the difference of like numbers: log q of the named entries
    and of the rest, near 0 both.  What is named has at least 0.9 of the weight.  Its exponentials and those that join the
    sums are off by less than 2^-31 each, a sum of the others, x of the weight, by 2^-22 of a term plus 128 additions of a thread, half a
    step each, 2^-17 at most, and scale^-1 in 32 bits (2^-24 of an exponent of at most 30): x (2^-22 + 2^-17 + 2^-19) at
    most.  The loss is r log r - r log q_r + sum p (log p - log q): an error d of the others' sum moves log q by x d and log
    q_r by d (1 - x), so the loss by about |x - r| d, and r and x are alike within a tenth of 0.1; and it is rounded once."""
    t = torch_cuda
    rows, k = 24, 40
    x = rng.normal(0, 1, (rows, cols)).astype(np.float32)
    at = np.stack([rng.choice(cols, k, replace=False) for _ in range(rows)]).astype(np.int32)
    np.put_along_axis(x, at, rng.uniform(14, 18, (rows, k)).astype(np.float32) * temperature, 1)
    x = place(t, x, kind)
    z = numbers(x)
    teacher = z + rng.normal(0, 0.01, z.shape)
    tv = t.from_numpy(np.take_along_axis(teacher, at, 1)).float().cuda()
    lse = t.from_numpy(np.array([np.log(np.exp(row / temperature).sum()) for row in teacher])).float().cuda()
    ti, loss = t.from_numpy(at).cuda(), t.empty(rows, device="cuda")
    ctx.distill_rows(x, tv, ti, loss, teacher_lse=lse, temperature=temperature)
    ctx.sync()
    for r in range(rows):
        want = distill(z[r], numbers(tv)[r], at[r], float(lse[r]), 1.0, temperature)[0]
        named = np.exp(z[r][at[r]] / temperature).sum()
        share = 1 - named / np.exp(z[r] / temperature).sum()
        rest = max(0.0, 1 - np.exp(numbers(tv)[r] / temperature - float(lse[r])).sum())
        assert share < 0.1
        d = 2.0**-22 + 2.0**-17 + 2.0**-19
        allowance = abs(share - rest) * d + 2.0**-30 + 2.0**-24 * abs(want)
        assert abs(float(loss[r]) - want) <= allowance, (r, float(loss[r]), want, allowance)


@pytest.mark.parametrize("rest", [False, True])
def test_distill_gradient_against_differences(ctx, torch_cuda, rng, rest):
    """Central differences of the loss, 32 bits: h = 2^-3, the third derivative of a log-sum-exp is below 1, so the
    difference is off by h^2 / 6 at most, plus the loss's own error over 2 h."""
    t = torch_cuda
    n, k, h = 40, 6, 0.125
    x = rng.normal(0, 1, n).astype(np.float32)
    at = rng.choice(n, k, replace=False).astype(np.int32)
    rows = np.repeat(x[None], 2 * n + 1, 0)
    for j in range(n):
        rows[2 * j, j] += h
        rows[2 * j + 1, j] -= h
    tv = t.from_numpy(rng.normal(1, 1, k).astype(np.float32)).cuda().repeat(2 * n + 1, 1)
    ti = t.from_numpy(at).cuda().repeat(2 * n + 1, 1)
    lse = t.full((2 * n + 1,), float(np.log(np.exp(numbers(tv)[0]).sum()) + 0.5), device="cuda") if rest else None
    loss, grad = t.empty(2 * n + 1, device="cuda"), t.empty(2 * n + 1, n, device="cuda")
    ctx.distill_rows(place(t, rows, "float32"), tv, ti, loss, grad=grad, teacher_lse=lse, temperature=1.0)
    ctx.sync()
    loss = numbers(loss)
    d = (loss[0:2 * n:2] - loss[1:2 * n:2]) / (2 * h)
    assert np.abs(d - numbers(grad)[2 * n]).max() <= h * h / 6 + (2 * SUM_ERROR + 2.0**-23 * loss.max()) / h


# ------------------------------------------------------------- in use
def test_rows_nobody_asked_for_stay_as_they_were(ctx, torch_cuda, rng):
    t = torch_cuda
    x = scores(t, rng, 4, 1001, "bfloat16", 1008, 0)
    tv, ti, _ = teacher_of(t, rng, x, 4, "float32", 1.0, False)
    memory = t.full((6, 1008), 5.0, dtype=t.bfloat16, device="cuda")
    loss = t.full((6,), 5.0, device="cuda")
    ctx.distill_rows(x, tv, ti, loss[1:5], grad=memory[1:5, 3:1004])
    token = t.full((6,), 5, dtype=t.int32, device="cuda")
    ctx.sample_rows(x, t.rand(4, device="cuda"), token[1:5])
    ctx.sync()
    assert (memory[0] == 5).all() and (memory[5] == 5).all() and (memory[:, :3] == 5).all() and (memory[:, 1004:] == 5).all()
    assert loss[0] == 5 and loss[5] == 5 and token[0] == 5 and token[5] == 5


def test_no_rows(ctx, torch_cuda):
    t = torch_cuda
    x = t.empty(0, 100, device="cuda")
    e = lambda *shape, kind=t.float32: t.empty(shape, dtype=kind, device="cuda")  # noqa: E731
    ctx.top_rows(x, e(0, 5), e(0, 5, kind=t.int32), lse=e(0))
    ctx.sample_rows(x, e(0), e(0, kind=t.int32))
    ctx.distill_rows(x, e(0, 5), e(0, 5, kind=t.int32), e(0), grad=e(0, 100), stats=e(0, 4))
    ctx.distill_rows_backward(x, e(0, 5), e(0, 5, kind=t.int32), e(0, 4), None, e(0, 100))
    ctx.sync()


def test_teacher_to_student_to_answer_on_a_stream_and_as_a_graph(accb, ctx, torch_cuda, rng):
    """The operators as they are used together: a teacher's best scores, the student's loss and gradient, a step along
    it, and a token of the new scores; eagerly on a stream of its own, and replayed as a graph with new inputs."""
    t = torch_cuda
    rows, cols, k = 6, 20011, 32
    teacher, student = scores(t, rng, rows, cols, "bfloat16"), scores(t, rng, rows, cols, "float32")
    u = t.from_numpy(rng.random(rows).astype(np.float32)).cuda()
    top_k = t.full((rows,), 20, dtype=t.int32, device="cuda")
    values, index, lse = t.empty(rows, k, dtype=t.bfloat16, device="cuda"), t.empty(rows, k, dtype=t.int32, device="cuda"), t.empty(rows, device="cuda")
    loss, grad, token = t.empty(rows, device="cuda"), t.empty(rows, cols, device="cuda"), t.empty(rows, dtype=t.int32, device="cuda")

    def run(stream):
        ctx.top_rows(teacher, values, index, lse=lse, stream=stream)
        ctx.distill_rows(student, values, index, loss, grad=grad, teacher_lse=lse, stream=stream)
        ctx.sample_rows(student, u, token, top_k=top_k, stream=stream)

    s = t.cuda.Stream()
    s.wait_stream(t.cuda.current_stream())
    with t.cuda.stream(s):
        run(None)  # the current stream
    s.synchronize()
    for r in range(rows):
        v, i, m = top(numbers(teacher)[r], k, 1.0)
        assert np.array_equal(numbers(values)[r], v) and np.array_equal(index.cpu().numpy()[r], i)
        want = distill(numbers(student)[r], v, i, float(lse[r]), 1.0, 1.0)[0]
        assert abs(float(loss[r]) - want) <= 2 * SUM_ERROR + 2.0**-23 * abs(want)
        assert int(token[r]) == sample(numbers(student)[r], float(u[r]), top_k=20)[0]
    eager = [a.clone() for a in (values, index, lse, loss, grad, token)]
    graph, second = t.cuda.CUDAGraph(), t.cuda.CUDAGraph()
    with t.cuda.graph(graph):
        run(None)
    with t.cuda.graph(second):
        run(None)
    other = scores(t, rng, rows, cols, "bfloat16")
    kept, was = teacher.clone(), student.clone()
    for g in (graph, second, graph):
        teacher.copy_(other)
        student.copy_(other)
        g.replay()
        teacher.copy_(kept)
        student.copy_(was)
        for a in (values, index, lse, loss, grad, token):
            a.zero_()
        g.replay()
        t.cuda.synchronize()
        for a, b in zip((values, index, lse, loss, grad, token), eager):
            assert t.equal(a, b)


def test_first_calls_are_captured():
    """A program whose first call of each kind is made while its stream is captured."""
    code = """
import importlib, torch
accb = importlib.import_module("accelerate-cuda_b200")
ctx = accb.Context(0)
x = torch.randn(40, 9000, device="cuda").bfloat16()
u = torch.full((40,), 0.5, device="cuda")
values, index, token = torch.empty_like(x[:, :8]), torch.empty(40, 8, dtype=torch.int32, device="cuda"), torch.empty(40, dtype=torch.int32, device="cuda")
loss, grad, lse = torch.empty(40, device="cuda"), torch.empty_like(x), torch.empty(40, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
def run():
    ctx.top_rows(x, values, index, lse=lse)
    ctx.sample_rows(x, u, token)
    ctx.distill_rows(x, values, index, loss, grad=grad, teacher_lse=lse)
with torch.cuda.graph(graph):
    run()
graph.replay()
torch.cuda.synchronize()
got = [t.clone() for t in (values, index, lse, token, loss, grad)]
run()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, (values, index, lse, token, loss, grad)))
print("captured")
"""
    done = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("blocks", [1, 2, 3, 4, 5, 6, 7, 8])
@pytest.mark.parametrize("kind", ["bfloat16", "float32"])
def test_rows_by_any_number_of_blocks(ctx, torch_cuda, rng, kind, blocks):
    """Enough rows that a row gets as few blocks as hold it."""
    t = torch_cuda
    rows, cols = 300 if blocks == 1 else 150, (69632 * blocks - 300) // (2 if kind == "bfloat16" else 4)
    x = scores(t, rng, rows, cols, kind)
    few = (rows - 1) // 3
    check_top(ctx, t, x, 50, every=few)
    check_top(ctx, t, x, 900, 2.0, every=few)
    for cuts in (dict(), dict(top_k=40), dict(top_p=0.8), dict(top_k=700, top_p=0.9), dict(min_p=0.02), dict(temperature=0.0)):
        check_sample(ctx, t, x, uniform=rng.random(rows), every=few, **cuts)
    some = t.arange(0, rows, few, device="cuda")
    tv, ti, lse = t.randn(rows, 60, device="cuda"), t.randint(0, cols, (rows, 60), device="cuda", dtype=t.int32), t.full((rows,), 6.0, device="cuda")
    for rest in (None, lse):
        loss, grad, stats = t.empty(rows, device="cuda"), t.empty_like(x), t.empty(rows, 4, device="cuda")
        ctx.distill_rows(x, tv, ti, loss, grad=grad, stats=stats, teacher_lse=rest)
        ctx.sync()
        one = np.ones(some.numel())
        part = lambda a: None if a is None else a[some]  # noqa: E731
        check_gradient(numbers(grad[some]), x[some], tv[some], ti[some], part(rest), one, one, 1.0, kind)
        for r in some.tolist():
            want = distill(numbers(x[r]), numbers(tv[r]), ti[r].cpu().numpy(), None if rest is None else 6.0, 1.0, 1.0)[0]
            assert abs(float(loss[r]) - want) <= 2 * SUM_ERROR + 2.0**-23 * abs(want)
        grad.fill_(7.0)
        ctx.distill_rows_backward(x, tv, ti, stats, None, grad, teacher_lse=rest)
        ctx.sync()
        check_gradient(numbers(grad[some]), x[some], tv[some], ti[some], part(rest), one, one, 1.0, kind)


def test_calls_from_several_threads_and_contexts(accb, ctx, torch_cuda, rng):
    t = torch_cuda
    x = scores(t, rng, 200, 20011, "bfloat16")
    u = t.from_numpy(rng.random(200).astype(np.float32)).cuda()
    other = accb.Context(0)

    def call(c, stream, values, index, lse, token, loss, grad):
        for _ in range(10):
            c.top_rows(x, values, index, lse=lse, stream=stream)
            c.sample_rows(x, u, token, stream=stream)
            c.distill_rows(x, values, index, loss, grad=grad, teacher_lse=lse, stream=stream)

    def results():
        return (t.empty(200, 30, dtype=x.dtype, device="cuda"), t.empty(200, 30, dtype=t.int32, device="cuda"), t.empty(200, device="cuda"),
                t.empty(200, dtype=t.int32, device="cuda"), t.empty(200, device="cuda"), t.empty_like(x))

    want, out, streams = results(), [results() for _ in range(4)], [t.cuda.Stream() for _ in range(4)]
    call(ctx, None, *want)
    t.cuda.synchronize()
    threads = [threading.Thread(target=call, args=((ctx, other)[i % 2], streams[i].cuda_stream, *out[i])) for i in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    t.cuda.synchronize()
    for got in out:
        assert all(t.equal(a, b) for a, b in zip(got, want))


def test_device_arrays(accb, ctx, torch_cuda, rng):
    """Memory that is not torch's, and a stream by number."""
    t = torch_cuda
    x = scores(t, rng, 5, 3000, "float16")
    raw = lambda a, dtype: accb.DeviceArray(a.data_ptr(), a.shape, dtype)  # noqa: E731
    values, index = t.empty(5, 7, dtype=t.float16, device="cuda"), t.empty(5, 7, dtype=t.int32, device="cuda")
    t.cuda.synchronize()
    ctx.top_rows(raw(x, np.float16), raw(values, np.float16), raw(index, np.int32), stream=0)
    t.cuda.synchronize()
    for r, row in enumerate(numbers(x)):
        v, i, _ = top(row, 7, 1.0)
        assert np.array_equal(numbers(values)[r], v) and np.array_equal(index[r].cpu().numpy(), i)


def test_rows_of_more_lengths_than_are_remembered(ctx, torch_cuda, rng):
    """The context remembers how many clusters the GPU holds for the last 64 kinds of launch."""
    lengths = list(range(40, 40 + 8 * 80, 8)) * 2
    x = scores(torch_cuda, rng, 400, 700, "float32")
    for n in lengths:
        check_top(ctx, torch_cuda, x[:, :n], 3, every=133)


def test_calls_on_two_streams_at_once(ctx, torch_cuda, rng):
    t = torch_cuda
    x = scores(t, rng, 300, 30011, "bfloat16")
    u = t.from_numpy(rng.random(300).astype(np.float32)).cuda()
    p = t.full((300,), 0.9, device="cuda")
    streams = [t.cuda.Stream() for _ in range(4)]
    out = [t.empty(300, dtype=t.int32, device="cuda") for _ in range(5)]
    ctx.sample_rows(x, u, out[4], top_p=p)
    t.cuda.synchronize()
    for _ in range(20):
        for s, o in zip(streams, out):
            ctx.sample_rows(x, u, o, top_p=p, stream=s.cuda_stream)
    t.cuda.synchronize()
    assert all(t.equal(o, out[4]) for o in out)


def test_same_rows_alone_and_in_a_batch(ctx, torch_cuda, rng):
    """How many blocks hold a row depends on how many rows there are; what is drawn does not."""
    t = torch_cuda
    x = scores(t, rng, 400, 40000, "bfloat16")
    u = t.from_numpy(rng.random(400).astype(np.float32)).cuda()
    p = t.full((400,), 0.95, device="cuda")
    batch, one = t.empty(400, dtype=t.int32, device="cuda"), t.empty(1, dtype=t.int32, device="cuda")
    lp, lp1 = t.empty(400, device="cuda"), t.empty(1, device="cuda")
    ctx.sample_rows(x, u, batch, logprob=lp, top_p=p)
    for r in (0, 1, 7, 399):
        ctx.sample_rows(x[r:r + 1], u[r:r + 1], one, logprob=lp1, top_p=p[r:r + 1])
        ctx.sync()
        assert t.equal(one, batch[r:r + 1]) and t.equal(lp1, lp[r:r + 1])


def test_offsets_past_32_bits(ctx, torch_cuda, rng):
    """Rows that start more than 2^32 elements into the matrix."""
    t = torch_cuda
    rows, cols, pitch = 5, 1000, (1 << 30) + 8
    memory = t.empty((rows - 1) * pitch + cols, dtype=t.bfloat16, device="cuda")
    x = memory.as_strided((rows, cols), (pitch, 1))
    x.copy_(t.from_numpy(rng.normal(0, 2, (rows, cols)).astype(np.float32)))
    check_top(ctx, t, x, 10)
    check_sample(ctx, t, x, uniform=rng.random(rows), top_p=0.9)
    tv, ti, _ = teacher_of(t, rng, x, 5, "float32", 1.0, False)
    host, loss = x.contiguous(), t.empty(rows, device="cuda")
    ctx.distill_rows(x, tv, ti, loss, grad=x)
    ctx.sync()
    check_gradient(numbers(x), host, tv, ti, None, np.ones(rows), np.ones(rows), 1.0, "bfloat16")


def test_gradient_beside_the_scores(ctx, torch_cuda, rng):
    """Scores and gradient side by side in the rows of one matrix; any other overlap is refused."""
    t = torch_cuda
    both = t.full((5, 2100), 7.0, dtype=t.bfloat16, device="cuda")
    x, grad = both[:, :1000], both[:, 1003:2003]
    x.copy_(scores(t, rng, 5, 1000, "bfloat16"))
    tv, ti, _ = teacher_of(t, rng, x, 5, "float32", 1.0, False)
    host, loss = x.clone(), t.empty(5, device="cuda")
    ctx.distill_rows(x, tv, ti, loss, grad=grad)
    ctx.sync()
    check_gradient(numbers(grad), host, tv, ti, None, np.ones(5), np.ones(5), 1.0, "bfloat16")
    assert t.equal(x, host) and (both[:, 1000:1003] == 7).all() and (both[:, 2003:] == 7).all()


def test_overlaps_and_misaligned_pointers_are_refused(accb, ctx, torch_cuda):
    t = torch_cuda
    L = accb.lib()
    import ctypes as C
    m = t.zeros(4096, device="cuda")
    p, off = C.c_void_p(m.data_ptr()), C.c_void_p(m.data_ptr() + 2)
    rows = lambda at=0, pitch=10, rows=4: C.byref(accb.accb_rows_array(m.data_ptr() + 4 * at, 0, 8, rows, pitch))  # noqa: E731
    for a, b in ((rows(), rows(1)), (rows(5), rows()), (rows(), rows(9)), (rows(), rows(12)), (rows(), rows(0, 11)), (rows(0, 10, 1), rows(7, 10, 1)),
                 (rows(20, 8), rows(51, 8))):
        assert L.accb_distill_rows(ctx.handle, None, a, p, 0, p, 2, None, None, 1.0, p, None, b) == accb.EINVAL
        assert L.accb_distill_rows_backward(ctx.handle, None, a, p, 0, p, 2, None, None, 1.0, p, None, b) == accb.EINVAL
    x = rows(1024)
    for i in range(3):
        v = [off if i == j else p for j in range(3)]
        assert L.accb_top_rows(ctx.handle, None, x, 1.0, 2, *v) == accb.EINVAL
    for i in range(8):
        v = [off if i == j else p for j in range(8)]
        assert L.accb_sample_rows(ctx.handle, None, x, v[0], 1, *v[1:]) == accb.EINVAL
    assert L.accb_sample_rows(ctx.handle, None, x, p, 1 << 60, *([p] * 7)) == accb.EINVAL
    for i in range(6):
        v = [off if i == j else p for j in range(6)]
        assert L.accb_distill_rows(ctx.handle, None, x, v[0], 0, v[1], 2, v[2], v[3], 1.0, v[4], v[5], None) == accb.EINVAL
        assert L.accb_distill_rows_backward(ctx.handle, None, x, v[0], 0, v[1], 2, v[2], v[3], 1.0, v[4], v[5], rows(2048)) == accb.EINVAL
    ctx.sync()


# ------------------------------------------------------------ refusals
def test_refusals_of_the_library(accb, ctx, torch_cuda):
    t = torch_cuda
    L = accb.lib()
    import ctypes as C
    x, out = t.zeros(2, 8, device="cuda"), t.zeros(64, device="cuda")
    p, q = C.c_void_p(x.data_ptr()), C.c_void_p(out.data_ptr())
    array = lambda ptr=x.data_ptr(), kind=0, cols=8, rows=2, pitch=8: C.byref(accb.accb_rows_array(ptr, kind, cols, rows, pitch))  # noqa: E731
    top_call = lambda a, tau=1.0, k=2, v=q, i=q: L.accb_top_rows(ctx.handle, None, a, tau, k, v, i, None)  # noqa: E731
    for bad in (array(kind=3), array(rows=-1), array(cols=(1 << 20) + 1, pitch=1 << 21), array(pitch=7), array(ptr=None),
                array(ptr=x.data_ptr() + 2), array(rows=1 << 40), array(rows=1 << 20, pitch=1 << 50), None):
        assert top_call(bad) == accb.EINVAL
        assert L.accb_last_error(ctx.handle)
        assert L.accb_sample_rows(ctx.handle, None, bad, None, 0, p, None, None, None, None, q, None) == accb.EINVAL
        assert L.accb_distill_rows(ctx.handle, None, bad, p, 0, p, 2, None, None, 1.0, q, None, None) == accb.EINVAL
    assert top_call(array(cols=0)) == accb.EBOUNDS
    for bad in (dict(k=0), dict(k=9), dict(tau=0.0), dict(tau=-1.0), dict(tau=float("nan")), dict(tau=float("inf")), dict(v=None), dict(i=None)):
        assert top_call(array(), **bad) == accb.EINVAL
    assert L.accb_top_rows(None, None, array(), 1.0, 1, q, q, None) == accb.EINVAL
    assert L.accb_sample_rows(ctx.handle, None, array(), None, 0, None, None, None, None, None, q, None) == accb.EINVAL
    assert L.accb_sample_rows(ctx.handle, None, array(), None, 0, p, None, None, None, None, None, None) == accb.EINVAL
    assert L.accb_sample_rows(ctx.handle, None, array(), p, 0, p, None, None, None, None, q, None) == accb.EINVAL
    d = lambda teacher=p, kind=0, index=p, k=2, tau=1.0, loss=q, grad=None: L.accb_distill_rows(  # noqa: E731
        ctx.handle, None, array(), teacher, kind, index, k, None, None, tau, loss, None, grad)
    for bad in (dict(teacher=None), dict(kind=9), dict(index=None), dict(k=0), dict(k=1025), dict(tau=0.0), dict(loss=None),
                dict(grad=array(cols=7)), dict(grad=array(rows=1)), dict(grad=array(kind=2)), dict(grad=array(ptr=None))):
        assert d(**bad) == accb.EINVAL
    b = lambda stats=p, grad=array(): L.accb_distill_rows_backward(ctx.handle, None, array(), p, 0, p, 2, None, None, 1.0, stats, None, grad)  # noqa: E731
    assert b(stats=None) == accb.EINVAL and b(grad=None) == accb.EINVAL
    ctx.sync()  # and nothing was launched that could have failed
