"""What a weight of grx_kv8_attend is held to: many small ones beside a large
one are not lost, and pages of large values that a query hardly looks at cost
the others nothing. Against the definition in 64 bits, within what 32-bit
sums of weights held to a relative 2^-22 (float16 outputs: 2^-12) allow.

A row's error, with p_j the softmax and v_j the values of the n keys it sees:
  Σ p_j |v_j| · (2·ds + 2^-20 + (n/16 + 32)·2^-23) + n·2^-32·127·max p_j s_j
The score is off by ds (kv8_ref.attend has the terms) in p and in the sum that
divides it; a weight by ex2's 2^-22 and its own two halves' 2^-22, doubled for
the sum's; sums by a step (2^-23) of what they hold for each of n/16 products
and of the joins. The last term is what weights far below the largest product
of a softmax weight and a value scale are held to (half a step of 2^-32 of a unit
that is up to twice it).

The log-sum-exp is off by as much as the scores are, ds (a mean of theirs, and
the query's largest value of 80 leaves 80·2^-23 of every product here), and by
the roundings of a score and a logarithm of up to |lse| + 8."""

import numpy as np
import pytest
import torch

from tests.kv8_ref import EPS2, TORCH
from tests.test_gpu_kv8 import DEV, Side, stream, up

pytestmark = pytest.mark.gpu


def expected(s, i, q, scale, window, dtype):
    """Rows of sequence i that are looked at, and out, lse and the bounds there."""
    k, v = s.ref.values(s.table[i], s.lens[i], 0), s.ref.values(s.table[i], s.lens[i], 1)
    sv = np.abs(s.ref.scale[s.table[i][:-(-s.lens[i] // s.page)], :, 1].astype(np.float64)).repeat(s.page, 0)
    out, lse, tol, score = np.zeros(q.shape), np.zeros(q.shape[:2]), np.zeros(q.shape), np.zeros(q.shape[:2])
    t, heads, _ = q.shape
    checked = range(t) if s.lens[i] < 2000 else sorted({0, t // 2, t - 1})  # of long sequences three rows
    for r in checked:
        p = s.lens[i] - t + r
        lo = max(0, p - window + 1) if window else 0
        for h in range(heads):
            hk = h * s.heads // heads
            kk, vv = k[hk, lo:p + 1], v[hk, lo:p + 1]
            x = kk @ q[r, h].astype(np.float64) * scale
            e = np.exp(x - x.max())
            w, n = e / e.sum(), len(x)
            out[r, h], lse[r, h] = w @ vv, x.max() + np.log(e.sum())
            # of the keys whose softmax is above 2^-60 (the others' errors are theirs)
            near = w > 2.0**-60
            ds = (2.0**-22 * np.abs(q[r, h]).max() * np.abs(kk[near]).sum(1).max() * abs(scale)
                  + 4 * 2.0**-24 * np.abs(x[near]).max())
            score[r, h] = ds
            half = 2.0**-11 if dtype != "f32" else 0.0
            tol[r, h] = (w @ np.abs(vv) * (2 * ds + 2.0**-20 + half + (n / 16 + 32) * 2.0**-23)
                         + n * 2.0**-32 * 127 * (w * sv[lo:p + 1, hk]).max())
    tol += EPS2[dtype] * np.abs(out) * (dtype != "f32")
    return list(checked), out, lse, tol, score + 2.0**-19 * (np.abs(lse) + 8)


def check(s, heads, dtype, q, scale=1.0, window=0):
    dt = getattr(torch, TORCH[dtype])
    dq, out = up(q).to(dt), torch.full((s.rows, heads, s.d), 7.0, dtype=dt, device=DEV)
    lse = torch.full((s.rows, heads), 7.0, device=DEV)
    s.kv.attend(s.seqs(), heads, dq.data_ptr(), out.data_ptr(), dtype=dtype, scale=scale, window=window,
                d_lse=lse.data_ptr(), stream=stream())
    got, gl, qs = out.double().cpu().numpy(), lse.double().cpu().numpy(), dq.double().cpu().numpy()
    for i in range(len(s.lens)):
        a, b = s.row0[i], s.row0[i + 1]
        rows, want, wl, tol, ltol = expected(s, i, qs[a:b], scale, window, dtype)
        want, wl, tol, ltol = want[rows], wl[rows], tol[rows], ltol[rows]
        err = np.abs(got[a:b][rows] - want)
        assert (err <= tol).all(), (i, np.nanmax(err / np.maximum(tol, 1e-300)), np.nanmax(err), np.isnan(err).sum())
        assert (np.abs(gl[a:b][rows] - wl) <= ltol).all()
    assert s.status.item() == 0


SHAPES = [(1, 1, 1), (4, 1, 1), (2, 1, 6), (4, 1, 7), (1, 1, 40), (3, 1, 50)]  # heads, key heads, new tokens


@pytest.mark.parametrize("heads,kv_heads,new", SHAPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("below", [11.0, 16.6, 17.4])
@pytest.mark.parametrize("values", ["alike", "apart"])
def test_many_small_weights_beside_a_large_one(have_gpu, heads, kv_heads, new, d, dtype, below, values):
    """One key that a query likes, and thousands `below` nats under it: their
    common weight (up to a tenth of the sum, a few thousandths at 16.6) is in
    the output as it is in the sum that divides it."""
    n = 32768
    s = Side([n], [new], heads=kv_heads, d=d, page=64, seed=1)
    s.ref.k[:] = 0
    s.ref.v[:] = 100
    s.ref.scale[:] = 0.01
    first = s.table[0][0]
    s.ref.k[first, :, 0, 0] = 100  # 1 in value 0
    if values == "apart":
        s.ref.v[first, :, 0] = 0
    s.upload()
    q = np.zeros((new, heads, d), np.float32)
    q[..., 0] = below
    check(s, heads, dtype, q)


@pytest.mark.parametrize("heads,kv_heads,new", SHAPES)
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("at", [0, 3, -1])
@pytest.mark.parametrize("window", [0, 40])
def test_large_values_that_are_not_looked_at(have_gpu, heads, kv_heads, new, d, page, dtype, at, window):
    """A page whose values are 2^20 times the others' and whose scores are 80
    nats below them: first, in the middle or last, seen by all queries or,
    through a window, by some."""
    s = Side([450, 321], [new, new], heads=kv_heads, d=d, page=page, seed=5)
    s.ref.k[..., 0] = 0
    for row, m in zip(s.table, s.lens):
        p = row[:-(-m // page)][at]
        s.ref.scale[p, :, 1] *= 2.0**20
        s.ref.k[p, :, :, 0] = -127
        s.ref.scale[p, :, 0] = 1 / 127
    # the last token of a sequence has itself to look at, on whichever page
    s.upload()
    q = s.rng.normal(0, 0.1, (s.rows, heads, d)).astype(np.float32)
    q[..., 0] = 80
    check(s, heads, dtype, q, window=window)


@pytest.mark.parametrize("heads,kv_heads,new", SHAPES)
@pytest.mark.parametrize("size", [1e-30, 1e30])
@pytest.mark.parametrize("order", [1, -1])
def test_values_of_any_size(have_gpu, heads, kv_heads, new, size, order):
    """All values tiny or huge, pages' scales growing or falling by 2^4 each
    over a factor of 2^40."""
    s = Side([170], [new], heads=kv_heads, d=64, page=16, seed=7)
    row = s.table[0][::order]
    s.ref.scale[row, :, 1] *= (np.float32(size) * 2.0 ** (4 * np.arange(len(row)) - 20)).astype(np.float32)[:, None]
    s.upload()
    check(s, heads, "f32", s.rng.normal(0, 1, (s.rows, heads, 64)).astype(np.float32), scale=0.125)
