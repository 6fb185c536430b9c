"""grx_logprobs on a B200 against 64-bit numpy. Ids are compared exactly,
numbers within the roundings of 32-bit sums of positive terms (bound)."""

import numpy as np
import pytest
import torch

import gorelaxor_b200 as g
from tests.kv8_ref import TORCH

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def reference(x, targets, top):
    """x [rows][vocab] float64 (the logits' exact values)."""
    with np.errstate(invalid="ignore", divide="ignore"):
        m = x.max(1, keepdims=True)
        fine = np.isfinite(m[:, 0])
        e = np.exp(x - m)
        at = np.argmax(x, 1)
        rest = e.copy()
        rest[np.arange(len(x)), at] = 0
        z = rest.sum(1)
        lz = np.log1p(z)
        gap = np.where(e > 0, (m - x) * e, 0).sum(1)
        entropy = lz + gap / (1 + z)
        lp = x - m - lz[:, None]
    lp[~fine], entropy[~fine] = np.nan, np.nan
    ok = (targets >= 0) & (targets < x.shape[1])
    tl = np.where(ok, lp[np.arange(len(x)), np.where(ok, targets, 0)], np.nan)
    # the larger value first, then the lower index; NaN last
    keys = np.where(np.isnan(x), np.inf, -x)
    nan = np.isnan(x)
    ids = np.stack([np.lexsort((np.arange(x.shape[1]), keys[r], nan[r]))[:top] for r in range(len(x))]) \
        if top else np.zeros((len(x), 0), int)
    return tl, entropy, ids, np.take_along_axis(lp, ids, 1)


def bound(lp, vocab):
    """Roundings of a log probability or an entropy: the difference to the
    largest logit (2^-24 of it), and the sums: an exponential is off by ex2's
    2^-22 and by its argument's two roundings (2^-23 of a gap d that counts
    e^-d: at most 2^-23), a sum of positive terms by 2^-24 for every addition
    behind another, at most vocab/256 + 24 of them."""
    rel = 2.0**-22 + 2.0**-23 + (vocab / 256 + 24) * 2.0**-24
    return 2.0**-23 * np.abs(lp) + rel * np.maximum(np.minimum(np.abs(lp), 1.0), 0)


def call(x, targets, top, dtype="f32", stride=None, offset=0, **kw):
    dt = getattr(torch, TORCH[dtype])
    r, v = x.shape
    stride = stride or v
    buf = torch.full((offset + max(r, 1) * stride,), 99.0, dtype=dt, device=DEV)
    view = buf[offset:].view(-1, stride)[:r, :v]
    view.copy_(torch.from_numpy(x).to(DEV))
    t = torch.from_numpy(targets.astype(np.int32)).to(DEV)
    lp, en = torch.full((r + 1,), 5.0, device=DEV), torch.full((r + 1,), 5.0, device=DEV)
    ids, tl = torch.full((r + 1, top), 5, dtype=torch.int32, device=DEV), torch.full((r + 1, top), 5.0, device=DEV)
    a = dict(d_targets=t.data_ptr(), top=top, d_logprob=lp.data_ptr(), d_entropy=en.data_ptr(),
             d_top_ids=ids.data_ptr() if top else None, d_top_logprobs=tl.data_ptr() if top else None)
    g.logprobs(view.data_ptr(), r, v, dtype=dtype, row_stride=stride,
               stream=torch.cuda.current_stream().cuda_stream, **{**a, **kw})
    exact = view.double().cpu().numpy()
    for o in (lp, en, ids, tl):
        assert (o[r:] == 5).all()
    return [o[:r].cpu().numpy() for o in (lp, en, ids, tl)], exact


def check(x, targets, top, **kw):
    (lp, en, ids, tl), exact = call(x, targets, top, **kw)
    wl, we, wi, wt = reference(exact, targets, top)
    assert np.array_equal(ids, wi)
    v = x.shape[1]
    for got, want, name in ((lp, wl, "logprob"), (en, we, "entropy"), (tl, wt, "top")):
        # a log probability below the lowest 32-bit number (-6e38) is -inf there
        want = np.where(want < -3.4028236e38, -np.inf, want)
        fin = np.isfinite(want)
        assert np.array_equal(got[~fin], want[~fin], equal_nan=True), name
        # an entropy counts each gap twice: in the exponential and before it
        off = np.abs(got[fin] - want[fin])
        tol = bound(want[fin], v) * (4 if name == "entropy" else 1) + 2.0**-126
        assert (off <= tol).all(), (name, off.max(), tol[np.argmax(off - tol)], want[fin][np.argmax(off - tol)])
    return lp, en, ids, tl


SIZES = [(1, 1), (3, 2), (2, 31), (5, 32), (4, 33), (9, 511), (7, 513), (3, 1030), (11, 1281), (2, 2048), (3, 2049),
         (2, 4093), (5, 16383), (2, 16385), (1, 51864), (33, 51865), (2, 100003)]


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_sizes(have_gpu, rows, vocab, dtype, top):
    rng = np.random.default_rng(rows * vocab + top)
    x = rng.normal(0, 3, (rows, vocab)).astype(np.float32)
    x[rng.random(x.shape) < 0.02] = -np.inf
    x[:, rng.integers(0, vocab)] = 4  # at least one finite logit a row
    check(x, rng.integers(0, vocab, rows), min(top, vocab), dtype=dtype)


@pytest.mark.parametrize("vocab", [2049, 4100, 9001, 24576, 24577])
@pytest.mark.parametrize("dtype,top", [("f32", 5), ("f16", 32), ("bf16", 0), ("f32", 32), ("bf16", 1)])
def test_many_rows(have_gpu, vocab, dtype, top):
    """Enough rows that smaller blocks take them, around the longest that do;
    a few with equal values, masked values or none that is a number."""
    rng = np.random.default_rng(vocab + top)
    rows = 310 if vocab < 9001 else 297
    x = rng.normal(0, 3, (rows, vocab)).astype(np.float32)
    x[3] = 1.5                        # all alike
    x[4, 10:] = -np.inf
    x[5] = np.round(x[5])             # many alike
    x[6, 7], x[7, vocab - 1] = np.nan, np.inf
    x[8] = -np.inf
    x[9, vocab - 1] = 60000.0
    with np.errstate(invalid="ignore"):
        check(x, rng.integers(0, vocab, rows), top, dtype=dtype, stride=vocab + 3, offset=1)


@pytest.mark.parametrize("vocab", [50, 1030, 3001, 40000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides_and_offsets(have_gpu, vocab, dtype):
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 3, (6, vocab)).astype(np.float32)
    for offset, pad in ((0, 8), (1, 0), (3, 5), (7, 1)):
        check(x, rng.integers(0, vocab, 6), 4, dtype=dtype, offset=offset, stride=vocab + pad)


@pytest.mark.parametrize("vocab", [40, 1500, 9000, 60000])
def test_ties(have_gpu, vocab):
    """Equal logits: the lower index first; a row of one value throughout,
    more equals than any list of candidates takes, and 0 beside −0."""
    rng = np.random.default_rng(vocab)
    x = rng.integers(0, 3, (6, vocab)).astype(np.float32)
    x[0] = 0
    x[1] = -7.5
    x[2] = np.where(np.arange(vocab) % 2, 0.0, -0.0)
    x[3] = np.arange(vocab) // 40  # rising: every value a new largest
    x[4] = -(np.arange(vocab) // 3)
    check(x, rng.integers(0, vocab, 6), 32)


@pytest.mark.parametrize("vocab", [37, 1030, 5000, 51864])
def test_sure_rows_keep_their_small_numbers(have_gpu, vocab):
    """One logit far above the rest: log probabilities of −1e-3 to −1e-30
    and entropies as small, to 32 bits of themselves."""
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 1, (6, vocab)).astype(np.float32)
    t = rng.integers(0, vocab, 6)
    x[np.arange(6), t] = [15, 20, 30, 45, 60, 80]
    lp, en, _, _ = check(x, t, 3)
    assert (lp < 0).all() and (en > 0).all()
    # and logits of any size: only their differences count
    check(x + 4096, t, 3)


@pytest.mark.parametrize("vocab", [37, 1030, 5000, 51864])
def test_masks_and_numbers_that_are_none(have_gpu, vocab):
    rng = np.random.default_rng(vocab)
    x = rng.normal(0, 2, (9, vocab)).astype(np.float32)
    x[0] = -np.inf                    # nothing allowed
    x[1] = -np.inf
    x[1, vocab // 2] = 1              # one token allowed
    x[2, 5] = np.nan
    x[3, 7] = np.inf
    x[4] = np.nan
    x[5, ::2] = -np.inf
    x[6] = -3.4028235e38              # a mask of the type's lowest value
    x[6, :3] = 2
    x[7, 0], x[7, 1] = 3e38, -3e38    # a gap past the largest number
    t = np.array([0, vocab // 2, 1, 7, 3, 0, 9, 1, -1])
    lp, en, ids, _ = check(x, t, 6)
    assert lp[1] == 0 and en[1] == 0 and np.isneginf(lp[5]) and np.isnan(lp[8])
    assert np.isnan(lp[[0, 2, 3, 4]]).all() and np.isnan(en[[0, 2, 3, 4]]).all()
    assert ids[0].tolist() == list(range(6)) and ids[3, 0] == 7


def test_targets_outside(have_gpu):
    x = np.zeros((4, 100), np.float32)
    (lp, en, _, _), _ = call(x, np.array([-1, 100, 2**31 - 1, 99]), 0)
    assert np.isnan(lp[:3]).all() and abs(lp[3] + np.log(100)) < 1e-6 and np.isfinite(en).all()


def test_outputs_left_out(have_gpu):
    """Each output by itself gives what all together give."""
    rng = np.random.default_rng(0)
    for vocab in (700, 5000):
        x, t = rng.normal(0, 3, (5, vocab)).astype(np.float32), rng.integers(0, vocab, 5)
        every, _ = call(x, t, 4)
        none = dict(d_logprob=None, d_entropy=None, d_top_ids=None, d_top_logprobs=None)
        for i, name in enumerate(none):
            kw = {k: v for k, v in none.items() if k != name}
            part, _ = call(x, t, 4, **kw)
            assert np.array_equal(part[i], every[i])


def test_same_bits_again_and_in_a_graph(have_gpu):
    rng = np.random.default_rng(1)
    for rows, vocab in ((1, 51864), (300, 3001), (40, 1030)):
        x, t = rng.normal(0, 3, (rows, vocab)).astype(np.float32), rng.integers(0, vocab, rows)
        first, _ = call(x, t, 8)
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            again, _ = call(x, t, 8)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))
        dx, dt = torch.zeros(rows, vocab, device=DEV), torch.from_numpy(t.astype(np.int32)).to(DEV)
        lp = torch.zeros(rows, device=DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            g.logprobs(dx.data_ptr(), rows, vocab, d_targets=dt.data_ptr(), d_logprob=lp.data_ptr(),
                       stream=torch.cuda.current_stream().cuda_stream)
        dx.copy_(torch.from_numpy(x))
        graph.replay()
        assert np.array_equal(lp.cpu().numpy(), first[0])


def test_many_rows_past_32_bits(have_gpu):
    """Rows whose offsets pass 2^32 elements."""
    rows, vocab = 70000, 61440
    if torch.cuda.mem_get_info()[0] < 10 << 30:
        pytest.skip("not enough device memory")
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device=DEV)
    x[-1, 61000], x[-1, 7] = 9.0, 8.0
    t = torch.full((rows,), 61000, dtype=torch.int32, device=DEV)
    lp, ids = torch.zeros(rows, device=DEV), torch.zeros(rows, 2, dtype=torch.int32, device=DEV)
    g.logprobs(x.data_ptr(), rows, vocab, dtype="bf16", d_targets=t.data_ptr(), d_logprob=lp.data_ptr(), top=2,
               d_top_ids=ids.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    z = 61438 * np.exp(-9.0) + np.exp(-1.0)
    assert abs(lp[-1].item() + np.log1p(z)) < 1e-5 and ids[-1].tolist() == [61000, 7]
    assert abs(lp[0].item() + np.log(61440)) < 1e-5 and ids[0].tolist() == [0, 1]
