"""grx_kv8_append, grx_kv8_read and grx_kv8_attend on a B200 against the
64-bit model of tests/kv8_ref.py. The cache's bytes and scales are compared
bit for bit (they are rounded in 64 bits), attention within a bound that
kv8_ref.attend computes with the result, plus half a step of a 16-bit output
type."""

import numpy as np
import pytest
import torch

import gorelaxor_b200 as g
from tests.kv8_ref import EPS2, TORCH, Cache, attend, rope_table

pytestmark = pytest.mark.gpu
ERANGE = -5
DEV = "cuda:0"


def up(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(DEV)


def stream():
    return torch.cuda.current_stream().cuda_stream


class Side:
    """A cache on both sides, with a scattered page table for sequences."""

    def __init__(self, lens, new, heads=2, d=64, page=16, seed=0, mode="none", spare=3, filled=True, positions=None):
        self.rng = np.random.default_rng(seed)
        self.lens, self.new, self.d, self.page, self.heads, self.mode = list(lens), list(new), d, page, heads, mode
        n = len(lens)
        width = max(1, max(-(-m // page) for m in lens))
        need = [-(-m // page) for m in lens]
        self.pages = sum(need) + spare
        order = self.rng.permutation(self.pages)
        self.table = np.full((n, width), -7, np.int32)
        at = 0
        for i, c in enumerate(need):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.ref = Cache(self.pages, heads, page, d, self.rng if filled else None)
        self.rope = rope_table(positions or width * page, d)
        self.row0 = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        self.rows = int(self.row0[-1])
        self.upload()

    def upload(self):
        self.k, self.v, self.s = up(self.ref.k), up(self.ref.v), up(self.ref.scale)
        self.t, self.n, self.r = up(self.table), up(np.array(self.lens, np.int32)), up(self.row0)
        self.cs = up(self.rope)
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.kv = g.KV8(self.k.data_ptr(), self.v.data_ptr(), self.s.data_ptr(), self.pages, self.page, self.heads,
                        self.d)

    def seqs(self, **kw):
        a = dict(n=len(self.lens), d_table=self.t.data_ptr(), table_width=self.table.shape[1],
                 d_len=self.n.data_ptr(), max_len=max(self.lens), d_row0=self.r.data_ptr(), rows=self.rows,
                 max_new=max(self.new), d_rope=self.cs.data_ptr(), rope_positions=len(self.rope), rope=self.mode,
                 d_status=self.status.data_ptr())
        return g.KV8Seqs(**{**a, **kw})

    def append(self, kv=None, dtype="f32", **kw):
        """Rows [rows][2][heads][d] to both sides; the device's as they are strided."""
        if kv is None:
            kv = self.rng.normal(0, 1, (self.rows, 2, self.heads, self.d)).astype(np.float32)
        x = up(kv).to(getattr(torch, TORCH[dtype]))
        size, hd = x.element_size(), self.heads * self.d
        self.kv.append(self.seqs(**kw), x.data_ptr(), x.data_ptr() + hd * size, dtype=dtype,
                       k_strides=(2 * hd, self.d), v_strides=(2 * hd, self.d), stream=stream())
        x = x.float().cpu().numpy()
        for i, m in enumerate(self.lens):
            a, b = self.row0[i], self.row0[i + 1]
            if b > a:
                self.ref.append(self.table[i], m, x[a:b, 0], x[a:b, 1], self.rope, self.mode)

    def same(self):
        assert torch.equal(self.k.cpu(), torch.from_numpy(self.ref.k)), "keys"
        assert torch.equal(self.v.cpu(), torch.from_numpy(self.ref.v)), "values"
        got, want = self.s.cpu().numpy(), self.ref.scale
        assert np.array_equal(got, want, equal_nan=True), "scales"

    def attend(self, heads, dtype="f32", window=0, first=None, sharp=1.5, offset=0, want_tol=1.0, q=None, seqs=None,
               **kw):
        dt = getattr(torch, TORCH[dtype])
        if q is None:
            q = self.rng.normal(0, sharp, (self.rows, heads, self.d)).astype(np.float32)
        qd = torch.zeros(q.size + offset, dtype=dt, device=DEV)
        qd[offset:] = up(q).to(dt).flatten()
        out = torch.full((self.rows + 2, heads, self.d), 7.0, dtype=dt, device=DEV)
        lse = torch.full((self.rows + 2, heads), 7.0, device=DEV)
        f = up(np.array(first, np.int32)) if first is not None else None
        sq = seqs or self.seqs(d_first=f.data_ptr() if f is not None else None, **kw)
        self.kv.attend(sq, heads, qd.data_ptr() + offset * qd.element_size(), out.data_ptr(), dtype=dtype,
                       window=window, d_lse=lse.data_ptr(), stream=stream())
        qs = qd[offset:].float().cpu().numpy().reshape(q.shape)
        got, gl = out.float().cpu().numpy(), lse.cpu().numpy()
        assert (got[self.rows:] == 7).all() and (gl[self.rows:] == 7).all(), "rows behind the last sequence"
        for i, m in enumerate(self.lens):
            a, b = self.row0[i], self.row0[i + 1]
            if b == a:
                continue
            want, wl, tol = attend(self.ref, self.table[i], m, qs[a:b], self.rope, self.mode, window=window,
                                   first=first[i] if first is not None else 0, half=dtype != "f32")
            tol = tol[..., None] + EPS2[dtype] * np.abs(want) * (dtype != "f32") + 2.0**-24 * (dtype == "f16")
            bad = ~(np.abs(got[a:b] - want) <= tol * want_tol)
            bad &= ~(np.isnan(want) & np.isnan(got[a:b]))
            assert not bad.any(), (i, m, np.argwhere(bad)[:3], np.abs(got[a:b] - want).max(), tol.max())
            fin = np.isfinite(wl)
            assert np.array_equal(gl[a:b][~fin], wl[~fin], equal_nan=True)
            # the largest score's and the sum's roundings, a step each of a score up to |wl| + 8
            assert (np.abs(gl[a:b][fin] - wl[fin]) <= 2.0**-19 * (np.abs(wl[fin]) + 8)).all()
        return got[:self.rows], gl[:self.rows]


# ------------------------------------------------------------- append


@pytest.mark.parametrize("d,page", [(64, 16), (64, 64), (128, 16), (128, 32), (128, 64)])
@pytest.mark.parametrize("mode", ["none", "pairs", "halves"])
def test_append_tokens_one_by_one(have_gpu, d, page, mode):
    """70 steps of single tokens: pages begin, fill and have their scales
    raised; bytes and scales are the definition's after every step."""
    s = Side([70, 70], [1, 1], d=d, page=page, mode=mode, seed=d + page, filled=False)
    big = s.rng.integers(0, 70, 6)
    for m in range(1, 71):
        s.lens = [m, m]
        s.n.fill_(m)
        x = s.rng.normal(0, 1, (2, 2, 2, d)).astype(np.float32)
        if m in big:
            x *= 4  # raises the scale in the middle of a page
        s.append(x, d_row0=None)
        if m % 9 == 0 or m == 70:
            s.same()
    s.same()
    assert s.status.item() == 0


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("d,page,heads", [(64, 16, 3), (64, 32, 1), (128, 64, 2), (128, 16, 5)])
def test_append_ragged(have_gpu, dtype, d, page, heads):
    """Rows of several tokens a sequence: none, one, a page's end, several
    pages, from the start and behind held tokens."""
    s = Side([5, 16, 17, 64, 200, 33, 100, 1], [0, 16, 1, 33, 170, 2, 100, 1], heads=heads, d=d, page=page,
             mode="halves", seed=page)
    s.append(dtype=dtype)
    s.same()
    assert s.status.item() == 0


@pytest.mark.parametrize("mode", ["none", "halves"])
@pytest.mark.parametrize("new", [(64, 64), (20, 150)])
def test_append_heads_in_turn(have_gpu, mode, new):
    """So many pages that a block takes several heads of one after another;
    values of very different sizes from head to head."""
    rng = np.random.default_rng(5)
    n = 100
    lens = rng.integers(150, 260, n)
    s = Side(lens.tolist(), rng.integers(new[0], new[1] + 1, n).tolist(), heads=8, d=64, page=64, mode=mode, seed=1)
    kv = s.rng.normal(0, 1, (s.rows, 2, 8, 64)).astype(np.float32) * (4.0 ** np.arange(8, dtype=np.float32))[:, None]
    for _ in range(2):
        s.append(kv[..., ::-1, :].copy())
    s.same()
    assert s.status.item() == 0


def test_append_strides_and_offsets(have_gpu):
    """Heads outermost, and rows that begin off every wide boundary."""
    s = Side([40, 21], [17, 9], heads=3, d=64, mode="pairs", seed=5)
    kv = s.rng.normal(0, 1, (26, 2, 3, 64)).astype(np.float32)
    x = torch.zeros(2 * 3 * 26 * 67 + 1, device=DEV)
    view = x[1:].view(2, 3, 26, 67)[..., :64]
    view.copy_(up(kv).permute(1, 2, 0, 3))
    s.kv.append(s.seqs(), view[0].data_ptr(), view[1].data_ptr(), k_strides=(67, 26 * 67), v_strides=(67, 26 * 67),
                stream=stream())
    for i in range(2):
        a, b = s.row0[i], s.row0[i + 1]
        s.ref.append(s.table[i], s.lens[i], kv[a:b, 0], kv[a:b, 1], s.rope, "pairs")
    s.same()


def test_append_zeros_tiny_and_not_finite(have_gpu):
    s = Side([16, 20, 20, 20, 33], [4, 4, 4, 4, 33], heads=2, d=64, seed=3)
    kv = s.rng.normal(0, 1, (s.rows, 2, 2, 64)).astype(np.float32)
    kv[0:4] = 0                       # nothing larger than what the page holds
    kv[4:8] *= 1e-42                  # below the smallest normal number
    kv[8:12, 0, 1, 3] = np.inf
    kv[12:16, 1, 0, 5] = np.nan
    kv[16:32] = 0                     # a page of zeros from its first token on
    with np.errstate(over="ignore"):
        kv[32:33] *= 3e38             # past the largest number: keys and values of both heads are not finite
    s.append(kv)
    s.same()
    assert np.isnan(s.ref.scale).sum() == 2 + 4
    # a NaN stays until its page begins anew
    s.lens = [16, 20, 21, 21, 33]
    s.n.copy_(torch.tensor(s.lens))
    s.new, s.row0, s.rows = [0, 0, 1, 1, 0], np.array([0, 0, 0, 1, 2, 2], np.int32), 2
    s.r.copy_(torch.from_numpy(s.row0))
    s.append()
    s.same()
    assert np.isnan(s.ref.scale).sum() == 2 + 4
    s.lens, s.new, s.row0 = [16, 20, 17, 17, 33], [0, 0, 1, 1, 0], s.row0
    s.n.copy_(torch.tensor(s.lens))
    s.append()
    s.same()
    assert np.isnan(s.ref.scale).sum() == 4


@pytest.mark.parametrize("mode", ["none", "pairs", "halves"])
def test_append_largest_numbers(have_gpu, mode):
    """Rotated keys pass the largest 32-bit number, their scale does not."""
    s = Side([20], [9], heads=1, d=64, mode=mode, seed=4)
    s.append(np.where(s.rng.random((9, 2, 1, 64)) < 0.5, -1, 1).astype(np.float32) * np.float32(3.4e38))
    s.same()
    assert np.isfinite(s.ref.scale).all()


def test_append_leaves_out_what_does_not_fit(have_gpu):
    """A page that is none, a length past the table, rows past the rows: left
    out and reported; the other sequences are appended as ever. (The host's
    check of the same arrays is in test_kv8.py.)"""
    s = Side([20, 20, 20, 20, 20], [3, 3, 3, 3, 3], seed=9)
    kv = s.rng.normal(0, 1, (s.rows, 2, 2, 64)).astype(np.float32)
    t, lens, row0 = s.table.copy(), list(s.lens), s.row0.copy()
    s.t[1, 1] = s.pages
    s.n[2] = 33
    s.n[3] = -4
    s.r[5] = 16
    keep = [0]
    x = up(kv)
    s.kv.append(s.seqs(), x.data_ptr(), x.data_ptr() + 512, k_strides=(256, 64), v_strides=(256, 64), stream=stream())
    for i in keep:
        s.ref.append(t[i], lens[i], kv[row0[i]:row0[i + 1], 0], kv[row0[i]:row0[i + 1], 1])
    s.same()
    assert s.status.item() == ERANGE


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read(have_gpu, dtype):
    s = Side([5, 50, 0, 130], [5, 17, 0, 130], heads=3, d=128, page=32, seed=2)
    dt = getattr(torch, TORCH[dtype])
    k = torch.full((s.rows + 1, 3, 128), 9.0, dtype=dt, device=DEV)
    v = torch.full((3, s.rows + 1, 128), 9.0, dtype=dt, device=DEV)
    s.kv.read(s.seqs(), k.data_ptr(), v.data_ptr(), dtype=dtype, v_strides=(128, (s.rows + 1) * 128), stream=stream())
    for i, m in enumerate(s.lens):
        a, b = s.row0[i], s.row0[i + 1]
        for j, got in ((0, k[a:b].permute(1, 0, 2)), (1, v[:, a:b])):
            p = s.table[i][:-(-m // 32)]
            # byte times scale in 32 bits, then the type's rounding: the same bits
            raw = torch.from_numpy((s.ref.k, s.ref.v)[j][p]).float() * torch.from_numpy(s.ref.scale[p][..., j, None, None])
            want = raw.permute(1, 0, 2, 3).reshape(3, -1, 128)[:, m - (b - a):m].to(dt)
            assert torch.equal(got.cpu(), want)
    assert (k[-1] == 9).all() and (v[:, -1] == 9).all()
    one = torch.empty_like(k)
    s.kv.read(s.seqs(), None, one.data_ptr(), dtype=dtype, stream=stream())  # values alone
    assert torch.equal(one[:-1].permute(1, 0, 2), v[:, :-1])


# ------------------------------------------------------------- attend

LENGTHS = [1, 2, 15, 16, 17, 31, 33, 64, 65, 127, 129, 257, 700]


@pytest.mark.parametrize("d,page", [(64, 16), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (3, 1), (20, 2), (33, 3)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_attend_single_tokens(have_gpu, d, page, heads, kv_heads, dtype):
    s = Side(LENGTHS, [1] * len(LENGTHS), heads=kv_heads, d=d, page=page, mode="pairs", seed=heads)
    s.attend(heads, dtype)
    assert s.status.item() == 0


@pytest.mark.parametrize("d,page,heads,kv_heads,mode", [(64, 16, 2, 2, "pairs"), (64, 32, 6, 2, "halves"),
                                                        (128, 64, 4, 1, "halves"), (128, 16, 2, 2, "none")])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("window", [0, 1, 16, 45])
def test_attend_several_tokens(have_gpu, d, page, heads, kv_heads, mode, dtype, window):
    """Prompts, and a few tokens at a time, behind what the cache holds; with
    windows smaller and larger than a block's queries."""
    s = Side([1, 70, 129, 40, 300, 18], [1, 70, 100, 3, 5, 0], heads=kv_heads, d=d, page=page, mode=mode, seed=page)
    s.attend(heads, dtype, window=window)


@pytest.mark.parametrize("new", [[1, 1, 1, 1, 1, 1], [3, 40, 1, 17, 64, 9]])
def test_attend_first_keys(have_gpu, new):
    """Left padding: some queries see no key (zeros, −inf), some one."""
    s = Side([3, 40, 20, 80, 64, 90], new, heads=2, d=64, mode="pairs", seed=11)
    got, lse = s.attend(4, first=[3, 39, -5, 1 << 30, 50, 88])
    assert (got[:s.row0[1]] == 0).all() and np.isneginf(lse[:s.row0[1]]).all()


def test_attend_slots_without_tokens(have_gpu):
    """len 0 in a call of one row for each sequence: zeros and −inf, and
    nothing is appended."""
    s = Side([0, 5, 0, 40], [1, 1, 1, 1], seed=4)
    kv = s.rng.normal(0, 1, (4, 2, 2, 64)).astype(np.float32)
    x = up(kv)
    s.kv.append(s.seqs(d_row0=None), x.data_ptr(), x.data_ptr() + 512, k_strides=(256, 64), v_strides=(256, 64),
                stream=stream())
    for i in (1, 3):
        s.ref.append(s.table[i], s.lens[i], kv[i:i + 1, 0], kv[i:i + 1, 1])
    s.same()
    got, lse = s.attend(2, d_row0=None)
    assert (got[[0, 2]] == 0).all() and np.isneginf(lse[[0, 2]]).all()
    assert s.status.item() == 0


@pytest.mark.parametrize("hint", [0, 100, 1 << 20])
def test_attend_any_split(have_gpu, hint):
    """max_len decides how the keys are split, not what comes out."""
    s = Side([3000, 1, 40, 1500], [1, 1, 1, 1], heads=1, d=128, page=64, mode="halves", seed=8)
    s.attend(4, "f32", max_len=hint)
    s = Side([2000, 45], [9, 45], heads=1, d=64, page=16, seed=8)
    s.attend(1, "f32", max_len=hint)


def test_attend_sharp_and_flat(have_gpu):
    """Scores of hundreds (the running maximum moves, all weights but one
    vanish), growing along the keys, and scores of zero."""
    for sharp in (60.0, 0.0):
        s = Side([900, 700], [1, 40], heads=2, d=64, seed=21)
        s.attend(2, sharp=sharp)
    s = Side([800], [2], heads=1, d=64, page=16, seed=22)
    s.ref.k[:] = 1
    for b, p in enumerate(s.table[0]):
        s.ref.scale[p, 0, 0] = 0.02 * (b + 1)  # every page's scores above the last's
    s.upload()
    s.attend(1, q=np.ones((2, 1, 64), np.float32))


def test_attend_numbers_that_are_none(have_gpu):
    """A NaN scale matters to the queries that see its page alone; a query
    that is not finite is NaN and no other."""
    s = Side([80, 80], [80, 1], heads=1, d=64, page=16, seed=6)
    s.ref.scale[s.table[0][2]] = np.nan   # positions 32..47
    s.ref.scale[s.table[1][0]] = np.nan   # behind the first key
    s.upload()
    q = s.rng.normal(0, 1, (81, 1, 64)).astype(np.float32)
    q[5, 0, 3], q[6, 0, 3] = np.inf, np.nan
    dq, out = up(q), torch.zeros(81, 1, 64, device=DEV)
    first = up(np.array([0, 16], np.int32))
    s.kv.attend(s.seqs(d_first=first.data_ptr()), 1, dq.data_ptr(), out.data_ptr(), stream=stream())
    nan = torch.isnan(out).all(-1).flatten().cpu().numpy()
    assert (nan == torch.isnan(out).any(-1).flatten().cpu().numpy()).all()
    assert np.flatnonzero(nan).tolist() == [5, 6] + list(range(32, 80))
    with_window = torch.zeros_like(out)
    s.kv.attend(s.seqs(d_first=first.data_ptr()), 1, dq.data_ptr(), with_window.data_ptr(), window=10, stream=stream())
    nan = torch.isnan(with_window).any(-1).flatten().cpu().numpy()
    assert np.flatnonzero(nan).tolist() == [5, 6] + list(range(32, 57))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_strides_and_offsets(have_gpu, dtype):
    """Queries inside a packed row and off wide boundaries; outputs with the
    heads outermost."""
    s = Side([50, 300], [4, 1], heads=2, d=64, mode="halves", seed=13)
    s.attend(4, dtype, offset=1)
    dt = getattr(torch, TORCH[dtype])
    wide = torch.randn(5, 3, 4, 64, device=DEV).to(dt)
    packed = wide[:, 1].contiguous()
    a, b = torch.zeros(5, 4, 64, dtype=dt, device=DEV), torch.zeros(4, 5, 65, dtype=dt, device=DEV)
    s.kv.attend(s.seqs(), 4, packed.data_ptr(), a.data_ptr(), dtype=dtype, stream=stream())
    s.kv.attend(s.seqs(), 4, wide[:, 1].data_ptr(), b.data_ptr(), dtype=dtype, q_strides=(12 * 64, 64),
                out_strides=(65, 5 * 65), stream=stream())
    assert torch.equal(a, b[..., :64].permute(1, 0, 2))
    assert (b[..., 64] == 0).all()


def test_attend_leaves_out_what_does_not_fit(have_gpu):
    """A page that is none is not there (its tokens are masked); a sequence
    whose rows or length do not fit keeps its outputs as they were."""
    s = Side([40, 40, 40, 40], [2, 2, 2, 2], heads=1, d=64, page=16, seed=17)
    q = s.rng.normal(0, 1, (8, 1, 64)).astype(np.float32)
    want0, _, tol0 = attend(s.ref, s.table[0], 40, q[0:2])
    k, v = s.ref.values(s.table[1], 40, 0)[0], s.ref.values(s.table[1], 40, 1)[0]
    s.t[1, 1] = -1
    s.n[2] = 49
    s.r[4] = 9
    dq, out = up(q), torch.full((8, 1, 64), 5.0, device=DEV)
    s.kv.attend(s.seqs(), 1, dq.data_ptr(), out.data_ptr(), stream=stream())
    got = out.cpu().numpy()
    assert (np.abs(got[0:2] - want0) <= tol0[..., None]).all()
    for r in (0, 1):
        see = [j for j in range(39 + r) if not 16 <= j < 32]
        w = np.exp(k[see] @ q[2 + r, 0].astype(np.float64) / 8)
        assert (np.abs(got[2 + r, 0] - w @ v[see] / w.sum()) <= 2 * tol0.max()).all()
    assert (got[4:] == 5).all()
    assert s.status.item() == ERANGE


def test_attend_shared_pages_and_two_calls(have_gpu):
    """Sequences of one beginning share its pages; two calls give the same
    bits, on a stream of their own too."""
    s = Side([64, 80, 75], [1, 1, 1], heads=2, d=64, page=16, seed=31)
    s.table[1, :4] = s.table[0, :4]
    s.table[2, :4] = s.table[0, :4]
    s.upload()
    a, la = s.attend(4, q=np.ones((3, 4, 64), np.float32))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b, lb = s.attend(4, q=np.ones((3, 4, 64), np.float32))
    assert np.array_equal(a, b) and np.array_equal(la, lb)


def test_graph_replays_with_new_lengths(have_gpu):
    """A step captured once and replayed while tokens arrive: lengths and
    rows are read when the kernels run."""
    s = Side([40, 70], [1, 1], heads=2, d=64, page=16, mode="pairs", seed=41)
    s.lens = [3, 31]
    s.n.copy_(torch.tensor(s.lens))
    kv = torch.zeros(2, 2, 2, 64, device=DEV)
    q, out = torch.zeros(2, 4, 64, device=DEV), torch.zeros(2, 4, 64, device=DEV)
    sq = s.seqs(d_row0=None, max_len=70)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = stream()
        s.kv.append(sq, kv.data_ptr(), kv.data_ptr() + 512, k_strides=(256, 64), v_strides=(256, 64), stream=st)
        s.kv.attend(sq, 4, q.data_ptr(), out.data_ptr(), stream=st)
    for step in range(25):
        s.lens = [3 + step, 31 + step]
        x = s.rng.normal(0, 1, (2, 2, 2, 64)).astype(np.float32)
        y = s.rng.normal(0, 1.5, (2, 4, 64)).astype(np.float32)
        s.n.copy_(torch.tensor(s.lens))
        kv.copy_(up(x))
        q.copy_(up(y))
        graph.replay()
        got = out.cpu().numpy()
        for i in range(2):
            s.ref.append(s.table[i], s.lens[i], x[i:i + 1, 0], x[i:i + 1, 1], s.rope, "pairs")
            want, _, tol = attend(s.ref, s.table[i], s.lens[i], y[i:i + 1], s.rope, "pairs")
            assert (np.abs(got[i:i + 1] - want) <= tol[..., None]).all(), step
    s.same()


def test_offsets_past_32_bits(have_gpu):
    """Pages behind the first 2^32 bytes of the keys and of the values."""
    pages = (1 << 32) // (8 * 64 * 128) + 40
    if torch.cuda.mem_get_info()[0] < 3 * pages * 8 * 64 * 128:
        pytest.skip("not enough device memory")
    s = Side([200, 64], [3, 64], heads=8, d=128, page=64, mode="halves", seed=51)
    n = s.pages
    k = torch.empty((pages, 8, 64, 128), dtype=torch.int8, device=DEV)
    v = torch.empty_like(k)
    sc = torch.zeros((pages, 8, 2), device=DEV)
    k[-n:], v[-n:], sc[-n:] = s.k, s.v, s.s
    s.k, s.v, s.s = k[-n:], v[-n:], sc[-n:]
    s.t += pages - n
    s.kv = g.KV8(k.data_ptr(), v.data_ptr(), sc.data_ptr(), pages, 64, 8, 128)
    s.append()
    s.same()
    s.attend(8)
    assert s.status.item() == 0


@pytest.mark.parametrize("heads,d,page,new", [(1, 128, 16, 4096), (4, 64, 16, 4096)])
def test_append_of_more_blocks_than_2_to_the_24(have_gpu, heads, d, page, new):
    """One long prompt among 65534 single tokens: so many groups of threads
    that a count of their threads passes 32 bits. Every sequence's token is
    appended once, the first ones' and the last ones' too. (The numbering
    itself is tested in test_kv8_host.py.)"""
    n = 65535
    rng = np.random.default_rng(heads)
    lens = np.full(n, 2, np.int32)
    lens[n // 2] = new
    row0 = np.concatenate([[0], np.cumsum(np.where(lens == new, new, 1))]).astype(np.int32)
    rows, width = int(row0[-1]), new // page
    table = torch.full((n, width), -1, dtype=torch.int32)
    table[:, 0] = torch.arange(n, dtype=torch.int32)
    table[n // 2] = torch.arange(n, n + width, dtype=torch.int32)
    table[n - 1, 0] = n // 2  # the page that the long one does not use
    t, ln, r0 = table.to(DEV), up(lens), up(row0)
    pools = [torch.randint(-127, 128, (n + width, heads, page, d), dtype=torch.int8, device=DEV) for _ in range(2)]
    scale = torch.full((n + width, heads, 2), 1 / 254, device=DEV)
    held = [p[:, :, 0].clone() for p in pools]
    kv = torch.from_numpy(rng.normal(0, 1, (rows, 2, heads, d)).astype(np.float32)).to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    c = g.KV8(pools[0].data_ptr(), pools[1].data_ptr(), scale.data_ptr(), n + width, page, heads, d)
    seqs = g.KV8Seqs(n, t.data_ptr(), width, ln.data_ptr(), new, d_row0=r0.data_ptr(), rows=rows, max_new=new,
                     d_status=status.data_ptr())
    hd = heads * d
    c.append(seqs, kv.data_ptr(), kv.data_ptr() + 4 * hd, k_strides=(2 * hd, d), v_strides=(2 * hd, d), stream=stream())
    assert status.item() == 0
    # the single tokens: slot 1 of their pages, whose slot 0 is rounded to the new scale once
    at = torch.cat([torch.arange(n // 2), torch.arange(n // 2 + 1, n - 1), torch.tensor([n // 2])]).to(DEV)
    x = torch.cat([kv[:n // 2], kv[n // 2 + new:]])
    for j in range(2):
        amax = x[:, j].abs().amax(-1).double() / 127
        want = torch.maximum(amax.float(), torch.tensor(1 / 254, device=DEV))
        assert torch.equal(scale[at, :, j], want)
        q = (x[:, j].double() / want.double()[..., None]).round().clamp(-127, 127).to(torch.int8)
        assert torch.equal(pools[j][at, :, 1], q)
        old = (held[j][at].double() * float(np.float32(1 / 254)) / want.double()[..., None]).round().to(torch.int8)
        assert torch.equal(pools[j][at, :, 0], old)
    # the long prompt
    y = kv[n // 2:n // 2 + new].view(width, page, 2, heads, d)
    for j in range(2):
        want = (y[:, :, j].abs().amax((1, -1)).double() / 127).float()
        assert torch.equal(scale[n:, :, j], want)
        q = (y[:, :, j].double() / want.double()[:, None, :, None]).round().clamp(-127, 127).to(torch.int8)
        assert torch.equal(pools[j][n:].transpose(1, 2), q)


@pytest.mark.parametrize("heads", [1, 2, 3, 5])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("mode", ["none", "pairs", "halves"])
def test_append_units_of_one_warp_that_differ(have_gpu, heads, d, mode):
    """Single tokens, several units (a head's keys or values) to a warp: keys
    that are rotated beside values that are not, and ordinary numbers beside
    tiny, huge and non-finite ones in every order of sequences and heads."""
    n = 24
    s = Side(list(range(1, n + 1)), [1] * n, heads=heads, d=d, mode=mode, seed=heads)
    kv = s.rng.normal(0, 1, (n, 2, heads, d)).astype(np.float32)
    by = np.array([1, 1e-36, 1, 1e37, 1, 1e-42, 0, 1], np.float32)
    kv *= by[s.rng.integers(0, 8, (n, 2, heads))][..., None]
    kv[5, 0, 0, 3], kv[11, 1, heads - 1, d - 1] = np.inf, np.nan
    s.append(kv, d_row0=None)
    s.same()
    assert np.isnan(s.ref.scale).sum() == 2 and s.status.item() == 0


def test_read_with_the_largest_bounds(have_gpu):
    """rows and max_new are bounds: with the largest numbers there the same
    tokens are read."""
    s = Side([5, 50, 33], [5, 17, 20], heads=2, d=64, seed=2)
    got = [torch.zeros(s.rows, 2, 64, device=DEV) for _ in range(4)]
    s.kv.read(s.seqs(), got[0].data_ptr(), got[1].data_ptr(), stream=stream())
    s.kv.read(s.seqs(rows=2**31 - 1, max_new=2**31 - 1), got[2].data_ptr(), got[3].data_ptr(), stream=stream())
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3]) and got[0].abs().sum() > 0
    assert s.status.item() == 0


@pytest.mark.parametrize("heads,new", [(1, 1), (4, 1), (4, 3), (1, 50)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bad", [(np.nan, 1.0), (1.0, np.nan), (1.0, np.inf), (1.0, -0.5), (-np.inf, 1.0)])
def test_attend_unsound_scales_reach_output_and_lse(have_gpu, heads, new, dtype, bad):
    """A page whose keys' or values' scale is not finite, or whose values' is
    below 0: output and log-sum-exp of who sees it are NaN, in each kernel,
    and those of who does not are not."""
    s = Side([90, 90], [new, new], heads=1, d=64, page=16, seed=6)
    s.ref.scale[s.table[1][2], 0] = bad  # positions 32 .. 47 of the second sequence
    s.upload()
    q = s.rng.normal(0, 1, (s.rows, heads, 64)).astype(np.float32)
    dt = getattr(torch, TORCH[dtype])
    dq, out, lse = up(q).to(dt), torch.zeros(s.rows, heads, 64, dtype=dt, device=DEV), torch.zeros(s.rows, heads, device=DEV)
    for window, sees in ((0, lambda p: p >= 32), (10, lambda p: 32 <= p < 57)):
        s.kv.attend(s.seqs(), heads, dq.data_ptr(), out.data_ptr(), dtype=dtype, window=window, d_lse=lse.data_ptr(),
                    stream=stream())
        want = np.array([False] * new + [sees(90 - new + r) for r in range(new)])
        assert np.array_equal(torch.isnan(out).all(-1).all(-1).cpu().numpy(), want)
        assert np.array_equal(torch.isnan(out).any(-1).any(-1).cpu().numpy(), want)
        assert np.array_equal(torch.isnan(lse).all(-1).cpu().numpy(), want)
        assert np.array_equal(torch.isnan(lse).any(-1).cpu().numpy(), want)
