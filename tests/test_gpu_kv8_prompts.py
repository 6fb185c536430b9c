"""Attention of prompts over the 8-bit paged cache (grx_kv8_attend with many
queries to a key head) against its definition in 64 bits: sizes around a
block's 128 query rows and a tile's 64 keys, windows, left padding, missing
pages, scales that grow, strides, replay from a graph."""

import numpy as np
import pytest
import torch

from tests.kv8_ref import TORCH, attend
from tests.test_gpu_kv8 import DEV, ERANGE, Side, stream, up

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,page,heads,kv_heads,mode", [(64, 16, 1, 1, "pairs"), (64, 64, 6, 2, "none"),
                                                        (128, 32, 5, 1, "halves"), (128, 64, 2, 2, "pairs")])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("new", [17, 42, 64, 65, 129])
def test_rows_and_tiles(have_gpu, d, page, heads, kv_heads, mode, dtype, new):
    """`new` tokens alone and behind others, so that a block's last row lies
    before, on and behind 128 and the keys fill one to six tiles; sequences
    with fewer new tokens, and with none, among them."""
    s = Side([new, new + 1, 64, 192, 191, 390, 30], [new, new, min(new, 64), 1, new, new, 0], heads=kv_heads, d=d,
             page=page, mode=mode, seed=new)
    s.attend(heads, dtype)
    assert s.status.item() == 0


@pytest.mark.parametrize("heads,kv_heads,d", [(20, 1, 64), (68, 2, 128), (130, 1, 64), (17, 1, 128)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_many_query_heads_to_a_key_head(have_gpu, heads, kv_heads, d, dtype):
    """Single tokens whose key heads serve more than 16 query heads, slots
    without tokens among them."""
    lens = [1, 0, 64, 65, 300, 0, 17]
    s = Side(lens, [1] * len(lens), heads=kv_heads, d=d, page=16, mode="pairs", seed=heads)
    q = s.rng.normal(0, 1.5, (len(lens), heads, d)).astype(np.float32)
    dt = getattr(torch, TORCH[dtype])
    dq, out = up(q).to(dt), torch.full((len(lens), heads, d), 7.0, dtype=dt, device=DEV)
    lse = torch.full((len(lens), heads), 7.0, device=DEV)
    s.kv.attend(s.seqs(d_row0=None), heads, dq.data_ptr(), out.data_ptr(), dtype=dtype, d_lse=lse.data_ptr(),
                stream=stream())
    got, gl, qs = out.float().cpu().numpy(), lse.cpu().numpy(), dq.float().cpu().numpy()
    for i, m in enumerate(lens):
        if m == 0:
            assert (got[i] == 0).all() and np.isneginf(gl[i]).all()
            continue
        want, wl, tol = attend(s.ref, s.table[i], m, qs[i:i + 1], s.rope, "pairs", half=dtype != "f32")
        tol = tol[..., None] + 2.0**-11 * np.abs(want) * (dtype == "f16") + 2.0**-24 * (dtype == "f16")
        assert (np.abs(got[i:i + 1] - want) <= tol).all(), i
        assert (np.abs(gl[i] - wl[0]) <= 2.0**-19 * (np.abs(wl[0]) + 8)).all()
    assert s.status.item() == 0


@pytest.mark.parametrize("d,heads,kv_heads", [(64, 2, 2), (128, 8, 2)])
def test_long_sequences_of_many_blocks(have_gpu, d, heads, kv_heads):
    s = Side([1500, 1101] + [20] * 20, [18, 3] + [18] * 20, heads=kv_heads, d=d, page=64, mode="halves", seed=d)
    s.attend(heads, "bf16")
    s.attend(heads, "f32")


@pytest.mark.parametrize("window", [1, 63, 64, 65, 100])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_windows_and_first_keys(have_gpu, window, dtype):
    """The first tile that a block reads is odd or even, and some rows see
    nothing of it; with left padding some see nothing at all."""
    s = Side([300, 200, 90, 64], [150, 33, 90, 20], heads=2, d=64, page=16, mode="pairs", seed=window)
    s.attend(2, dtype, window=window)
    got, lse = s.attend(2, dtype, window=window, first=[140, 400, 89, -3])
    assert (got[150:183] == 0).all() and np.isneginf(lse[150:183]).all()
    assert (got[183:272] == 0).all() and np.isneginf(lse[183:272]).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_scores_and_scales_that_grow(have_gpu, dtype):
    """Scores of hundreds, of zero, and growing from page to page; value
    scales that grow (what was summed is scaled) and fall."""
    for sharp in (60.0, 0.0):
        s = Side([400, 130], [70, 130], heads=2, d=64, seed=3)
        s.attend(2, "f32", sharp=sharp)
    for order in (1, -1):
        s = Side([700], [40], heads=1, d=128, page=16, seed=9)
        n = len(s.table[0])
        s.ref.k[:] = np.sign(s.ref.k) + (s.ref.k == 0)
        for b, p in enumerate(s.table[0][::order]):
            s.ref.scale[p] = 0.004 * (b + 1), 0.5 + b / n
        s.upload()
        s.attend(2, dtype)


def test_scales_of_zero_and_none(have_gpu):
    """Scales of zero count their keys with scores (or values) of zero; a
    scale that is no number matters to the rows that see its page alone."""
    s = Side([200], [200], heads=1, d=64, page=64, seed=5)
    s.ref.scale[s.table[0][0], 0] = 0, 0
    s.ref.scale[s.table[0][1], 0, 1] = 0
    s.ref.scale[s.table[0][2], 0, 0] = 0
    s.upload()
    s.attend(1)
    for j in (0, 1):
        s = Side([200], [200], heads=2, d=128, page=32, seed=6)
        s.ref.scale[s.table[0][3], 1, j] = np.nan  # positions 96 .. 127 of head 1
        s.upload()
        q = s.rng.normal(0, 1, (200, 2, 128)).astype(np.float32)
        q[5, 0, 3], q[150, 0, 100] = np.inf, np.nan
        dq, out = up(q), torch.zeros(200, 2, 128, device=DEV)
        for window, want in ((0, list(range(96, 200))), (10, list(range(96, 137)))):
            s.kv.attend(s.seqs(), 2, dq.data_ptr(), out.data_ptr(), window=window, stream=stream())
            nan = torch.isnan(out)
            assert torch.equal(nan.any(-1), nan.all(-1))
            assert np.flatnonzero(nan[:, 0, 0].cpu().numpy()).tolist() == [5, 150]
            assert np.flatnonzero(nan[:, 1, 0].cpu().numpy()).tolist() == want


def test_pages_that_are_not_there(have_gpu):
    """Tokens of a missing page are masked, a whole tile's and a whole
    sequence's too; a sequence that does not fit keeps its outputs."""
    s = Side([200, 100, 60, 60], [40, 40, 40, 40], heads=1, d=64, page=16, seed=7)
    q = s.rng.normal(0, 1, (160, 1, 64)).astype(np.float32)
    _, _, tol = attend(s.ref, s.table[0], 200, q[:40])
    k, v = s.ref.values(s.table[0], 200, 0)[0], s.ref.values(s.table[0], 200, 1)[0]
    s.t[0, 2] = -1
    s.t[0, 4:8] = s.pages
    s.t[1, :] = -9
    s.n[2] = 39
    s.r[4] = 161
    dq, out = up(q), torch.full((160, 1, 64), 5.0, device=DEV)
    s.kv.attend(s.seqs(), 1, dq.data_ptr(), out.data_ptr(), stream=stream())
    got = out.cpu().numpy()
    for r in range(40):
        see = [j for j in range(161 + r) if not (32 <= j < 48 or 64 <= j < 128)]
        w = np.exp(k[see] @ q[r, 0].astype(np.float64) / 8)
        assert (np.abs(got[r, 0] - w @ v[see] / w.sum()) <= 2 * tol.max()).all()
    assert (got[40:80] == 0).all()
    assert (got[80:] == 5).all()
    assert s.status.item() == ERANGE


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_strides_and_offsets(have_gpu, dtype):
    s = Side([150, 90], [90, 33], heads=2, d=64, mode="halves", seed=13)
    s.attend(4, dtype, offset=1)
    dt, n = getattr(torch, TORCH[dtype]), 123
    wide = torch.randn(n, 3, 4, 64, device=DEV).to(dt)
    packed = wide[:, 1].contiguous()
    a, b = torch.zeros(n, 4, 64, dtype=dt, device=DEV), torch.zeros(4, n, 65, dtype=dt, device=DEV)
    s.kv.attend(s.seqs(), 4, packed.data_ptr(), a.data_ptr(), dtype=dtype, stream=stream())
    s.kv.attend(s.seqs(), 4, wide[:, 1].data_ptr(), b.data_ptr(), dtype=dtype, q_strides=(12 * 64, 64),
                out_strides=(65, n * 65), stream=stream())
    assert torch.equal(a, b[..., :64].permute(1, 0, 2))
    assert (b[..., 64] == 0).all()


def test_graph_replays_and_two_calls_at_once(have_gpu):
    """A captured call reads lengths when it runs; calls on two streams that
    read one cache give the bits of one call."""
    s = Side([300, 250], [60, 60], heads=2, d=128, page=64, mode="pairs", seed=41)
    q = s.rng.normal(0, 1.5, (120, 4, 128)).astype(np.float32)
    dq, out = up(q), torch.zeros(120, 4, 128, device=DEV)
    sq = s.seqs()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.kv.attend(sq, 4, dq.data_ptr(), out.data_ptr(), stream=stream())
    for lens in ([300, 250], [60, 129], [64, 61]):
        s.n.copy_(torch.tensor(lens))
        graph.replay()
        got = out.cpu().numpy()
        for i in range(2):
            want, _, tol = attend(s.ref, s.table[i], lens[i], q[60 * i:60 * i + 60], s.rope, "pairs")
            assert (np.abs(got[60 * i:60 * i + 60] - want) <= tol[..., None]).all()
    s.n.copy_(torch.tensor([300, 250]))
    graph.replay()
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in range(2)]
    both = [torch.zeros_like(out) for _ in side]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, o in zip(side, both):
            s.kv.attend(sq, 4, dq.data_ptr(), o.data_ptr(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(both[0], out) and torch.equal(both[1], out)
