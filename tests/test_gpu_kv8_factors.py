"""grx_kv8_attend with factors of every sign: scale below, at and above 0, and
pages whose keys' scale is below 0, for single tokens, a few and many queries
to a key head, against the definition in 64 bits (tests/kv8_ref.py)."""

import numpy as np
import pytest
import torch

from tests.kv8_ref import EPS2, TORCH, attend
from tests.test_gpu_kv8 import DEV, Side, stream, up

pytestmark = pytest.mark.gpu


def check(s, heads, dtype, q, scale=None, window=0):
    """One call against the definition, within kv8_ref's bound and half a step
    of the output's type."""
    dt = getattr(torch, TORCH[dtype])
    dq, out = up(q).to(dt), torch.full((s.rows, heads, s.d), 7.0, dtype=dt, device=DEV)
    lse = torch.full((s.rows, heads), 7.0, device=DEV)
    s.kv.attend(s.seqs(), heads, dq.data_ptr(), out.data_ptr(), dtype=dtype, scale=scale, window=window,
                d_lse=lse.data_ptr(), stream=stream())
    got, gl, qs = out.double().cpu().numpy(), lse.double().cpu().numpy(), dq.float().cpu().numpy()
    for i, m in enumerate(s.lens):
        a, b = s.row0[i], s.row0[i + 1]
        if a == b:
            continue
        want, wl, tol = attend(s.ref, s.table[i], m, qs[a:b], s.rope, s.mode, scale=scale, window=window,
                               half=dtype != "f32")
        tol = tol[..., None] + EPS2[dtype] * np.abs(want) * (dtype != "f32") + 2.0**-24 * (dtype == "f16")
        err = np.abs(got[a:b] - want)
        assert (err <= tol).all(), (i, m, np.nanmax(err), tol.max(), np.isnan(err).sum())
        assert (np.abs(gl[a:b] - wl) <= 2.0**-19 * (np.abs(wl) + 8)).all()
    assert s.status.item() == 0


SHAPES = [  # heads, key heads, new tokens: each kernel's rows to a key head
    (2, 2, [1, 1, 1]), (8, 2, [1, 1, 1]), (4, 1, [3, 4, 2]), (4, 2, [30, 9, 1]), (1, 1, [70, 129, 200]),
    (4, 1, [40, 33, 64]),
]


@pytest.mark.parametrize("heads,kv_heads,new", SHAPES)
@pytest.mark.parametrize("d,page,dtype", [(64, 16, "f32"), (128, 64, "bf16"), (128, 32, "f16"), (64, 64, "f16")])
@pytest.mark.parametrize("scale", [-0.125, -1.0, 0.0, 0.5])
def test_scales_of_either_sign(have_gpu, heads, kv_heads, new, d, page, dtype, scale):
    """Scores of tens: the largest product has the smallest score where the
    scale is below 0."""
    s = Side([200, 330, 511], new, heads=kv_heads, d=d, page=page, mode="halves", seed=3)
    check(s, heads, dtype, s.rng.normal(0, 3, (s.rows, heads, d)).astype(np.float32), scale)


@pytest.mark.parametrize("heads,kv_heads,new", SHAPES)
@pytest.mark.parametrize("d,dtype", [(64, "f32"), (128, "bf16")])
@pytest.mark.parametrize("scale", [None, -0.25])
def test_key_scales_below_zero(have_gpu, heads, kv_heads, new, d, dtype, scale):
    """Pages whose keys count negatively stand between others: a byte q is
    q·scale, whatever the scale's sign."""
    s = Side([200, 330, 511], new, heads=kv_heads, d=d, page=16, mode="pairs", seed=4)
    s.ref.scale[::3, :, 0] *= -1
    s.ref.scale[::5, 0, 0] *= -2
    s.upload()
    check(s, heads, dtype, s.rng.normal(0, 3, (s.rows, heads, d)).astype(np.float32), scale, window=150)
