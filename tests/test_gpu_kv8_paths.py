"""The paths that call the 8-bit cache and the token log probabilities: the
flow LM's streams on 8-bit caches, a Whisper batch's scores, and the
operators one after the other as a host with layers of its own calls them."""

import numpy as np
import pytest
import torch

import gorelaxor_b200 as g
from gorelaxor_b200 import synth
from tests.helpers import SMALL, bits_equal, voice_kv
from tests.kv8_ref import Cache, attend, rope_table

pytestmark = pytest.mark.gpu


def model(seed=0, **kw):
    cfg = synth.FlowLMConfig(**{**SMALL, **kw})
    return cfg, g.FlowLM(synth.flowlm_gguf(cfg, synth.flowlm_tensors(cfg, seed)))


def voices(cfg, gm, n, positions=lambda i: 6 + i % 5):
    return [gm.voice(voice_kv(cfg, positions(i), 1 + i)) for i in range(n)]


def noise(cfg, n, frames):
    return np.stack([synth.noise_frames(1 + i, frames, cfg.ldim, cfg.temperature) for i in range(n)], axis=1)


def stored(cfg, x, page):
    """A voice's caches [layers][2][positions][d] as an 8-bit cache holds them."""
    L, _, P, d = x.shape
    out = np.empty(x.shape, np.float64)
    for l in range(L):
        c = Cache(-(-P // page), d // 64, page, 64)
        c.append(list(range(c.k.shape[0])), P, x[l, 0].reshape(P, -1, 64), x[l, 1].reshape(P, -1, 64))
        for j in range(2):
            out[l, j] = c.values(range(c.k.shape[0]), P, j).transpose(1, 0, 2).reshape(P, d)
    return out


@pytest.mark.parametrize("page", [16, 32, 64])
def test_a_voice_in_8_bits(have_gpu, page):
    """A new set's caches are its voices', rounded as defined (bit for bit),
    also where streams share a voice and after frames and a reset."""
    cfg, gm = model()
    kvs = [voice_kv(cfg, p, 1 + p) for p in (5, 16, 40, 64)]
    vs = [gm.voice(k) for k in kvs]
    of = [2, 0, 2, 1, 3, 2]
    st = g.Streams(gm, [vs[i] for i in of], 20, kv8_page=page)
    want = [stored(cfg, k, page).astype(np.float32) for k in kvs]
    for again in range(2):
        for s, i in enumerate(of):
            assert bits_equal(st.kv(s), want[i]), (again, s)
        assert [st.pos(s) for s in range(6)] == [kvs[i].shape[2] for i in of]
        for f in range(18):
            st.step(noise(cfg, 6, 18)[f])
        st.reset()


def test_kv_of_float_streams(have_gpu):
    """grx_streams_kv of float32 caches: a voice comes back as it went in, and
    stays in front of the frames that follow it."""
    cfg, gm = model()
    kv = voice_kv(cfg, 9, 3)
    st = g.Streams(gm, [gm.voice(kv), gm.voice(voice_kv(cfg, 4, 1))], 12)
    assert bits_equal(st.kv(0), kv)
    z = noise(cfg, 2, 6)
    for f in range(3):
        st.step(z[f])
    assert st.kv(0).shape[2] == 12 and bits_equal(st.kv(0)[:, :, :9], kv)
    with pytest.raises(g.GrxError):
        st.kv(2)


@pytest.mark.parametrize("n,page", [(1, 16), (3, 32), (9, 64), (40, 16)])
def test_first_layer_keys_of_a_frame(have_gpu, n, page):
    """The first frame's keys and values of the first layer come from bos
    alone: the 8-bit set's are the float32 set's within half a step of their
    page's scale (one more half for each later token that raised it: none
    here), the voice's tokens within a step."""
    cfg, gm = model()
    vs = voices(cfg, gm, n)
    a, b = g.Streams(gm, vs, 8), g.Streams(gm, vs, 8, kv8_page=page)
    z = noise(cfg, n, 1)
    a.step(z[0])
    b.step(z[0])
    for i in range(n):
        x, y = a.kv(i)[0].astype(np.float64), b.kv(i)[0].astype(np.float64)
        assert x.shape == y.shape
        P = x.shape[1]
        for j in range(2):
            for h in range(cfg.heads):
                for lo in range(0, P, page):
                    u, v = (w[j, lo:lo + page, h * 64:(h + 1) * 64] for w in (x, y))
                    step = np.abs(u).max() / 127
                    tol = np.full(len(u), 1.0 if lo + page >= P else 0.5)
                    if lo + len(u) == P:
                        tol[-1] = 0.5
                    assert (np.abs(u - v).max(1) <= tol * step * (1 + 1e-5)).all(), (i, j, h, lo)


@pytest.mark.parametrize("n", [1, 5, 130])
def test_frames_near_the_float_set(have_gpu, n):
    """A frame's output on 8-bit caches against float32 ones: within the 2 %
    of its RMS that the int8 path is held to (a stored value is off by at
    most 1/254 of its page's largest, 0.8 % of the values' RMS as they are
    spread here, and attention averages that)."""
    cfg, gm = model(seed=2)
    vs = voices(cfg, gm, n, lambda i: 30 + i % 40)
    a, b = g.Streams(gm, vs, 4), g.Streams(gm, vs, 4, kv8_page=16)
    if n == 1:
        assert not b.persistent()
    z = noise(cfg, n, 1)
    la, _, _, oa = a.step(z[0], want_lm_out=True)
    lb, _, _, ob = b.step(z[0], want_lm_out=True)
    assert np.sqrt(np.mean((oa - ob) ** 2)) <= 0.02 * np.sqrt(np.mean(oa**2))
    assert np.isfinite(lb).all()


def test_steps_device_runs_and_texts_agree(have_gpu):
    """Frame by frame, as one device-resident run, in parts or not, and again
    after a reset: the same bits. Text before the frames too."""
    cfg, gm = model(seed=3)
    n, frames = 132, 11  # two parts; more than one replay of eight frames
    vs = voices(cfg, gm, n)
    ids = [[(7 * i + j) % cfg.text_vocab for j in range(i % 7)] for i in range(n)]
    z = noise(cfg, n, frames)
    st = g.Streams(gm, vs, frames + 8, kv8_page=16)
    assert st.parts() == 2
    t0 = st.text(ids)
    want = [st.step(z[f])[:2] for f in range(frames)]
    last = st.kv(131)
    st.reset()
    assert bits_equal(st.text(ids), t0)
    dn = torch.from_numpy(z).cuda()
    dl, de = torch.empty_like(dn), torch.empty((frames, n), device="cuda")
    st.run_device(frames, dn.data_ptr(), dl.data_ptr(), de.data_ptr())
    st.sync()
    for f in range(frames):
        assert bits_equal(dl[f].cpu().numpy(), want[f][0]) and bits_equal(de[f].cpu().numpy(), want[f][1]), f
    assert bits_equal(st.kv(131), last)


@pytest.mark.parametrize("page", [16, 64])
def test_long_texts_near_the_float_set(have_gpu, page):
    """Texts from none to hundreds of tokens in one call: the first layer's
    caches are the float32 set's within a step; and the last token's output
    is that of a float32 set whose voice is what the 8-bit caches hold of the
    tokens before it, within the 2 % that a frame's is (the two differ in the
    one token's own key and value)."""
    cfg, gm = model(seed=4)
    lens = [0, 1, 20, 70, 150, 17, 64, 201]
    n = len(lens)
    vs = voices(cfg, gm, n, lambda i: 10 + 9 * i)
    ids = [[(11 * i + 3 * j) % cfg.text_vocab for j in range(m)] for i, m in enumerate(lens)]
    a, b = g.Streams(gm, vs, 210), g.Streams(gm, vs, 210, kv8_page=page)
    a.text(ids)
    tb = b.text(ids)
    for i, m in enumerate(lens):
        assert b.pos(i) == a.pos(i) == 10 + 9 * i + m
        if m:
            c = g.Streams(gm, [gm.voice(np.ascontiguousarray(b.kv(i)[:, :, :-1]))], 4)
            tc = c.text([ids[i][-1:]])[0]
            assert np.sqrt(np.mean((tc - tb[i]) ** 2)) <= 0.02 * np.sqrt(np.mean(tc**2)), i
        x, y = a.kv(i)[0].astype(np.float64), b.kv(i)[0].astype(np.float64)
        for lo in range(0, x.shape[1], page):
            u, v = x[:, lo:lo + page], y[:, lo:lo + page]
            for j in range(2):
                for h in range(cfg.heads):
                    c = slice(h * 64, h * 64 + 64)
                    # a page that the voice began was rounded once before its scale rose
                    assert np.abs(u[j, :, c] - v[j, :, c]).max() <= np.abs(u[j, :, c]).max() / 127 * (1 + 1e-5)
    again = g.Streams(gm, vs, 210, kv8_page=page)
    assert bits_equal(again.text(ids), tb)


def test_what_streams_refuse(have_gpu):
    cfg, gm = model()
    v = voices(cfg, gm, 1)
    for page in (0, 8, 48, 128):
        with pytest.raises(g.GrxError) as e:
            g.Streams(gm, v, 4, kv8_page=page)
        assert e.value.code == -1
    st = g.Streams(gm, v, 2, kv8_page=16)
    z = noise(cfg, 1, 3)
    st.step(z[0])
    st.step(z[1])
    with pytest.raises(g.GrxError) as e:  # past the room it was made with
        st.step(z[2])
    assert e.value.code == -5
    d = torch.zeros(64, device="cuda")
    with pytest.raises(g.GrxError) as e:
        st.run_device_timed(0, d.data_ptr(), d.data_ptr(), None, d.data_ptr())
    assert e.value.code == -1


def test_whisper_scores(have_gpu):
    """grx_whisper_score is log softmax of grx_whisper_logits; the token that
    greedy decoding would take without rules leads the list."""
    cfg = synth.WhisperConfig(n_state=128, n_head=2, n_text_layer=2, n_text_ctx=64)
    gm = g.Whisper(synth.whisper_ggml(cfg, synth.whisper_tensors(cfg, 0), synth.whisper_words(cfg)))
    for n in (1, 3):
        b = g.WhisperBatch(gm, n)
        b.set_audio(np.stack([synth.whisper_encoder_out(1 + i, cfg) for i in range(n)]))
        with pytest.raises(g.GrxError):
            b.score([0] * n, 3)
        b.prompt([gm.prev, 100, 200, gm.sot], 3)
        for _ in range(2):
            x = b.logits().astype(np.float64)
            lp = x - x.max(1, keepdims=True)
            lp -= np.log(np.exp(lp).sum(1, keepdims=True))
            tok = [5 + i for i in range(n)]
            got, ent, ids, lps = b.score(tok, 4)
            want = lp[np.arange(n), tok]
            assert np.abs(got - want).max() <= 2.0**-20 * np.abs(want).max()
            we = -(np.exp(lp) * lp).sum(1)
            assert np.abs(ent - we).max() <= 2.0**-18 * np.abs(we).max()
            order = np.argsort(-x, 1, kind="stable")[:, :4]
            assert np.array_equal(ids, order)
            assert np.abs(lps - np.take_along_axis(lp, order, 1)).max() <= 2.0**-20 * np.abs(lp).max()
            none, e2, i2, _ = b.score()
            assert none is None and np.array_equal(e2, ent) and i2.shape == (n, 0)
            b.run(2)
        with pytest.raises(g.GrxError):
            b.score(tok, 33)


def test_a_decoder_step_of_the_operators(have_gpu):
    """Two layers' caches, a head and its scores, token by token, as a host
    with its own layers calls them: each stage is checked against the 64-bit
    model on what the stage before left on the device."""
    rng = np.random.default_rng(5)
    n, heads, hk, d, page, layers, vocab, steps = 3, 4, 2, 64, 16, 2, 1000, 20
    width = 3
    table = rng.permutation(n * width).reshape(n, width).astype(np.int32)
    lens = np.array([1, 14, 25], np.int32) - 1
    rope = rope_table(width * page, d)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    refs = [Cache(n * width, hk, page, d, rng) for _ in range(layers)]
    pools = [(dev(r.k), dev(r.v), dev(r.scale)) for r in refs]
    kvs = [g.KV8(k.data_ptr(), v.data_ptr(), s.data_ptr(), n * width, page, hk, d) for k, v, s in pools]
    dt, dl, dr, status = dev(table), dev(lens), dev(rope), torch.zeros(1, dtype=torch.int32, device="cuda")
    seqs = g.KV8Seqs(n, dt.data_ptr(), width, dl.data_ptr(), width * page, d_rope=dr.data_ptr(),
                     rope_positions=len(rope), rope="halves", d_status=status.data_ptr())
    qkv_w = [g.Weight.f32(rng.normal(0, 0.06, ((heads + 2 * hk) * d, heads * d)).astype(np.float32)) for _ in range(layers)]
    head_w = g.Weight.f32(rng.normal(0, 0.1, (vocab, heads * d)).astype(np.float32))
    x = rng.normal(0, 1, (n, heads * d)).astype(np.float32)
    st = torch.cuda.current_stream().cuda_stream
    for step in range(steps):
        lens += 1
        dl += 1
        kvs[0].check(table, lens, rope_positions=len(rope), writes=True)
        for l in range(layers):
            qkv = g.linear(qkv_w[l], x)
            q = dev(qkv)
            row = (heads + 2 * hk) * d
            at = q.data_ptr()
            kvs[l].append(seqs, at + heads * d * 4, at + (heads + hk) * d * 4, k_strides=(row, d), v_strides=(row, d),
                          stream=st)
            out = torch.empty(n, heads, d, device="cuda")
            kvs[l].attend(seqs, heads, at, out.data_ptr(), q_strides=(row, d), stream=st)
            x = out.cpu().numpy().reshape(n, -1)
            for i in range(n):
                r = qkv[i].reshape(-1, d)
                refs[l].append(table[i], lens[i], r[None, heads:heads + hk], r[None, heads + hk:], rope, "halves")
                want, _, tol = attend(refs[l], table[i], lens[i], r[None, :heads], rope, "halves")
                assert (np.abs(x[i].reshape(heads, d) - want[0]) <= tol[0][:, None]).all(), (step, l, i)
        logits = g.linear(head_w, x)
        dx, tgt = dev(logits), dev(np.arange(n, dtype=np.int32))
        lp, ids = torch.zeros(n, device="cuda"), torch.zeros(n, 1, dtype=torch.int32, device="cuda")
        g.logprobs(dx.data_ptr(), n, vocab, d_targets=tgt.data_ptr(), top=1, d_logprob=lp.data_ptr(),
                   d_top_ids=ids.data_ptr(), stream=st)
        y = logits.astype(np.float64)
        want = y[np.arange(n), np.arange(n)] - y.max(1) - np.log(np.exp(y - y.max(1, keepdims=True)).sum(1))
        assert np.abs(lp.cpu().numpy() - want).max() <= 2.0**-20 * np.abs(want).max()
        assert np.array_equal(ids[:, 0].cpu().numpy(), y.argmax(1))
        x = np.tanh(x * 4 + rng.normal(0, 1, x.shape).astype(np.float32)).astype(np.float32)
    for r, (k, v, s) in zip(refs, pools):
        assert np.array_equal(k.cpu().numpy(), r.k) and np.array_equal(v.cpu().numpy(), r.v)
        assert np.array_equal(s.cpu().numpy(), r.scale)
    assert status.item() == 0
