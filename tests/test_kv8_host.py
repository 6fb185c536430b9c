"""The host's side of the 8-bit paged cache's calls, without a GPU: the index
arithmetic that kernels and host share, compiled here; and calls on a CUDA
runtime that writes launches down instead of running them (fake_cuda.c)."""

import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def compiled(tmp_path, body):
    """Runs `body` as a C++ main over the kernels' shared header."""
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text('#include "kv8.h"\n#include <cstdio>\n#include <initializer_list>\nusing namespace grx;\n'
                   "int main() {\n" + body + "\nreturn 0;\n}\n")
    cuda = Path(os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")).parents[1] / "include"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", str(ROOT / "gorelaxor_b200/csrc"), "-I", str(cuda), str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()


def test_append_groups_past_2_to_the_24_blocks(tmp_path):
    """A launch's groups of threads are numbered from 0 up without a gap or a
    repeat, however many blocks there are: the first and the last groups of a
    block, and of the largest launch that the entry point takes."""
    out = compiled(tmp_path, """
  for (int threads : {8, 16, 32, 256}) {
    const uint32_t per = 256 / threads;
    for (int64_t groups : {int64_t(1), int64_t(per) + 1, int64_t(16842495), int64_t(268697600), int64_t(2147483647)}) {
      const uint32_t grid = kv8_append_grid(groups, threads);
      if (int64_t(grid) * per < groups || int64_t(grid - 1) * per >= groups || grid > 2147483647u) std::puts("grid");
      for (uint32_t block : {0u, 1u, (1u << 24) - 1, 1u << 24, (1u << 24) + 1, 1u << 27, grid - 1}) {
        if (block >= grid) continue;
        for (uint32_t thread : {0u, 255u})
          if (kv8_append_group(block, thread, threads) != int64_t(block) * per + thread / threads)
            std::printf("group:%d:%u\\n", threads, block);
      }
    }
  }
  // pages that a sequence's new tokens can touch
  for (int page : {16, 32, 64})
    for (int64_t t : {int64_t(1), int64_t(2), int64_t(page), int64_t(page) + 1, int64_t(4096), int64_t(2147483647)})
      if (kv8_append_pages(int(t), page) != (page - 1 + t - 1) / page + 1) std::puts("pages");""")
    assert out == []


HEAD = """
import ctypes as C
import dataclasses, sys
import numpy as np
import gorelaxor_b200 as g
from gorelaxor_b200 import synth
from tests.helpers import SMALL, voice_kv
fake = C.CDLL(None)
fake.fake_first_unordered.restype = C.c_char_p

def launched():
    name, grid, out = C.create_string_buffer(400), (C.c_uint * 3)(), []
    for i in range(fake.fake_launches()):
        fake.fake_launch(i, name, 400, grid)
        out.append((name.value.decode(), tuple(grid)))
    return out

def flow(n=3, positions=lambda i: 5 + 11 * i):
    cfg = synth.FlowLMConfig(**SMALL)
    gm = g.FlowLM(synth.flowlm_gguf(cfg, synth.flowlm_tensors(cfg, 0)))
    return cfg, gm, [gm.voice(voice_kv(cfg, positions(i), 1 + i)) for i in range(n)]
"""


@pytest.fixture(scope="session")
def fake(tmp_path_factory):
    so = tmp_path_factory.mktemp("fake") / "libfakecuda.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-O1", "-Wall", "-o", str(so), str(ROOT / "tests/fake_cuda.c")], check=True)

    def run(body):
        env = {**os.environ, "LD_PRELOAD": str(so), "PYTHONPATH": str(ROOT)}
        r = subprocess.run([sys.executable, "-c", HEAD + body], capture_output=True, text=True, cwd=ROOT, env=env,
                           timeout=120)
        assert r.returncode == 0, r.stdout + r.stderr
        return r.stdout.split("\n")

    return run


SETS = {
    "flow lm, 8 bits": """
cfg, gm, vs = flow()
for page in (16, 64):
    st = g.Streams(gm, vs + vs[:1], 20, kv8_page=page)
    st.text([[1, 2, 3], [], [4], [5] * 9])
    st.step(np.zeros((4, cfg.ldim), np.float32))
    st.kv(2)
    st.reset()
""",
    "flow lm": """
cfg, gm, vs = flow()
for n in (1, 3):
    st = g.Streams(gm, vs[:n], 20)
    st.text([[1, 2, 3]] * n)
    st.step(np.zeros((n, cfg.ldim), np.float32))
    st.kv(n - 1)
    st.reset()
st = g.Streams(gm, (vs * 50)[:130], 20)
st.step(np.zeros((130, cfg.ldim), np.float32))
""",
    "whisper": """
cfg = synth.WhisperConfig(n_state=128, n_head=2, n_text_layer=2, n_text_ctx=64)
gm = g.Whisper(synth.whisper_ggml(cfg, synth.whisper_tensors(cfg, 0), synth.whisper_words(cfg)))
for n in (1, 3):
    b = g.WhisperBatch(gm, n)
    b.set_audio(np.stack([synth.whisper_encoder_out(1 + i, cfg) for i in range(n)]))
    b.prompt([gm.prev, 100, 200, gm.sot], 3)
    b.run(2)
    b.score([1] * n, 3)
    b.run(7)
""",
    "mimi": """
mc = synth.MimiConfig()
gm = g.Mimi(synth.flowlm_gguf(synth.FlowLMConfig(ldim=32), synth.mimi_tensors(mc, 32, 0), mimi=mc))
s = g.MimiStreams(gm, 2, max_frames=4)
s.decode(np.zeros((2, 32), np.float32))
""",
    "tdt": """
cfg = synth.TDTConfig(H=128, V=65, J=96, D=128)
gm = g.TDT(synth.tdt_gguf(cfg, synth.tdt_tensors(cfg, 0)))
b = g.TDTBatch(gm, 2, 8, 256)
b.decode(np.zeros((2, 8, 128), np.float32), [8, 8])
""",
}


@pytest.mark.parametrize("what", list(SETS))
def test_set_up_copies_are_waited_for(fake, what):
    """Copies that the legacy stream orders alone (from pageable memory, on
    the device) are waited for before a set's own streams use what they
    brought."""
    n, first = fake(SETS[what] + "print(fake.fake_unordered()); print(fake.fake_first_unordered().decode())")[:2]
    assert (int(n), first) == (0, "")


@pytest.mark.parametrize("page", [None, 16])
@pytest.mark.parametrize("kernel,nth", [("k_ln", 0), ("k_q8", 1), ("k_kv8_append", 0), ("k_kv8_append", 9),
                                        ("k_kv8_attend", 1), ("k_flin", 3)])
def test_a_refused_launch_fails_the_set(fake, page, kernel, nth):
    """A launch that the runtime refuses while a frame is captured leaves no
    node in its graph: the set is not made. (Appends before the capture, of
    the voice's two layers, are refused at once.)"""
    if page is None and "kv8" in kernel:
        pytest.skip("float32 caches have no such kernel")
    out = fake(f"""
cfg, gm, vs = flow(2)
fake.fake_fail(b"{kernel}", {nth})
try:
    g.Streams(gm, vs, 20, kv8_page={page})
    print("made")
except g.GrxError as e:
    print(e.code, e)
fake.fake_fail(b"", -1)
st = g.Streams(gm, vs, 20, kv8_page={page})  # nothing is left of the refusal
st.step(np.zeros((2, cfg.ldim), np.float32))
""")
    assert out[0].startswith("-4 ") and "invalid configuration" in out[0], out


def test_a_refused_launch_fails_a_text(fake):
    out = fake("""
cfg, gm, vs = flow(2)
st = g.Streams(gm, vs, 20, kv8_page=16)
for kernel, nth in (("k_q8", 0), ("k_kv8_append", 1), ("k_kv8_attend", 0)):
    fake.fake_fail(kernel.encode(), nth)
    try:
        st.text([[1, 2], [3]])
        print("ok")
    except g.GrxError as e:
        print(e.code)
    st.text([[1, 2], [3]])  # reported once
""")
    assert out[:3] == ["-4"] * 3


@pytest.mark.parametrize("width,max_new", [(2, 2**31 - 1), (2**25 - 1, 2**31 - 1), (2**25 - 1, 100), (2, 1)])
def test_reads_of_any_max_new(fake, width, max_new):
    """max_new may be any bound, the largest number too: the blocks go no
    further than the table's tokens, so the last block's token numbers have 32
    bits."""
    out = fake(f"""
c = g.KV8(4096, 4096, 4096, 8, 64, 2, 64)
s = g.KV8Seqs(2, 4096, {width}, 4096, 32, d_row0=4096, rows=2**31 - 1, max_new={max_new})
c.read(s, 4096, 4096)
print(launched()[0][1][0])
""")
    per, most = 16, min(max_new, 64 * width)  # tokens a block: 64 threads to a token of two heads' float32
    assert int(out[0]) == -(-most // per)
    assert int(out[0]) * per < 2**31


def test_a_refused_launch_is_reported_once(fake):
    """An attention or a scoring that the runtime refuses says so; the append
    and the read behind it are queued and say nothing."""
    out = fake("""
c = g.KV8(4096, 4096, 4096, 8, 16, 2, 64)
s = g.KV8Seqs(2, 4096, 2, 4096, 32)
many = g.KV8Seqs(2, 4096, 9, 4096, 99, d_row0=4096, rows=99, max_new=90)
calls = [("k_kv8_attend", lambda: c.attend(s, 2, 4096, 4096)), ("k_kv8_attend", lambda: c.attend(s, 8, 4096, 4096)),
         ("k_kv8_prompt", lambda: c.attend(many, 2, 4096, 4096)), ("k_kv8_append", lambda: c.append(s, 4096, 4096)),
         ("k_kv8_read", lambda: c.read(s, 4096, 4096)), ("k_logp", lambda: g.logprobs(4096, 3, 100, d_entropy=4096)),
         ("k_logp", lambda: g.logprobs(4096, 3, 99999, d_entropy=4096))]
for name, call in calls:
    fake.fake_fail(name.encode(), 0)
    try:
        call()
        print("queued")
    except g.GrxError as e:
        print(e.code)
    c.append(s, 4096, 4096)
    c.read(s, 4096, 4096)
    call()
print(fake.cudaPeekAtLastError())
""")
    assert out[:8] == ["-4"] * 7 + ["0"]
