"""The 8-bit paged cache and the token log probabilities without a GPU: the
host's check of a call's pages, lengths and rows (the arithmetic that the
kernels bound every access with), and what the entry points refuse."""

import numpy as np
import pytest

import gorelaxor_b200 as g
from tests.kv8_ref import Cache, rope_table

EINVAL, ERANGE = -1, -5


def cache(**kw):
    a = dict(d_k=4096, d_v=4096, d_scale=4096, pages=8, page_tokens=16, kv_heads=2, head_dim=64)
    return g.KV8(**{**a, **kw})


def refused(fn, code, word=""):
    with pytest.raises(g.GrxError) as e:
        fn()
    assert e.value.code == code, e.value
    assert word in str(e.value), e.value


@pytest.mark.parametrize("table,lens,kw", [
    ([[0, 1], [2, 3]], [17, 32], {}),
    ([[0, 1], [2, 3]], [0, 1], {}),                                         # a slot without tokens
    ([[0, 99], [2, -1]], [16, 5], {}),                                      # entries behind the tokens are not looked at
    ([[0, 1], [0, 3]], [17, 18], dict(writes=True)),                        # a shared first page, appended to by neither
    ([[0, 1], [2, 3]], [20, 30], dict(row0=[0, 20, 25], rows=25, max_new=20)),
    ([[0, 1], [2, 3]], [20, 30], dict(row0=[0, 0, 0], rows=0, max_new=5)),  # no new tokens
    ([[0, 1], [2, 3]], [20, 30], dict(rope_positions=30)),
])
def test_check_takes(table, lens, kw):
    cache().check(np.array(table), lens, **kw)


@pytest.mark.parametrize("table,lens,kw,word", [
    ([[0, 1], [2, 8]], [17, 32], {}, "page 1 is 8"),
    ([[0, 1], [-1, 3]], [17, 32], {}, "page 0 is -1"),
    ([[0, 1], [2, 3]], [17, 33], {}, "33 tokens"),
    ([[0, 1], [2, 3]], [17, -1], {}, "-1 tokens"),
    ([[0, 1], [2, 3]], [20, 30], dict(row0=[0, 20, 26], rows=25, max_new=20), "rows 20 to 26"),
    ([[0, 1], [2, 3]], [20, 30], dict(row0=[0, 20, 19], rows=25, max_new=20), "rows 20 to 19"),
    ([[0, 1], [2, 3]], [20, 30], dict(row0=[-1, 2, 3], rows=25, max_new=20), "rows -1 to 2"),
    ([[0, 1], [2, 3]], [20, 30], dict(row0=[0, 20, 25], rows=25, max_new=19), "rows 0 to 20"),
    ([[0, 1], [2, 3]], [2, 30], dict(row0=[0, 3, 25], rows=25, max_new=25), "2 tokens"),
    ([[0, 1], [2, 3]], [20, 31], dict(rope_positions=30), "31 tokens"),
    ([[0, 1], [2, 1]], [17, 20], dict(writes=True), "appends to page 1"),
    ([[0, 1], [1, 2]], [17, 20], dict(writes=True), "holds page 1"),
    ([[0, 0], [2, 3]], [17, 20], dict(writes=True), "holds page 0"),
    ([[0, 0], [2, 3]], [17, 20], dict(row0=[0, 17, 18], rows=18, max_new=17, writes=True), "appends to page 0"),
])
def test_check_refuses(table, lens, kw, word):
    refused(lambda: cache().check(np.array(table), lens, **kw), ERANGE, word)


def test_check_of_a_vast_cache():
    """The check's memory goes by the table, not by what pages could be."""
    kv = cache(pages=2**31 - 1)
    kv.check(np.array([[5, 2**31 - 2], [7, 8]]), [20, 20], writes=True)
    refused(lambda: kv.check(np.array([[5, 2**31 - 2], [7, 2**31 - 2]]), [20, 20], writes=True), ERANGE, "appends")


def seqs(**kw):
    a = dict(n=2, d_table=4096, table_width=2, d_len=4096, max_len=32)
    return g.KV8Seqs(**{**a, **kw})


@pytest.mark.parametrize("kw,word", [
    (dict(page_tokens=8), "pages of 8"), (dict(page_tokens=48), "pages of 48"), (dict(head_dim=96), "heads of 96"),
    (dict(kv_heads=0), "0 heads"), (dict(pages=0), "0 pages"), (dict(d_k=None), "null cache"),
    (dict(d_v=4104), "16-byte"), (dict(d_scale=4100), "of 8"),
])
def test_caches_refused(kw, word):
    c = cache(**kw)
    refused(lambda: c.append(seqs(), 4096, 4096), EINVAL, word)
    refused(lambda: c.read(seqs(), 4096, 4096), EINVAL, word)
    refused(lambda: c.attend(seqs(), 2, 4096, 4096), EINVAL, word)


@pytest.mark.parametrize("kw,word", [
    (dict(n=-1), "-1 sequences"), (dict(n=65536), "65536"), (dict(d_table=None), "null table"),
    (dict(d_len=None), "null table"), (dict(table_width=0), "0 pages wide"), (dict(table_width=1 << 26), "wide"),
    (dict(rows=1), "1 rows for 2"), (dict(rows=-1, d_row0=4096), "-1 rows"), (dict(max_new=2), "max_new is 1"),
    (dict(rope="pairs"), "no positions"), (dict(rope="halves", rope_positions=9, d_rope=4104), "16-byte"),
    (dict(rope="halves", rope_positions=9), "16-byte"),
])
def test_sequences_refused(kw, word):
    refused(lambda: cache().append(seqs(**kw), 4096, 4096), EINVAL, word)
    refused(lambda: cache().attend(seqs(**kw), 2, 4096, 4096), EINVAL, word)


def test_rows_refused():
    c = cache()
    refused(lambda: c.append(seqs(), 4098, 4096), EINVAL, "keys")
    refused(lambda: c.append(seqs(), 4096, 4097, dtype="bf16"), EINVAL, "values")
    refused(lambda: c.append(seqs(), 4096, 4096, k_strides=(-64, 64)), EINVAL, "keys")
    refused(lambda: c.append(seqs(), None, 4096), EINVAL, "null keys")
    refused(lambda: c.attend(seqs(), 3, 4096, 4096), EINVAL, "3 query heads over 2")
    refused(lambda: c.attend(seqs(), 0, 4096, 4096), EINVAL, "query heads")
    refused(lambda: c.attend(seqs(), 2, 4096, 4096, window=-1), EINVAL, "window")
    refused(lambda: c.attend(seqs(), 2, 4096, 4096, scale=float("nan")), EINVAL, "scale")
    refused(lambda: c.attend(seqs(), 2, 4096, None), EINVAL, "null")
    refused(lambda: c.attend(seqs(), 2, 4096, 4096, d_lse=4098), EINVAL, "lse")
    big = dict(n=65535, rows=1 << 30, d_row0=4096, max_new=1 << 30)
    refused(lambda: c.append(seqs(**big), 4096, 4096), ERANGE, "fewer")
    refused(lambda: c.attend(seqs(**big), 2, 4096, 4096), ERANGE, "parts")
    with pytest.raises(KeyError):
        c.append(seqs(), 4096, 4096, dtype="f64")


def test_nothing_to_do_is_no_error():
    c = cache()
    c.append(seqs(n=0, d_table=None, d_len=None), None, None)
    c.attend(seqs(n=2, d_row0=4096, rows=0, max_new=0), 2, None, None)
    c.read(seqs(), None, None)
    g.logprobs(None, 0, 100)
    g.logprobs(4096, 5, 100)  # no output asked for


@pytest.mark.parametrize("kw,word", [
    (dict(rows=-1), "rows"), (dict(vocab=0), "rows of 0"), (dict(vocab=2**31 - 1), "rows of"),
    (dict(top=33, d_top_ids=4096), "33 alternatives"), (dict(top=-1, d_top_ids=4096), "-1 alternatives"),
    (dict(vocab=4, top=5, d_top_ids=4096), "5 alternatives"), (dict(d_logprob=4096), "without targets"),
    (dict(d_logits=4098, d_entropy=4096), "boundary"), (dict(d_logits=4097, dtype="f16", d_entropy=4096), "boundary"),
    (dict(d_entropy=4097), "boundary"), (dict(d_logits=None, d_entropy=4096), "null logits"),
    (dict(row_stride=-5, d_entropy=4096), "rows"),
])
def test_logprobs_refused(kw, word):
    a = dict(d_logits=4096, rows=3, vocab=100)
    refused(lambda: g.logprobs(**{**a, **kw}), EINVAL, word)


def test_without_a_device():
    if g.device_count() > 0:
        pytest.skip("a device is present")
    for fn in (lambda: cache().append(seqs(), 4096, 4096), lambda: cache().attend(seqs(), 2, 4096, 4096),
               lambda: cache().read(seqs(), 4096, 4096), lambda: g.logprobs(4096, 3, 100, d_entropy=4096)):
        refused(fn, -6)


def test_reference_cache_rounds_as_defined():
    """The tests' own model of the cache: half a step at most for a token
    whose page's scale does not grow afterwards, and for others half a step
    more for each time that it does."""
    rng = np.random.default_rng(1)
    c = Cache(3, 2, 16, 64)
    x = rng.normal(0, 1, (40, 2, 2, 64)).astype(np.float32)
    grown = np.zeros((40, 2))
    for t in range(40):
        before = c.scale.copy()
        c.append([2, 0, 1], t + 1, x[t:t + 1, 0], x[t:t + 1, 1])
        p = [2, 0, 1][t // 16]
        for h in range(2):
            if t % 16 and c.scale[p, h, 0] > before[p, h, 0]:
                grown[t // 16 * 16:t, h] += 1
    got = c.values([2, 0, 1], 40, 0).transpose(1, 0, 2)
    step = c.scale[[2, 0, 1]][np.arange(40) // 16, :, 0]
    assert (np.abs(got - x[:, 0]).max(-1) <= (0.5 + 0.5 * grown) * step * (1 + 1e-6)).all()
    assert rope_table(3, 64).shape == (3, 32, 2)


def test_bounds_of_ragged_calls():
    """A check of a ragged call takes the bounds that it is not given from the
    rows."""
    kv, t = cache(), np.array([[0, 1], [2, 3], [4, 5]])
    kv.check(t, [20, 30, 7], row0=[0, 20, 25, 25])
    kv.check(t, [20, 30, 7], row0=[0, 0, 0, 0], writes=True)
    kv.check(t, [1, 30, 7], writes=True)
    refused(lambda: kv.check(t, [20, 30, 7], row0=[0, 20, 25, 25], rows=24), ERANGE, "rows 20 to 25")
    refused(lambda: kv.check(t, [20, 30, 7], row0=[0, 20, 25, 25], max_new=19), ERANGE, "rows 0 to 20")
    refused(lambda: kv.check(t, [20, 4, 7], row0=[0, 20, 25, 25]), ERANGE, "rows 20 to 25")
    refused(lambda: kv.check(t, [20, 30, 7], row0=[0, 20, 15, 25]), ERANGE, "rows 20 to 15")
