"""Workloads of the operators of a served language model's step: the 8-bit
paged key/value cache (appending to it, attending over it) and the log
probabilities of given tokens.

``listed()`` gives the cases, ``draw()`` more of the same ranges, ``run()`` one
pass: in elementary torch operations, or (``own``) through this package's
entry points. ``exact()`` states the same results in 64 bits from the
definitions.

The cache. Tokens live in pages of ``page`` tokens; a sequence's row of the
page table names its pages in order. For each page and key/value head there
are two scales, one for the page's keys and one for its values; a stored
byte q stands for q * scale. Appending tokens to a page raises its scale to
max(scale so far, largest new magnitude / 127), rounds what the page held to
the new scale and then the new values; a page's first token starts it afresh.
"""

import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------- the cases


def listed():
    return [
        # One speaking stream of the flow LM (16 heads of 64 values): one frame's
        # keys and values, the call whose latency counts.
        dict(name="append one stream", op="append", n=1, kv_heads=16, head_dim=64, page=16, type="f32",
             len_min=100, len_max=100, new_min=1, new_max=1, rope="pairs"),
        # 256 streams of it in one step, between their voice prompts and 512 frames.
        dict(name="append 256 streams", op="append", n=256, kv_heads=16, head_dim=64, page=16, type="f32",
             len_min=65, len_max=576, new_min=1, new_max=1, rope="pairs"),
        # Prompts of several requests entering the cache at once, ragged.
        dict(name="append prompts", op="append", n=24, kv_heads=8, head_dim=128, page=64, type="bf16",
             len_min=200, len_max=4000, new_min=1, new_max=1024, rope="halves"),
        # One stream's attention, 577 keys, single token.
        dict(name="attend one stream", op="attend", n=1, heads=16, kv_heads=16, head_dim=64, page=16, type="f32",
             len_min=577, len_max=577, new_min=1, new_max=1, rope="pairs", window=0, first=False),
        # A step of 256 streams: the serving case of the flow LM.
        dict(name="attend 256 streams", op="attend", n=256, heads=16, kv_heads=16, head_dim=64, page=16, type="f32",
             len_min=65, len_max=576, new_min=1, new_max=1, rope="pairs", window=0, first=False),
        # One long conversation, four query heads to a key head: work split over the long axis.
        dict(name="attend one long", op="attend", n=1, heads=32, kv_heads=8, head_dim=128, page=64, type="bf16",
             len_min=32768, len_max=32768, new_min=1, new_max=1, rope="halves", window=0, first=False),
        # A ragged batch, from empty to long, with left padding that leaves some rows nothing to see.
        dict(name="attend ragged", op="attend", n=48, heads=16, kv_heads=4, head_dim=128, page=32, type="f16",
             len_min=1, len_max=12001, new_min=1, new_max=1, rope="none", window=0, first=True),
        # Prompt chunks against what the cache already holds: several queries to a sequence.
        dict(name="attend prompts", op="attend", n=8, heads=16, kv_heads=4, head_dim=128, page=64, type="bf16",
             len_min=300, len_max=2500, new_min=1, new_max=512, rope="halves", window=0, first=False),
        # One decoded token of Whisper base.en's vocabulary: its probability and five alternatives.
        dict(name="logprobs one row", op="logprobs", rows=1, vocab=51864, type="f32", top=5),
        # 32 Whisper streams.
        dict(name="logprobs 32 streams", op="logprobs", rows=32, vocab=51864, type="f32", top=5),
        # Scoring given texts with a large odd vocabulary.
        dict(name="logprobs texts", op="logprobs", rows=2048, vocab=100003, type="bf16", top=20),
        # The joint network's outputs of 32 transducer streams of 750 frames: many short rows.
        dict(name="logprobs frames", op="logprobs", rows=24000, vocab=1030, type="f32", top=1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "logprobs":
        vocab = _log_int(rng, 33, 200001)
        rows = _log_int(rng, 1, min(20000, (2048 if kind != "f32" else 1024) * 100003 // vocab))
        return dict(op=op, rows=rows, vocab=vocab, type=kind, top=rng.randint(0, min(32, vocab)))
    head_dim = rng.choice([64, 128])
    kv_heads = _log_int(rng, 1, 16)
    page = rng.choice([16, 32, 64])
    n = _log_int(rng, 1, 256)
    rope = rng.choice(["none", "pairs", "halves"])
    if op == "append":
        new_max = _log_int(rng, 1, max(1, min(1024, (24 * 1024 * 1024) // (n * kv_heads * head_dim))))
        len_max = max(new_max, _log_int(rng, 1, 8000))
        return dict(op=op, n=n, kv_heads=kv_heads, head_dim=head_dim, page=page, type=kind,
                    len_min=rng.randint(new_max, len_max), len_max=len_max, new_min=rng.randint(1, new_max),
                    new_max=new_max, rope=rope)
    group = rng.choice([1, 1, 2, 3, 4, 8])
    # as much to read as the longest listed cases at most
    len_max = _log_int(rng, 1, max(1, min(32768, (64 * 1024 * 1024) // (n * kv_heads * head_dim))))
    new_max = 1
    if rng.random() < 0.4:  # several queries to a sequence
        most = (1 << 31) // (n * kv_heads * group * head_dim * len_max)
        new_max = _log_int(rng, 1, max(1, min(512, len_max, most)))
    window = _log_int(rng, 1, len_max) if rng.random() < 0.25 else 0
    return dict(op=op, n=n, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim, page=page, type=kind,
                len_min=rng.randint(new_max, max(new_max, len_max)), len_max=max(new_max, len_max),
                new_min=rng.randint(1, new_max), new_max=new_max, rope=rope, window=window,
                first=rng.random() < 0.25)


# ------------------------------------------------- sizes that a case implies


def _spread(lo, hi, n, step):
    """n whole numbers from lo to hi, evenly spread, in a scattered order."""
    if n == 1:
        return [hi]
    while math.gcd(step, n) != 1:
        step += 1
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _shape(case):
    """Each sequence's tokens (the new ones among them), its new tokens and
    the first key that its queries see."""
    n = case["n"]
    lens = _spread(case["len_min"], case["len_max"], n, 37)
    new = [min(t, m) for t, m in zip(_spread(case["new_min"], case["new_max"], n, 53), lens)]
    first = [0] * n
    if case.get("first"):  # a third padded, some beyond the last key: they see nothing
        first = [0 if i % 3 else (m if i % 6 == 0 else m // 3) for i, m in enumerate(lens)]
    return lens, new, first


def _visible(case):
    """Query/key pairs that the masks leave, and keys that some query sees."""
    pairs = keys = 0
    w = case["window"]
    for m, t, f in zip(*_shape(case)):
        lo_all = m
        for p in range(m - t, m):
            lo = max(f, p - w + 1 if w else 0, 0)
            pairs += max(0, p + 1 - lo)
            lo_all = min(lo_all, lo)
        keys += max(0, m - lo_all)
    return pairs, keys


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["type"]]
    if case["op"] == "logprobs":
        e = case["rows"] * case["vocab"]
        return dict(bytes=e * size + case["rows"] * (12 + 8 * case["top"]), flops=6 * e)
    lens, new, _ = _shape(case)
    hd = case["kv_heads"] * case["head_dim"]
    if case["op"] == "append":
        p = case["page"]
        block = [m - (m - t) // p * p for m, t in zip(lens, new)]  # tokens of the pages that are written
        # the new rows and what the pages held in, the pages' bytes and their values out
        held = sum(b - t for b, t in zip(block, new))
        return dict(bytes=2 * hd * (sum(new) * size + held + sum(block) + sum(block) * size),
                    flops=2 * hd * (6 * sum(new) + 3 * sum(block)))
    pairs, keys = _visible(case)
    rows = sum(new)
    return dict(bytes=2 * hd * keys + keys // case["page"] * case["kv_heads"] * 8
                + rows * case["heads"] * (2 * case["head_dim"] * size + 4),
                flops=4 * pairs * case["heads"] * case["head_dim"])


# ------------------------------------------------------------------ inputs


def _rope_table(positions, head_dim):
    """cos and sin of position * 10000^(-2i/head_dim), [positions][head_dim/2][2]."""
    f = 10000.0 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=DEV) / head_dim)
    a = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = TYPES[case["type"]]
    s = dict(case=case, stream=torch.cuda.current_stream().cuda_stream)
    if case["op"] == "logprobs":
        r, v, k = case["rows"], case["vocab"], case["top"]
        x = torch.empty(r, v, dtype=dt, device=DEV).normal_(0, 2.5, generator=g)
        # a few tokens that a decoder forbids, and a peak where the model is sure
        forbid = torch.randint(0, v, (r, min(v // 4, 90)), generator=g, device=DEV)
        x.scatter_(1, forbid, float("-inf"))
        peak = torch.randint(0, v, (r, 1), generator=g, device=DEV)
        x.scatter_(1, peak, (8 + 8 * torch.rand(r, 1, generator=g, device=DEV)).to(dt))
        other = torch.randint(0, v, (r, 1), generator=g, device=DEV)
        likely = torch.rand(r, 1, generator=g, device=DEV) < 0.7
        s.update(logits=x, targets=torch.where(likely, peak, other)[:, 0].int().contiguous(),
                 logprob=torch.zeros(r, device=DEV), entropy=torch.zeros(r, device=DEV),
                 ids=torch.zeros(r, k, dtype=torch.int32, device=DEV), top=torch.zeros(r, k, device=DEV))
        return s
    n, hk, d, page = case["n"], case["kv_heads"], case["head_dim"], case["page"]
    lens, new, first = _shape(case)
    width = -(-max(lens) // page)
    cpu = torch.Generator().manual_seed(seed)
    # The pages in a scattered order. An append touches a sequence's last
    # pages alone, so the earlier ones are one page that all share.
    pages_of = [-(-m // page) for m in lens]
    begin = [(m - t) // page if case["op"] == "append" else 0 for m, t in zip(lens, new)]
    pages = sum(p - b for p, b in zip(pages_of, begin)) + 1
    order = (torch.randperm(pages - 1, generator=cpu) + 1).tolist()
    table = torch.zeros(n, width, dtype=torch.int32)
    at = 0
    for i in range(n):
        c = pages_of[i] - begin[i]
        table[i, begin[i]:pages_of[i]] = torch.tensor(order[at:at + c], dtype=torch.int32)
        at += c
    row0 = torch.tensor([0] + new).cumsum(0).int()
    rows = int(row0[-1])
    # what the pages hold: bytes over the whole range, values of about unit size
    s.update(
        table=table.to(DEV), lens=torch.tensor(lens, dtype=torch.int32, device=DEV), row0=row0.to(DEV), rows=rows,
        first=torch.tensor(first, dtype=torch.int32, device=DEV) if case.get("first") else None,
        max_len=max(lens), max_new=max(new), pages=pages,
        pk=torch.randint(-127, 128, (pages, hk, page, d), generator=g, device=DEV, dtype=torch.int8),
        pv=torch.randint(-127, 128, (pages, hk, page, d), generator=g, device=DEV, dtype=torch.int8),
        scale=(0.5 + torch.rand(pages, hk, 2, generator=g, device=DEV)) / 73,
        rope=None if case["rope"] == "none" else _rope_table(width * page, d),
    )
    if case["op"] == "append":
        # keys and values side by side in one row, as a product of the layer leaves them
        kv = torch.empty(rows, 2, hk, d, dtype=dt, device=DEV).normal_(0, 1, generator=g)
        block = [m - (m - t) // page * page for m, t in zip(lens, new)]
        brow0 = torch.tensor([0] + block).cumsum(0).int()
        brows = int(brow0[-1])
        s.update(kv=kv, brow0=brow0.to(DEV), brows=brows, max_block=max(block),
                 out_k=torch.zeros(brows, hk, d, dtype=dt, device=DEV),
                 out_v=torch.zeros(brows, hk, d, dtype=dt, device=DEV))
    else:
        s.update(q=torch.empty(rows, case["heads"], d, dtype=dt, device=DEV).normal_(0, 1.5, generator=g),
                 out=torch.zeros(rows, case["heads"], d, dtype=dt, device=DEV),
                 lse=torch.zeros(rows, case["heads"], device=DEV))
    return s


# ------------------------------------------------------------------ the pass


def run(s):
    op = s["case"]["op"]
    if own:
        return _own(s, op)
    return {"append": _append, "attend": _attend, "logprobs": _logprobs}[op](s)


def _own(s, op):
    import gorelaxor_b200 as grx

    c, stream = s["case"], s["stream"]
    if op == "logprobs":
        grx.logprobs(s["logits"].data_ptr(), c["rows"], c["vocab"], dtype=c["type"], d_targets=s["targets"].data_ptr(),
                     top=c["top"], d_logprob=s["logprob"].data_ptr(), d_entropy=s["entropy"].data_ptr(),
                     d_top_ids=s["ids"].data_ptr(), d_top_logprobs=s["top"].data_ptr(), stream=stream)
        return s["logprob"], s["entropy"], s["ids"], s["top"]
    if "cache" not in s:  # the handles that a program makes once
        s["cache"] = grx.KV8(s["pk"].data_ptr(), s["pv"].data_ptr(), s["scale"].data_ptr(), s["pages"], c["page"],
                             c["kv_heads"], c["head_dim"])
        seqs = dict(n=c["n"], d_table=s["table"].data_ptr(), table_width=s["table"].shape[1],
                    d_len=s["lens"].data_ptr(), max_len=s["max_len"],
                    d_first=s["first"].data_ptr() if s["first"] is not None else None,
                    d_rope=s["rope"].data_ptr() if s["rope"] is not None else None,
                    rope_positions=s["rope"].shape[0] if s["rope"] is not None else 0, rope=c["rope"])
        one = s["max_new"] == 1  # a row for each sequence needs no row numbers
        s["seqs"] = grx.KV8Seqs(d_row0=None if one else s["row0"].data_ptr(), rows=s["rows"], max_new=s["max_new"],
                                **seqs)
        if op == "append":
            s["blocks"] = grx.KV8Seqs(d_row0=s["brow0"].data_ptr(), rows=s["brows"], max_new=s["max_block"], **seqs)
    if op == "append":
        h, d = c["kv_heads"], c["head_dim"]
        at, size = s["kv"].data_ptr(), s["kv"].element_size()
        s["cache"].append(s["seqs"], at, at + h * d * size, dtype=c["type"], k_strides=(2 * h * d, d),
                          v_strides=(2 * h * d, d), stream=stream)
        s["cache"].read(s["blocks"], s["out_k"].data_ptr(), s["out_v"].data_ptr(), dtype=c["type"], stream=stream)
        return s["out_k"], s["out_v"]
    s["cache"].attend(s["seqs"], c["heads"], s["q"].data_ptr(), s["out"].data_ptr(), dtype=c["type"],
                      window=c["window"], d_lse=s["lse"].data_ptr(), stream=stream)
    return s["out"], s["lse"]


# ---------------------------------------------------------- the plain forms


def _rows(lens, row0, rows):
    """The sequence and the position of each row."""
    new = row0[1:] - row0[:-1]
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEV), new, output_size=rows)
    return seq, lens[seq] - new[seq] + torch.arange(rows, device=DEV, dtype=torch.int32) - row0[seq]


def _rotate(x, pos, table, mode):
    """x [rows][heads][d] turned by the table's angles at its rows' positions."""
    if mode == "none":
        return x
    c, s = (table[pos.long()][:, None, :, j].to(x.dtype) for j in (0, 1))
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if mode == "pairs" else (x[..., :half], x[..., half:])
    y, z = a * c - b * s, a * s + b * c
    return torch.stack([y, z], -1).flatten(-2) if mode == "pairs" else torch.cat([y, z], -1)


def _append(s):
    """Rotation, scales and roundings in 64 bits: next to a border 32 would
    round some values to the other side."""
    case, page = s["case"], s["case"]["page"]
    seq, pos = _rows(s["lens"], s["row0"], s["rows"])
    at, slot = s["table"][seq, pos // page].long(), (pos % page).long()
    x = s["kv"].double()
    x = [_rotate(x[:, 0], pos, s["rope"], case["rope"]), x[:, 1]]
    begun = torch.zeros(s["pages"], dtype=torch.int32, device=DEV)  # pages that get their first token now
    begun.scatter_reduce_(0, at, (slot == 0).int(), "amax")
    for j, pool in enumerate((s["pk"], s["pv"])):
        amax = torch.zeros(s["pages"], case["kv_heads"], dtype=torch.float64, device=DEV)
        amax.scatter_reduce_(0, at[:, None].expand(-1, case["kv_heads"]), x[j].abs().amax(-1), "amax")
        old = s["scale"][:, :, j]
        old = torch.where(begun[:, None] > 0, torch.zeros_like(old), old)
        scale = torch.maximum(old, (amax / 127).float())
        back = torch.where(scale > 0, 1 / scale.double(), torch.zeros_like(amax))
        grown = (scale > old)[:, :, None, None]
        pool.copy_(torch.where(grown, (pool * (old.double() * back)[:, :, None, None]).round(), pool).to(torch.int8))
        pool[at, :, slot] = (x[j] * back[at][:, :, None]).round().clamp(-127, 127).to(torch.int8)
        s["scale"][:, :, j] = scale
    bseq, bpos = _rows(s["lens"], s["brow0"], s["brows"])
    bat, bslot = s["table"][bseq, bpos // page].long(), (bpos % page).long()
    return tuple((pool[bat, :, bslot].float() * s["scale"][bat][:, :, j, None]).to(TYPES[case["type"]])
                 for j, pool in enumerate((s["pk"], s["pv"])))


def _attend(s):
    case, page, d = s["case"], s["case"]["page"], s["case"]["head_dim"]
    n, hk = case["n"], case["kv_heads"]
    group = case["heads"] // hk
    seq, pos = _rows(s["lens"], s["row0"], s["rows"])
    width = s["table"].shape[1] * page
    pages = s["table"].long()

    def values(pool, j):  # [n][heads][tokens][d]
        x = pool[pages].float() * s["scale"][pages][..., j, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(n, hk, width, d)

    q = _rotate(s["q"].float(), pos, s["rope"], case["rope"])
    at = torch.arange(s["rows"], device=DEV, dtype=torch.int32) - s["row0"][seq]
    full = torch.zeros(n, s["max_new"], case["heads"], d, device=DEV)
    full[seq, at.long()] = q
    full = full.reshape(n, s["max_new"], hk, group, d).permute(0, 2, 1, 3, 4).reshape(n, hk, -1, d)
    w = full @ values(s["pk"], 0).mT
    w *= d ** -0.5
    # the query t of a sequence stands at the position len - new + t
    new = s["row0"][1:] - s["row0"][:-1]
    p = (s["lens"] - new)[:, None] + torch.arange(s["max_new"], device=DEV)
    key = torch.arange(width, device=DEV)
    seen = (key <= p[..., None]) & (key < s["lens"][:, None, None])
    if case["window"]:
        seen &= key > p[..., None] - case["window"]
    if s["first"] is not None:
        seen &= key >= s["first"][:, None, None]
    seen = seen[:, None, :, None].expand(n, 1, s["max_new"], group, width).reshape(n, 1, -1, width)
    w.masked_fill_(~seen, float("-inf"))
    top = w.amax(-1, keepdim=True)
    w = (w - torch.where(top > float("-inf"), top, torch.zeros_like(top))).exp_()
    total = w.sum(-1, keepdim=True)
    out = (w @ values(s["pv"], 1)) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + total.log())[..., 0]
    out = out.reshape(n, hk, s["max_new"], group, d).permute(0, 2, 1, 3, 4).reshape(n, s["max_new"], case["heads"], d)
    lse = lse.reshape(n, hk, s["max_new"], group).permute(0, 2, 1, 3).reshape(n, s["max_new"], case["heads"])
    return out[seq, at.long()].to(s["q"].dtype), lse[seq, at.long()].contiguous()


def _logprobs(s):
    """log softmax at the targets; the entropy as log1p(z) + sum p (m - x),
    whose terms are all positive; the largest logits, ties to the lowest index."""
    x = s["logits"].float()
    m, at = x.max(-1, keepdim=True)
    e = (x - m).exp_()
    rest = e.scatter(1, at, 0.0).sum(-1)
    lz = torch.log1p(rest)
    gap = torch.where(e > 0, (m - x) * e, torch.zeros_like(e))
    entropy = lz + gap.sum(-1) / (1 + rest)
    logprob = x.gather(1, s["targets"][:, None].long())[:, 0] - m[:, 0] - lz
    del e, gap
    # one whole number for value and index: the larger value first, then the lower index
    bits = (x + 0.0).view(torch.int32)
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    key += 0x7FFFFFFF - torch.arange(x.shape[1], device=DEV)
    ids = 0x7FFFFFFF - (key.topk(s["case"]["top"], -1).values & 0xFFFFFFFF)
    return logprob, entropy, ids.int(), x.gather(1, ids) - m - lz[:, None]


# ------------------------------------------------ the definitions in 64 bits


def _turn(x, pos, table, mode):
    """A pair (a, b) as the complex number a + ib, times cos + i sin."""
    if mode == "none":
        return x
    z = torch.view_as_complex(table[pos].double())[:, None]
    d = x.shape[-1]
    pair = x.reshape(*x.shape[:-1], d // 2, 2) if mode == "pairs" else torch.stack(x.split(d // 2, -1), -1)
    r = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
    return r.reshape(x.shape) if mode == "pairs" else torch.cat([r[..., 0], r[..., 1]], -1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        parts = []
        for x, t in zip(s["logits"].split(128), s["targets"].split(128)):
            lp = torch.log_softmax(x.double(), -1)
            k = case["top"]
            # from the logits, not from their logarithms, which may tie where the logits do not
            ids = torch.sort(x.double(), stable=True, dim=-1, descending=True).indices
            p = lp.exp()
            parts.append((lp.gather(1, t[:, None].long())[:, 0], -(p * lp).where(p > 0, 0.0).sum(-1),
                          ids[:, :k].int(), lp.gather(1, ids[:, :k])))
            del lp, ids, p
        return tuple(torch.cat(c) for c in zip(*parts))
    lens, new, first = _shape(case)
    page, d, hk = case["page"], case["head_dim"], case["kv_heads"]
    table = s["table"].tolist()
    out = ([], [])
    r = 0
    for i, (m, t) in enumerate(zip(lens, new)):
        pos = torch.arange(m - t, m, device=DEV)
        if case["op"] == "append":
            x = s["kv"][r:r + t].double()
            r += t
            x = (_turn(x[:, 0], pos, s["rope"], case["rope"]), x[:, 1])
            for j, pool in enumerate((s["pk"], s["pv"])):
                for b in range((m - t) // page, -(-m // page)):
                    lo, hi = max(m - t, b * page), min(m, (b + 1) * page)
                    held, mine = lo - b * page, x[j][lo - (m - t):hi - (m - t)]
                    old = s["scale"][table[i][b], :, j] if held else torch.zeros(hk, device=DEV)
                    # the definition's one 32-bit quantity: a stored scale
                    new_scale = torch.maximum(old, (mine.abs().amax((0, 2)) / 127).float()).double()
                    v = pool[table[i][b], :, :held].double()
                    again = (v * old[:, None, None]).div(new_scale[:, None, None]).round()
                    v = torch.where((new_scale > old)[:, None, None], again, v)
                    q = mine.div(new_scale[:, None]).round().clamp(-127, 127).nan_to_num(0.0)
                    v = torch.cat([v.permute(1, 0, 2), q])
                    out[j].append(v * new_scale[:, None])
            continue
        f, w = first[i], case["window"]
        q = _turn(s["q"][r:r + t].double(), pos, s["rope"], case["rope"])
        r += t
        pg = torch.tensor(table[i][:-(-m // page)], device=DEV)

        def tokens(pool, j):  # [heads][tokens][d]
            v = pool[pg].double() * s["scale"][pg][:, :, j, None, None].double()
            return v.transpose(0, 1).reshape(hk, -1, d)[:, :m]

        key = torch.arange(m, device=DEV)
        seen = (key <= pos[:, None]) & (key >= f) & ((key > pos[:, None] - w) if w else True)
        a = torch.einsum("thgd,hkd->htgk", q.reshape(t, hk, -1, d), tokens(s["pk"], 0)) / math.sqrt(d)
        a = a.masked_fill(~seen[None, :, None], float("-inf"))
        lse = torch.logsumexp(a, -1)
        a = (a - lse[..., None]).exp().nan_to_num(0.0)
        o = torch.einsum("htgk,hkd->thgd", a, tokens(s["pv"], 1))
        out[0].append(o.reshape(t, -1, d))
        out[1].append(lse.transpose(0, 1).reshape(t, -1))
    return tuple(torch.cat(c) for c in out)
