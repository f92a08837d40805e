"""Operators of a host that serves several conversations from one paged key-value cache, as cases that can be
timed and compared: the append (rotation of q and k, then k and v into their pages), attention over the pages for
single new tokens and for prompts (capped scores, a bias by distance, a window, prefix and document masks, the
attention weights summed per position), the eviction that goes by those sums, and the rules on logits that come
before sampling (penalties, biases, a mask of allowed tokens).

Head layouts are those of the 2.4B-shaped decoder (32/8 heads of 64) and of the reference file's geometry (16/2
heads of 128), both with 130,560 tokens, and generic ones (24/24 of 96, 8/1 of 256, 28/4 of 128, 20/4 of 80).

`own` false: each operator from elementary torch operations in 32 bits (positions' angles in 64).  `own` true: the
framework's entry points, called as a host program calls them.
"""
import math
import os
import random
import sys

import torch

own = False

VOCAB = 130560
HEADS = {"2.4b": (32, 8, 64), "ref": (16, 2, 128), "mha96": (24, 24, 96), "mqa256": (8, 1, 256),
         "gqa128": (28, 4, 128), "gqa80": (20, 4, 80)}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
ROPE_BASE = 10000.0


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one decode step of 64 conversations: each token's q and k rotated, k and v into its pages
        dict(name="append_decode", kind="append", heads="2.4b", type="f16", io="f32", page=16, n_seq=64,
             max_len=4096, new=1, mix=1),
        # four prompts of ragged lengths arrive together, one of them as the next turn of a long chat
        dict(name="append_prompts", kind="append", heads="ref", type="bf16", io="bf16", page=64, n_seq=4,
             max_len=8192, new=4096, mix=2),
        # one chat, one token, the framework's own fp32 rows: bound by latency
        dict(name="decode_one_513", kind="attention", heads="2.4b", type="f32", io="f32", page=64, n_seq=1,
             max_len=513, new=1, mix=0),
        # 48 conversations of ragged lengths, with the weights that eviction goes by and capped scores
        dict(name="decode_batch_weights", kind="attention", heads="2.4b", type="f16", io="f32", page=16, n_seq=48,
             max_len=4099, new=1, mix=3, softcap=30.0, weight=True),
        # two documents of 100,000 tokens, few heads: the length has to be split to fill the card
        dict(name="decode_long", kind="attention", heads="ref", type="bf16", io="bf16", page=128, n_seq=2,
             max_len=100003, new=1, mix=0),
        # a prompt up to its first token, fp32 activations
        dict(name="prompt_1024", kind="attention", heads="2.4b", type="f16", io="f32", page=16, n_seq=1,
             max_len=1024, new=1024, mix=0),
        # packed short documents and prefix-visible instructions, capped scores, a bias by distance
        dict(name="prompt_docs", kind="attention", heads="ref", type="bf16", io="bf16", page=32, n_seq=3,
             max_len=5003, new=5003, mix=4, softcap=50.0, slopes=True, prefix=77, docs=700),
        # the last chunk of a long prompt against all that came before it
        dict(name="prompt_chunk_16k", kind="attention", heads="ref", type="f16", io="f16", page=64, n_seq=1,
             max_len=16384, new=4096, mix=0),
        # eight chats grown to 4096 positions go back to 1024
        dict(name="evict_chats", kind="evict", heads="2.4b", type="f16", page=16, n_seq=8, max_len=4096, mix=5,
             budget=1024, first=4, recent=256),
        # a long document's cache to an eighth
        dict(name="evict_long", kind="evict", heads="ref", type="bf16", page=64, n_seq=1, max_len=65537, mix=0,
             budget=8192, first=16, recent=1000),
        # one conversation's logits before sampling
        dict(name="logits_one", kind="logits", n_seq=1, vocab=VOCAB, history=900, mix=0, biases=12, grammar=True),
        # a batch of 64, long histories
        dict(name="logits_batch", kind="logits", n_seq=64, vocab=VOCAB, history=8192, mix=6, biases=300,
             grammar=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "evict", "logits"])
    if kind == "logits":
        return dict(kind=kind, n_seq=_log_int(rng, 1, 64), vocab=_log_int(rng, 1000, VOCAB),
                    history=_log_int(rng, 1, 8192), mix=rng.randint(1, 1 << 20), biases=_log_int(rng, 1, 300),
                    grammar=rng.random() < 0.7)
    c = dict(kind=kind, heads=rng.choice(sorted(HEADS)), type=rng.choice(["f32", "f16", "bf16"]),
             page=rng.choice([8, 16, 32, 64, 128, 256]), mix=rng.randint(1, 1 << 20))
    H, KH, D = HEADS[c["heads"]]
    if kind == "evict":
        c["max_len"] = _log_int(rng, 64, 65536)
        c["n_seq"] = _log_int(rng, 1, max(1, min(32, 65536 // c["max_len"])))
        c["budget"] = rng.randint(16, max(17, c["max_len"] // 2))
        c["first"] = rng.randint(0, 4)
        c["recent"] = rng.randint(0, c["budget"] // 3)
        return c
    c["io"] = rng.choice(["f32", c["type"]])
    most = 2 ** 27 // (KH * D)  # positions of all sequences
    if kind == "append":
        c["max_len"] = _log_int(rng, 1, 16384)
        c["n_seq"] = _log_int(rng, 1, max(1, min(64, most // c["max_len"])))
        c["new"] = 1 if rng.random() < 0.4 else _log_int(rng, 1, min(c["max_len"], max(1, 16384 // c["n_seq"])))
        return c
    if rng.random() < 0.5:  # single tokens, now and then a few at once
        c["max_len"] = _log_int(rng, 1, 60000)
        c["n_seq"] = _log_int(rng, 1, max(1, min(64, most // c["max_len"])))
        c["new"] = 1 if rng.random() < 0.7 else min(c["max_len"], rng.randint(2, 5))
        c["weight"] = rng.random() < 0.4
    else:
        c["max_len"] = _log_int(rng, 16, 5600)
        c["n_seq"] = _log_int(rng, 1, max(1, min(8, 5600 // c["max_len"])))
        c["new"] = max(1, int(c["max_len"] * rng.choice([1.0, 1.0, rng.uniform(0.05, 1.0)])))
        if rng.random() < 0.4:
            c["docs"] = _log_int(rng, 20, 2000)
        if rng.random() < 0.3:
            c["prefix"] = _log_int(rng, 1, c["max_len"])
    if rng.random() < 0.4:
        c["softcap"] = round(rng.uniform(15.0, 60.0), 1)
    if rng.random() < 0.3:
        c["slopes"] = True
    if rng.random() < 0.3:
        c["window"] = _log_int(rng, 1, 4096)
    return c


# -------------------------------------------------- what a case's name leaves open

def _ragged(case, n, most, salt):
    """n sizes from 1 to most, the first of them the largest: lengths of conversations are ragged."""
    r = random.Random(case["mix"] * 8 + salt)
    return [most] + [r.randint(max(1, most // 16), most) for _ in range(n - 1)] if case["mix"] else [most] * n


def _lens(case):
    return _ragged(case, case["n_seq"], case["max_len"], 1)


def _news(case):
    if case["new"] == 1:
        return [1] * case["n_seq"]
    return [min(n, l) for n, l in zip(_ragged(case, case["n_seq"], case["new"], 2), _lens(case))]


def _doc_ids(case, b, length):
    """Document of each position: runs of ragged lengths; the last positions of a padded sequence have none."""
    r = random.Random(case["mix"] * 64 + b)
    ids, d = [], 0
    while len(ids) < length:
        ids += [d] * r.randint(max(1, case["docs"] // 4), 2 * case["docs"])
        d += 1
    ids = ids[:length]
    if length > 40:
        ids[-7:] = [-1] * 7
    return ids


def _prefix(case, b):
    return case["prefix"] if b % 2 == 0 else 0


def _histories(case):
    return _ragged(case, case["n_seq"], case["history"], 3)


# ---------------------------------------------------------------------- prepare

def _rand(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(g, first, n_seq, per_seq):
    """Each sequence's pages: the pool's pages in no order, as they come from a free list."""
    p = torch.randperm(n_seq * per_seq, generator=g, device="cuda").to(torch.int32) + first
    return p.view(n_seq, per_seq).contiguous()


def _starts(news):
    at = [0]
    for n in news:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["kind"] == "logits":
        n, V = case["n_seq"], case["vocab"]
        h = _starts(_histories(case))
        s["logits"] = _rand(g, (n, V), torch.float32, 2.5)
        # tokens come back: history is drawn from a part of the vocabulary that is dense at its start
        u = torch.rand(h[-1], generator=g, device="cuda")
        s["history"] = (u * u * u * V).to(torch.int32).clamp_(max=V - 1)
        s["history_starts"] = _ints(h)
        for name, lo, hi in (("repetition", 1.0, 1.3), ("presence", 0.0, 0.6), ("frequency", 0.0, 0.3)):
            s[name] = torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo
        ids = [torch.randperm(V, generator=g, device="cuda")[:case["biases"]] for _ in range(n)]
        s["bias_ids"] = torch.cat(ids).to(torch.int32)
        s["bias"] = _rand(g, (s["bias_ids"].numel(),), torch.float32, 3.0)
        s["bias_starts"] = _ints([i * ids[0].numel() for i in range(n + 1)])
        if case["grammar"]:
            words = (V + 31) // 32
            s["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (n, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        torch.cuda.synchronize()
        return s
    H, KH, D = HEADS[case["heads"]]
    dt, page, n = TYPES[case["type"]], case["page"], case["n_seq"]
    per_seq = -(-case["max_len"] // page)
    total = n * per_seq
    if case["kind"] == "evict":
        per_dst = -(-case["budget"] // page)
        s["dst_pages"] = _pages(g, total, n, per_dst)
        total += n * per_dst
    s["pages"] = _pages(g, 0, n, per_seq)
    s["lens"] = _ints(_lens(case))
    s["k"], s["v"] = (_rand(g, (total, page, KH, D), dt) for _ in range(2))
    if case["kind"] == "evict":
        # a few positions gather most of the weight
        s["weight"] = torch.empty((total, KH, page), device="cuda").exponential_(generator=g) ** 3
        s["kept"] = torch.zeros((n, KH, case["budget"]), dtype=torch.int32, device="cuda")
        s["dst_lens"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        return s
    io, at = TYPES[case["io"]], _starts(_news(case))
    s["starts"] = _ints(at)
    s["rows"] = at[-1]
    s["max_new"] = max(_news(case))
    s["q"] = _rand(g, (at[-1], H, D), io, 1.5)
    if case["kind"] == "append":
        s["k_new"], s["v_new"] = (_rand(g, (at[-1], KH, D), io) for _ in range(2))
    else:
        s["out"] = torch.zeros((at[-1], H, D), dtype=io, device="cuda")
        if case.get("weight"):
            s["weight"] = torch.zeros((total, KH, page), device="cuda")
        if case.get("slopes"):
            s["slopes"] = torch.exp2(-8.0 * torch.arange(1, H + 1, device="cuda", dtype=torch.float32) / H)
        if case.get("prefix"):
            s["prefix"] = _ints([_prefix(case, b) for b in range(n)])
        if case.get("docs"):
            L = case["max_len"]
            s["docs"] = _ints([d + [-1] * (L - len(d)) for d in (_doc_ids(case, b, l) for b, l in enumerate(_lens(case)))])
    torch.cuda.synchronize()
    return s


# -------------------------------------------------------- the framework's calls

_ctx = None


def _mcpm():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "minicpm5.cpp_amd", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    import mcpm
    return mcpm


def _bind(s):
    """The descriptors that a host fills once for its buffers, and the call they go into."""
    global _ctx
    mcpm, c = _mcpm(), s["case"]
    if _ctx is None:
        _ctx = mcpm.Context(0)
    lib, ctx = _ctx.lib, _ctx.h
    p = lambda name: s[name].data_ptr() if name in s else None  # noqa: E731
    if c["kind"] == "logits":
        rules = mcpm.LogitRules(n_seq=c["n_seq"], vocab=c["vocab"], stride=c["vocab"], history=p("history"),
                                history_starts=p("history_starts"), repetition=p("repetition"), presence=p("presence"),
                                frequency=p("frequency"), bias_ids=p("bias_ids"), bias=p("bias"),
                                bias_starts=p("bias_starts"), allowed=p("allowed"),
                                allowed_stride=(c["vocab"] + 31) // 32)
        return mcpm.check, lib.mcpm_process_logits, (ctx, p("logits"), rules)
    H, KH, D = HEADS[c["heads"]]
    types = {"f32": mcpm.TYPE_F32, "f16": mcpm.TYPE_F16, "bf16": mcpm.TYPE_BF16}
    kv = mcpm.PagedKV(type=types[c["type"]], n_pages=s["k"].shape[0], page_size=c["page"], n_kv_heads=KH, head_dim=D,
                      page_stride=c["page"] * KH * D, pos_stride=KH * D, head_stride=D, k=p("k"), v=p("v"),
                      weight=p("weight"))
    batch = mcpm.PagedBatch(n_seq=c["n_seq"], n_rows=s.get("rows", 0), max_new=s.get("max_new", 0),
                            max_len=c["max_len"], max_pages=s["pages"].shape[1], pages=p("pages"), lens=p("lens"),
                            starts=p("starts"))
    if c["kind"] == "evict":
        return mcpm.check, lib.mcpm_paged_evict, (ctx, kv, batch, c["budget"], c["first"], c["recent"], p("dst_pages"),
                                                  s["dst_pages"].shape[1], p("kept"), p("dst_lens"))
    if c["kind"] == "append":
        return mcpm.check, lib.mcpm_paged_append, (ctx, kv, batch, types[c["io"]], p("k_new"), p("v_new"), KH * D, p("q"),
                                                   H * D, H, ROPE_BASE)
    rules = mcpm.AttnRules(scale=0.0, softcap=c.get("softcap", 0.0), window=c.get("window", 0), slopes=p("slopes"),
                           prefix=p("prefix"), docs=p("docs"), docs_stride=c["max_len"])
    return mcpm.check, lib.mcpm_paged_attention, (ctx, p("out"), H * D, p("q"), H * D, types[c["io"]], H, kv, batch, rules)


def _outputs(s):
    names = {"logits": ["logits"], "append": ["k", "v", "q"], "evict": ["k", "v", "weight", "kept", "dst_lens"],
             "attention": ["out", "weight"]}[s["case"]["kind"]]
    return {n: s[n] for n in names if n in s}


def run(state):
    if own:
        if "call" not in state:
            state["call"] = _bind(state)
        check, fn, args = state["call"]
        check(fn(*args))
    else:
        _PLAIN[state["case"]["kind"]](state)
    return _outputs(state)


# -------------------------------------------------------------- the plain forms

def _rows_of(s):
    """Sequence and position of each row of q."""
    starts = s["starts"].long()
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    pos = s["lens"].long()[seq] - starts[seq + 1] + row
    return row, seq, pos


def _rotate(x, pos):
    D = x.shape[-1]
    i = torch.arange(0, D, 2, device="cuda", dtype=torch.float64)
    a = pos.double()[:, None] * torch.pow(ROPE_BASE, -i / D)
    c, sn = torch.cos(a).float()[:, None, :], torch.sin(a).float()[:, None, :]
    x0, x1 = x[..., 0::2].float(), x[..., 1::2].float()
    return torch.stack([x0 * c - x1 * sn, x0 * sn + x1 * c], dim=-1).flatten(-2)


def _plain_append(s):
    page = s["case"]["page"]
    row, seq, pos = _rows_of(s)
    at = s["pages"].long()[seq, pos // page], pos % page
    s["k"][at] = _rotate(s["k_new"], pos).to(s["k"].dtype)
    s["v"][at] = s["v_new"].float().to(s["v"].dtype)
    s["q"].copy_(_rotate(s["q"], pos).to(s["q"].dtype))


def _plain_attention(s):
    c = s["case"]
    H, KH, D = HEADS[c["heads"]]
    G, n, L, N, page = H // KH, c["n_seq"], c["max_len"], s["max_new"], c["page"]
    row, seq, pos = _rows_of(s)
    at = row - s["starts"].long()[seq]
    q = torch.zeros((n, N, H, D), device="cuda")
    q[seq, at] = s["q"].float()
    rpos = torch.full((n, N), -1, device="cuda", dtype=torch.int64)
    rpos[seq, at] = pos
    k, v = (s[x][s["pages"].long()].view(n, -1, KH, D)[:, :L].float().permute(0, 2, 1, 3).contiguous() for x in "kv")
    q = q.view(n, N, KH, G, D).permute(0, 2, 1, 3, 4).reshape(n, KH, N * G, D)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, KH, N, G, L)
    score *= 1.0 / math.sqrt(D)
    if c.get("softcap"):
        score = torch.tanh(score / c["softcap"]) * c["softcap"]
    j = torch.arange(L, device="cuda")
    far = rpos[:, :, None] - j
    if c.get("slopes"):
        score -= far.abs().float()[:, None, :, None, :] * s["slopes"].view(1, KH, 1, G, 1)
    seen = far >= 0
    if c.get("prefix"):
        seen |= j < s["prefix"].long()[:, None, None]
    if c.get("window"):
        seen &= far < c["window"]
    seen &= (rpos >= 0)[:, :, None] & (j < s["lens"].long()[:, None, None])
    if c.get("docs"):
        docs = s["docs"].long()
        mine = torch.gather(docs, 1, rpos.clamp(min=0))
        seen &= (docs[:, None, :] == mine[:, :, None]) & (mine >= 0)[:, :, None]
    score = torch.where(seen[:, None, :, None, :], score, -math.inf)
    top = score.amax(dim=-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(score - top)
    z = p.sum(dim=-1, keepdim=True)
    p = p / torch.where(z > 0, z, 1.0)
    out = torch.matmul(p.view(n, KH, N * G, L), v).view(n, KH, N, G, D).permute(0, 2, 1, 3, 4)
    s["out"].copy_(out.reshape(n, N, H, D)[seq, at].to(s["out"].dtype))
    if "weight" in s:
        b = torch.arange(n, device="cuda")[:, None].expand(n, L)
        inside = j[None, :] < s["lens"].long()[:, None]
        where = s["pages"].long()[b, j // page][inside], (j % page)[None, :].expand(n, L)[inside]
        s["weight"].transpose(1, 2)[where] += p.sum(dim=(2, 3)).transpose(1, 2)[inside]


def _plain_evict(s):
    c = s["case"]
    H, KH, D = HEADS[c["heads"]]
    page, n, L, B = c["page"], c["n_seq"], c["max_len"], c["budget"]
    lens, j = s["lens"].long(), torch.arange(L, device="cuda")
    w = s["weight"][s["pages"].long()].permute(0, 2, 1, 3).reshape(n, KH, -1)[:, :, :L]
    always = (j < c["first"]) | (j >= lens[:, None] - c["recent"])
    w = torch.where(always[:, None, :], math.inf, w)
    w = torch.where((j < lens[:, None])[:, None, :], w, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :, :B]
    keep = lens.clamp(max=B)
    slot = torch.arange(order.shape[-1], device="cuda")
    order = torch.where(slot < keep[:, None, None], order, L)  # those past a short sequence's end go last
    order = torch.sort(order, dim=-1).values
    s["kept"].fill_(-1)
    s["kept"][:, :, :order.shape[-1]] = torch.where(order < L, order, -1).to(torch.int32)
    s["dst_lens"].copy_(keep.to(torch.int32))
    b, h, t = torch.nonzero(order < L, as_tuple=True)
    src = order[b, h, t]
    sp, so = s["pages"].long()[b, src // page], src % page
    dp, do = s["dst_pages"].long()[b, t // page], t % page
    s["k"][dp, do, h] = s["k"][sp, so, h]
    s["v"][dp, do, h] = s["v"][sp, so, h]
    s["weight"][dp, h, do] = s["weight"][sp, h, so]


def _plain_logits(s):
    c = s["case"]
    n, V = c["n_seq"], c["vocab"]
    x = s["logits"]
    hs = s["history_starts"].long()
    seq = torch.searchsorted(hs, torch.arange(s["history"].numel(), device="cuda"), right=True) - 1
    count = torch.zeros((n, V), device="cuda")
    count.index_put_((seq, s["history"].long()), torch.ones(seq.numel(), device="cuda"), accumulate=True)
    rep = s["repetition"][:, None]
    y = torch.where(x > 0, x / rep, x * rep) - (s["frequency"][:, None] * count + s["presence"][:, None])
    y = torch.where(count > 0, y, x)
    bs = s["bias_starts"].long()
    seq = torch.searchsorted(bs, torch.arange(s["bias_ids"].numel(), device="cuda"), right=True) - 1
    y[seq, s["bias_ids"].long()] += s["bias"]
    if "allowed" in s:
        i = torch.arange(V, device="cuda")
        y = torch.where((s["allowed"][:, i // 32] >> (i % 32)) & 1 != 0, y, -math.inf)
    x.copy_(y)


_PLAIN = {"append": _plain_append, "attention": _plain_attention, "evict": _plain_evict, "logits": _plain_logits}


# ------------------------------------------------------- what a pass has to do

def _seen(case, b, length, new):
    """Visible pairs of (row, key) of one sequence, and how many of its keys are seen at all."""
    window, docs = case.get("window") or length, case.get("docs")
    prefix = min(length, _prefix(case, b)) if case.get("prefix") else 0
    if not docs:
        pairs, first = 0, length
        for pos in range(length - new, length):
            lo = max(0, pos - window + 1)
            pairs += max(pos + 1, prefix) - lo
            first = min(first, lo)
        return pairs, length - first
    ids = _doc_ids(case, b, length)
    begin, end, pairs, keys, top = {}, {}, 0, 0, 0
    for j, d in enumerate(ids):
        if d >= 0:
            begin.setdefault(d, j)
            end[d] = j + 1
    for pos in range(length - new, length):  # the rows' ranges of keys come in order
        d = ids[pos]
        if d < 0:
            continue
        lo, hi = max(begin[d], pos - window + 1), min(end[d], max(pos + 1, prefix))
        pairs += hi - lo
        keys += max(0, hi - max(lo, top))
        top = max(top, hi)
    return pairs, keys


def work(case):
    if case["kind"] == "logits":
        n, V = case["n_seq"], case["vocab"]
        nbytes = 8 * n * V + 4 * sum(_histories(case)) + 8 * n * case["biases"]
        nbytes += 4 * n * ((V + 31) // 32) if case["grammar"] else 0
        return {"bytes": nbytes, "flops": 4 * n * V}
    H, KH, D = HEADS[case["heads"]]
    e = SIZE[case["type"]]
    if case["kind"] == "evict":
        kept = sum(min(l, case["budget"]) for l in _lens(case))
        return {"bytes": KH * (4 * sum(_lens(case)) + kept * (4 * D * e + 8 + 4)), "flops": 4 * KH * sum(_lens(case))}
    rows, i = sum(_news(case)), SIZE[case["io"]]
    if case["kind"] == "append":
        return {"bytes": rows * D * (2 * KH * (i + e) + 2 * H * i), "flops": rows * D * 3 * (H + KH)}
    pairs = keys = 0
    for b, (l, new) in enumerate(zip(_lens(case), _news(case))):
        p, k = _seen(case, b, l, new)
        pairs, keys = pairs + p, keys + k
    nbytes = 2 * keys * KH * D * e + 2 * rows * H * D * i + (8 * keys * KH if case.get("weight") else 0)
    return {"bytes": nbytes, "flops": 4 * pairs * H * D}


# --------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "evict": lambda s: None, "logits": _exact_logits}[case["kind"]](s)


def _exact_rope(x, pos):
    """x [rows, heads, D] as complex pairs times exp(i angle)."""
    D = x.shape[-1]
    z = torch.view_as_complex(x.double().reshape(x.shape[0], x.shape[1], D // 2, 2).contiguous())
    a = pos.double()[:, None] * torch.exp(-math.log(ROPE_BASE) * 2.0 * torch.arange(D // 2, device="cuda", dtype=torch.float64) / D)
    return torch.view_as_real(z * torch.polar(torch.ones_like(a), a)[:, None, :]).reshape(x.shape)


def _exact_append(s):
    c = s["case"]
    k, v, q, page = s["k"].double(), s["v"].double(), s["q"].double(), c["page"]
    at = _starts(_news(c))
    for b, (l, new) in enumerate(zip(_lens(c), _news(c))):
        rows, pos = slice(at[b], at[b] + new), torch.arange(l - new, l, device="cuda")
        table = s["pages"][b].long()
        k[table[pos // page], pos % page] = _exact_rope(s["k_new"][rows], pos)
        v[table[pos // page], pos % page] = s["v_new"][rows].double()
        q[rows] = _exact_rope(s["q"][rows], pos)
    return {"k": k, "v": v, "q": q}


def _exact_attention(s):
    c = s["case"]
    H, KH, D = HEADS[c["heads"]]
    G, page = H // KH, c["page"]
    out, at = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda"), _starts(_news(c))
    weight = s["weight"].double() if "weight" in s else None
    for b, (l, new) in enumerate(zip(_lens(c), _news(c))):
        kc, vc = (s[x][s["pages"][b].long()].reshape(-1, KH, D)[:l] for x in "kv")
        j = torch.arange(l, device="cuda")
        doc = torch.tensor(_doc_ids(c, b, l), device="cuda") if c.get("docs") else None
        got = torch.zeros((KH, l), dtype=torch.float64, device="cuda")
        step = max(1, (1 << 25) // l)
        for t0 in range(0, new, step):
            pos = torch.arange(l - new + t0, l - new + min(new, t0 + step), device="cuda")
            see = j[None, :] <= pos[:, None]
            if c.get("prefix"):
                see = see | (j < _prefix(c, b))[None, :]
            if c.get("window"):
                see = see & (pos[:, None] - j[None, :] < c["window"])
            if doc is not None:
                see = see & (doc[None, :] == doc[pos][:, None]) & (doc >= 0)[None, :]
            rows = slice(at[b] + t0, at[b] + t0 + pos.numel())
            for h in range(H):
                x = (s["q"][rows, h].double() @ kc[:, h // G].double().t()) / math.sqrt(D)
                if c.get("softcap"):
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                if c.get("slopes"):
                    x = x - float(s["slopes"][h]) * (pos[:, None] - j[None, :]).abs().double()
                x = x.masked_fill(~see, -math.inf)
                p = torch.nan_to_num(torch.softmax(x, dim=-1), nan=0.0)
                out[rows, h] = p @ vc[:, h // G].double()
                got[h // G] += p.sum(dim=0)
        if weight is not None:
            weight[s["pages"][b].long()[j // page], :, j % page] += got.t()
    return {"out": out, "weight": weight} if weight is not None else {"out": out}


def _exact_logits(s):
    c = s["case"]
    V = c["vocab"]
    y, h, bs = s["logits"].double(), s["history_starts"].tolist(), s["bias_starts"].tolist()
    bit = torch.arange(V, device="cuda")
    for b in range(c["n_seq"]):
        n = torch.bincount(s["history"][h[b]:h[b + 1]].long(), minlength=V).double()
        r, row = float(s["repetition"][b]), y[b].clone()
        hit = n > 0
        row[hit] = torch.where(row[hit] > 0, row[hit] / r, row[hit] * r) - float(s["presence"][b]) - float(s["frequency"][b]) * n[hit]
        row[s["bias_ids"][bs[b]:bs[b + 1]].long()] += s["bias"][bs[b]:bs[b + 1]].double()
        if c["grammar"]:
            row[(s["allowed"][b].long()[bit // 32] >> (bit % 32)) & 1 == 0] = -math.inf
        y[b] = row
    return {"logits": y}
