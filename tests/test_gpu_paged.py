"""The operators over many sequences on the GPU against their definitions in 64 bits (paged_ref): the append,
attention of single tokens and of prompts, the eviction, the rules on logits, and a run of them together."""
import ctypes as C

import numpy as np
import pytest

import mcpm
import paged_ref as R
from conftest import announce
from paged_ref import BF16, F16, F32, NAME

pytestmark = pytest.mark.gpu

HEADS = {"mha": (4, 4, 64), "gqa4": (32, 8, 64), "gqa8": (16, 2, 128), "mqa256": (8, 1, 256), "gqa7_96": (14, 2, 96),
         "gqa5_80": (10, 2, 80), "g20_8": (20, 1, 8), "g3_40": (6, 2, 40), "g1_200": (2, 2, 200)}
TYPES = [(F32, F32), (F16, F32), (F16, F16), (BF16, F32), (BF16, BF16)]
IDS = [f"{NAME[t]}-{NAME[io]}" for t, io in TYPES]

_KEEP = []


@pytest.fixture(autouse=True)
def _keep_uploads(ctx):
    yield
    ctx.sync()
    _KEEP.clear()


def up(ctx, a):
    if a is None:
        return None
    buf = ctx.upload(np.ascontiguousarray(a) if np.asarray(a).size else np.zeros(4, np.int32))
    _KEEP.append(buf)
    return buf


def ptr(buf):
    return buf.ptr if buf is not None else None


class Dev:
    """A cache and a batch on the device, with their descriptors."""

    def __init__(self, ctx, cache, tables, lens, news=None, starts=None, n_rows=None, max_len=None, max_new=None):
        self.ctx, self.cache = ctx, cache
        tables = np.asarray(tables, np.int32)
        assert tables.ndim == 2 and len(tables) == len(lens)
        self.k, self.v, self.w = up(ctx, cache.k), up(ctx, cache.v), up(ctx, cache.weight)
        if starts is None and news is not None:
            starts = R.spans(lens, news)
        self.bufs = [up(ctx, tables), up(ctx, np.asarray(lens, np.int32)),
                     up(ctx, np.asarray(starts, np.int32)) if starts is not None else None]
        self.kv = mcpm.PagedKV(cache.t, cache.n_pages, cache.page, cache.kvh, cache.hd, *cache.strides, self.k.ptr,
                               self.v.ptr, ptr(self.w))
        rows = n_rows if n_rows is not None else (starts[-1] if starts is not None else len(lens))
        self.batch = mcpm.PagedBatch(len(lens), rows, max_new if max_new is not None else max([1] if news is None else news, default=0),
                                     max_len if max_len is not None else max(lens, default=0), tables.shape[1] if len(lens) else 0,
                                     *[ptr(b) for b in self.bufs])

    def image(self, which):
        buf = {"k": self.k, "v": self.v, "weight": self.w}[which]
        a = getattr(self.cache, which)
        return self.ctx.download(buf, a.dtype, a.shape)


def tables_of(rng, lens, page, n_pages, extra=0):
    per = max(1, max((-(-n // page) for n in lens), default=1)) + extra
    assert n_pages >= per * len(lens)
    return rng.permutation(n_pages)[:per * len(lens)].reshape(len(lens), per).astype(np.int32)


def rules_struct(ctx, rules):
    docs = rules.get("docs")
    return mcpm.AttnRules(rules.get("scale", 0.0), rules.get("softcap", 0.0), rules.get("window", 0),
                          ptr(up(ctx, rules.get("slopes"))), ptr(up(ctx, rules.get("prefix"))), ptr(up(ctx, docs)),
                          0 if docs is None else docs.shape[1])


def run_attention(ctx, dev, q, io, H, rules, pad=0, n_extra_rows=0):
    hd = dev.cache.hd
    step = 4 if io == F32 else 8
    stride = H * hd + pad * step
    img = R.store(np.full((q.shape[0], stride), 7.0), io)
    img[:, :H * hd] = q.reshape(q.shape[0], -1)
    qd = up(ctx, img)
    od = up(ctx, R.store(np.full((q.shape[0], stride), -3.0), io))
    mcpm.check(ctx.lib.mcpm_paged_attention(ctx.h, od.ptr, stride, qd.ptr, stride, io, H, C.byref(dev.kv),
                                            C.byref(dev.batch), C.byref(rules_struct(ctx, rules))))
    got = ctx.download(od, img.dtype, img.shape)
    assert (R.load(got[:, H * hd:], io) == -3.0).all(), "wrote between rows"
    return R.load(got[:, :H * hd], io).reshape(q.shape[0], H, hd)


def check_attention(ctx, name, heads, t, io, lens, news, page=16, rules=None, order="phd", pad=0, weight=False, seed=0,
                    scale_q=1.5, edit=None):
    """One call against the definition; edit(cache, tables) may spoil what no row sees."""
    H, KH, hd = heads
    rules = rules or {}
    rng = np.random.default_rng(seed)
    per = max(1, max(-(-n // page) for n in lens))
    cache = R.Cache(t, per * len(lens) + 3, page, KH, hd, order, pad, weight, rng)
    tables = tables_of(rng, lens, page, cache.n_pages)
    if weight:
        cache.weight[:] = rng.random(cache.weight.shape)
    q = R.store(rng.standard_normal((sum(news), H * hd)) * scale_q, io)
    if edit:
        edit(cache, tables)
    announce(f"attention {name} H={H}/{KH}x{hd} {NAME[t]}/{NAME[io]} lens={lens} news={news} page={page} {sorted(rules)}")
    dev = Dev(ctx, cache, tables, lens, news)
    want, bound, w, wb = R.attention(cache, tables, lens, news, q, io, H, rules)
    got = run_attention(ctx, dev, q, io, H, rules, pad)
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.size} outputs off, the worst by {np.abs(got - want).max()}"
    if weight:
        dw = np.abs(dev.image("weight").astype(np.float64) - cache.weight - w)
        # the sum is added to what the weight held: one more rounding of it
        assert (dw <= wb + 2.0 ** -23 * (w + cache.weight)).all(), dw.max()
    return dev, got


# ------------------------------------------------------------- single tokens

@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
@pytest.mark.parametrize("heads", sorted(HEADS))
def test_decode_heads_and_types(ctx, heads, t, io):
    check_attention(ctx, heads, HEADS[heads], t, io, [1, 37, 130, 16, 64], [1] * 5, seed=len(heads))


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 511, 513, 1025])
def test_decode_lengths(ctx, n):
    for t, io in ((F32, F32), (F16, F32), (BF16, BF16)):
        check_attention(ctx, "length", (8, 2, 64), t, io, [n], [1], page=32, seed=n)


@pytest.mark.parametrize("page", [1, 2, 8, 64, 256, 1024])
@pytest.mark.parametrize("order", ["phd", "hpd"])
def test_decode_pages_and_strides(ctx, page, order):
    check_attention(ctx, "strides", (8, 2, 64), F16, F32, [300, 5, 77], [1, 1, 1], page=page, order=order, pad=1, seed=page)
    check_attention(ctx, "strides", (4, 2, 40), F32, F32, [300, 5, 77], [1, 1, 1], page=page, order=order, pad=1, seed=page)


@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
def test_decode_long_is_split_and_joined(ctx, t, io):
    check_attention(ctx, "long", (8, 2, 128), t, io, [9001, 1, 2500], [1, 1, 1], page=64, seed=5)
    check_attention(ctx, "long weights", (8, 2, 64), t, io, [5003, 700], [1, 1], page=64, seed=6, weight=True)


@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
@pytest.mark.parametrize("heads", sorted(HEADS))
def test_decode_weights(ctx, heads, t, io):
    """The weights that groups of any number of heads add, for one token and a few."""
    check_attention(ctx, heads, HEADS[heads], t, io, [1, 65, 300], [1, 1, 1], rules=dict(softcap=30.0), weight=True, seed=21)
    if HEADS[heads][0] // HEADS[heads][1] * 3 <= 32:
        check_attention(ctx, heads, HEADS[heads], t, io, [70, 400], [3, 2], weight=True, seed=22)


@pytest.mark.parametrize("n_seq", [40, 256, 257, 300])
def test_many_ragged_sequences(ctx, n_seq):
    """More (sequence, kv head) pairs than CUs, lengths from 0 on, some sequences in several parts."""
    rng = np.random.default_rng(24)
    lens = [int(n) for n in rng.integers(0, 60, n_seq)]
    lens[3], lens[n_seq - 2] = 2500, 1300
    for t, io in ((F16, F32), (BF16, BF16)):
        check_attention(ctx, "many", (8, 8, 16), t, io, lens, [1] * n_seq, page=64, weight=True, seed=25)


@pytest.mark.parametrize("new", [2, 3, 4, 5, 16, 17])
def test_a_few_tokens_at_once(ctx, new):
    for t, io in ((F32, F32), (F16, F32), (BF16, BF16)):
        check_attention(ctx, "few", (8, 2, 64), t, io, [300, new, 40], [new, new, 1], page=16, seed=new, weight=True)


RULES = {
    "softcap": dict(softcap=4.0),
    "slopes": dict(slopes=True),
    "window1": dict(window=1),
    "window50": dict(window=50),
    "prefix": dict(prefix=[60, 0, 1000]),
    "docs": dict(docs=True),
    "all": dict(softcap=9.0, slopes=True, window=70, prefix=[20, 33, 0], docs=True, scale=0.21),
}


def make_rules(name, H, lens, rng):
    r = dict(RULES[name])
    if r.get("slopes"):
        r["slopes"] = (2.0 ** (-8.0 * np.arange(1, H + 1) / H)).astype(np.float32)
    if r.get("prefix"):
        r["prefix"] = np.array((r["prefix"] * len(lens))[:len(lens)], np.int32)
    if r.get("docs"):
        L = max(lens) + 3
        d = np.cumsum(rng.random((len(lens), L)) < 0.06, axis=1).astype(np.int32)
        d[:, 11:13] = -1  # positions of no document
        for b, n in enumerate(lens):
            d[b, max(0, n - 2):n] = -1 if b == 0 else d[b, max(0, n - 2):n]
        r["docs"] = d
    return r


@pytest.mark.parametrize("rule", sorted(RULES))
@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
def test_rules_single_tokens(ctx, rule, t, io):
    lens = [150, 97, 33]
    rules = make_rules(rule, 8, lens, np.random.default_rng(3))
    check_attention(ctx, rule, (8, 2, 64), t, io, lens, [1, 1, 1], rules=rules, weight=True, seed=7)


@pytest.mark.parametrize("rule", sorted(RULES))
@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
def test_rules_prompts(ctx, rule, t, io):
    lens, news = [150, 97, 33], [150, 40, 33]
    rules = make_rules(rule, 8, lens, np.random.default_rng(4))
    check_attention(ctx, rule, (8, 2, 64), t, io, lens, news, rules=rules, weight=True, seed=8)


# ------------------------------------------------------------------- prompts

@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
@pytest.mark.parametrize("heads", sorted(HEADS))
def test_prompt_heads_and_types(ctx, heads, t, io):
    check_attention(ctx, heads, HEADS[heads], t, io, [70, 131, 9], [70, 40, 1], seed=11)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 200])
def test_prompt_lengths(ctx, n):
    for t, io in ((F32, F32), (F16, F32), (F16, F16)):
        check_attention(ctx, "prompt length", (8, 2, 64), t, io, [n, n + 70], [n, n], page=32, seed=n)


@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
def test_prompt_long_past(ctx, t, io):
    """Few rows over a long past: the length is split."""
    check_attention(ctx, "long past", (4, 1, 64), t, io, [4200], [40], page=64, seed=2)
    check_attention(ctx, "long past", (4, 1, 128), t, io, [2200, 90], [30, 90], page=64, seed=3, order="hpd", pad=1)


@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
@pytest.mark.parametrize("heads", sorted(HEADS))
def test_prompt_weights(ctx, heads, t, io):
    """The weights that the rows of prompts add, also of chunks after a past."""
    check_attention(ctx, heads, HEADS[heads], t, io, [70, 131, 9], [70, 40, 9], weight=True, seed=18)


@pytest.mark.parametrize("rule", sorted(RULES))
def test_weights_of_a_few_tokens_of_many_heads(ctx, rule):
    """A few tokens of a large group after a long past: many rows, few of them tokens."""
    lens, news = [1500, 300, 70], [5, 3, 5]
    rules = make_rules(rule, 32, lens, np.random.default_rng(19))
    check_attention(ctx, rule, (32, 2, 64), F16, F32, lens, news, page=64, rules=rules, weight=True, seed=19)


def test_bounds_far_above_the_lengths(ctx):
    """max_len and tables for caches far longer than these are: too many scores to keep, so that the weights are formed
    from scores made again, and work groups for lengths that do not come."""
    KH, hd, page, n_seq, per = 1, 8, 65536, 16, 12
    rng = np.random.default_rng(20)
    cache = R.Cache(F16, n_seq, page, KH, hd, rng=rng, weight=True)
    cache.weight[:] = 0.0
    tables = np.full((n_seq, per), -1, np.int32)
    tables[:, 0] = rng.permutation(n_seq)
    lens = [int(n) for n in rng.integers(3, 700, n_seq)]
    for H, new in ((32, 1), (8, 3)):
        q = R.store(rng.standard_normal((n_seq * new, H * hd)), F32)
        news = [new] * n_seq
        for max_len in (per * page, 1 << 30):
            announce(f"bound {max_len} for lengths below 700, {new} new")
            dev = Dev(ctx, cache, tables, lens, news, max_len=max_len)
            got = run_attention(ctx, dev, q, F32, H, {})
            want, bound, w, wb = R.attention(cache, tables, lens, news, q, F32, H, {})
            assert (np.abs(got - want) <= bound).all()
            assert (np.abs(dev.image("weight") - w) <= wb + 2.0 ** -23 * w).all()


@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
def test_prompt_documents_of_many_tiles(ctx, t, io):
    """Documents longer than a tile of keys, so that tiles hold one alone; rows of no document between rows of one,
    in the same block of rows."""
    n = 400
    d = np.zeros((2, n), np.int32)
    d[0, 150:] = 1
    d[0, 333:] = 7
    d[0, [140, 141, 329, 395, 396, 397, 398, 399]] = -1
    d[1, -20:] = -1
    check_attention(ctx, "long documents", (8, 2, 64), t, io, [n, n - 30], [n, 260], page=64, rules=dict(docs=d), seed=15)
    check_attention(ctx, "long documents", (16, 1, 128), t, io, [n, 200], [90, 33], page=64, rules=dict(docs=d, softcap=20.0), weight=True, seed=16)


# ---------------------------------------------------------- what no row sees

def spoil(bad):
    def edit(cache, tables):
        """Values that no row may see: pages outside the tables, and rows past a sequence's end."""
        used = np.zeros((cache.n_pages, cache.page), bool)
        for b, n in enumerate(edit.lens):
            for j in range(n):
                used[tables[b][j // cache.page], j % cache.page] = True
        for p in range(cache.n_pages):
            for o in range(cache.page):
                if not used[p, o]:
                    for h in range(cache.kvh):
                        i = cache.index(p, o, h)
                        cache.k[i] = R.store(np.full(cache.hd, bad), cache.t)
                        cache.v[i] = R.store(np.full(cache.hd, bad), cache.t)
    return edit


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
def test_rows_past_the_end_take_no_part(ctx, bad, t, io):
    for lens, news in (([37, 5, 65], [1, 1, 1]), ([37, 5, 65], [30, 5, 64])):
        e = spoil(bad)
        e.lens = lens
        check_attention(ctx, f"past the end {bad}", (8, 2, 64), t, io, lens, news, edit=e, seed=9)


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
def test_masked_places_may_hold_anything(ctx, bad, t, io):
    """Positions inside the sequence that the rules hide from every row, and ones that only some rows see less:
    a later token's NaN must not reach an earlier row."""
    def edit(cache, tables):
        for j in (3, 17, 18, 40):
            for h in range(cache.kvh):
                i = cache.index(tables[0][j // cache.page], j % cache.page, h)
                cache.k[i], cache.v[i] = R.store(np.full(cache.hd, bad), cache.t), R.store(np.full(cache.hd, -bad), cache.t)

    docs = np.zeros((1, 90), np.int32)
    docs[0, [3, 17, 18, 40]] = -1
    check_attention(ctx, "masked", (8, 2, 64), t, io, [90], [1], rules=dict(docs=docs), edit=edit, weight=True, seed=10)
    check_attention(ctx, "masked", (8, 2, 64), t, io, [90], [90], rules=dict(docs=docs), edit=edit, weight=True, seed=10)


@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
@pytest.mark.parametrize("hd", [64, 128, 200])
def test_a_later_nan_does_not_reach_earlier_rows(ctx, t, io, hd):
    """One prompt whose position 50 holds NaN in v: rows before it are finite and right, rows from it on NaN."""
    H, KH, n = 4, 2, 100
    rng = np.random.default_rng(1)
    cache = R.Cache(t, 8, 16, KH, hd, rng=rng)
    tables = tables_of(rng, [n], 16, 8)
    clean = R.Cache(t, 8, 16, KH, hd, rng=np.random.default_rng(1))
    for h in range(KH):
        cache.v[cache.index(tables[0][50 // 16], 50 % 16, h)[3]] = R.store(np.array([np.nan]), t)[0]
    q = R.store(rng.standard_normal((n, H * hd)), io)
    announce(f"later NaN {NAME[t]}/{NAME[io]} hd={hd}")
    got = run_attention(ctx, Dev(ctx, cache, tables, [n], [n]), q, io, H, {})
    want, bound, _, _ = R.attention(clean, tables, [n], [n], q, io, H, {})
    touched = np.zeros(got.shape, bool)
    touched[50:, :, 3] = True
    assert np.isnan(got[touched]).all()
    assert (np.abs(got - want)[~touched] <= bound[~touched]).all()


@pytest.mark.parametrize("new", [1, 20])
def test_visible_nan_and_inf_come_through(ctx, new):
    """NaN in a seen key makes the row NaN; an infinite value with weight makes its element infinite."""
    H, KH, hd, n = 4, 2, 64, 60
    for t, io in TYPES:
        rng = np.random.default_rng(2)
        cache = R.Cache(t, 8, 16, KH, hd, rng=rng)
        tables = tables_of(rng, [n], 16, 8)
        q = R.store(rng.standard_normal((new, H * hd)), io)
        cache.k[cache.index(tables[0][0], 5, 0)[1]] = R.store(np.array([np.nan]), t)[0]
        cache.v[cache.index(tables[0][0], 7, 1)[2]] = R.store(np.array([np.inf]), t)[0]
        announce(f"visible NaN {NAME[t]}/{NAME[io]} new={new}")
        got = run_attention(ctx, Dev(ctx, cache, tables, [n], [new]), q, io, H, {})
        assert np.isnan(got[:, :2]).all()
        assert np.isposinf(got[:, 2:, 2]).all() and np.isfinite(got[:, 2:, 3:]).all()


def test_bad_pages_hold_nothing(ctx):
    """Page numbers outside the pool: their positions take no part; a sequence of only such pages gives zeros."""
    H, KH, hd = 8, 2, 64
    for t, io in TYPES:
        rng = np.random.default_rng(3)
        cache = R.Cache(t, 12, 16, KH, hd, rng=rng, weight=True)
        tables = np.array([[0, -1, 2, 12], [3, 4, 1 << 30, 5], [-7, -8, 99, 13]], np.int32)
        lens, news = [60, 64, 50], [1, 20, 1]
        q = R.store(rng.standard_normal((sum(news), H * hd)), io)
        announce(f"bad pages {NAME[t]}/{NAME[io]}")
        dev = Dev(ctx, cache, tables, lens, news)
        got = run_attention(ctx, dev, q, io, H, {})
        want, bound, w, wb = R.attention(cache, tables, lens, news, q, io, H, {})
        assert (np.abs(got - want) <= bound).all()
        assert (got[-1] == 0).all()
        assert (np.abs(dev.image("weight") - w) <= wb + 2.0 ** -23 * w).all()


def test_bounds_and_odd_batches(ctx):
    """Empty sequences, sequences without new tokens, rows of no sequence, more rows than positions, lengths past
    the table: each as the header says, and what is not a sequence's row stays as it was."""
    H, KH, hd, page = 4, 2, 64, 16
    for t, io in TYPES:
        rng = np.random.default_rng(4)
        cache = R.Cache(t, 20, page, KH, hd, rng=rng)
        tables = rng.permutation(20)[:16].reshape(4, 4).astype(np.int32)
        lens, news = [0, 40, 30, 3], [1, 0, 2, 5]
        starts = [2, 3, 3, 5, 10]  # rows 0, 1 and 10, 11 belong to no sequence
        q = R.store(rng.standard_normal((12, H * hd)), io)
        announce(f"odd batch {NAME[t]}/{NAME[io]}")
        dev = Dev(ctx, cache, tables, lens, news, starts=starts, n_rows=12)
        got = run_attention(ctx, dev, q, io, H, {})
        want, bound, _, _ = R.attention(cache, tables, lens, news, q, io, H, {}, starts=starts)
        for r in (0, 1, 10, 11):
            assert (got[r] == -3.0).all()
        assert (np.abs(got - want) <= bound)[2:10].all()
        assert (got[2] == 0).all() and (got[5:7] == 0).all()  # no position, and positions below 0
        # lens past the table: as many positions as the table holds
        dev = Dev(ctx, cache, tables, [64, 1000, 64, 64], [1, 1, 1, 1], max_len=2000)
        q = R.store(rng.standard_normal((4, H * hd)), io)
        got = run_attention(ctx, dev, q, io, H, {})
        want, bound, _, _ = R.attention(cache, tables, [64] * 4, [1] * 4, q, io, H, {})
        assert (np.abs(got - want) <= bound).all()
        # without starts, and a max_len below the lengths
        dev = Dev(ctx, cache, tables, [64, 20, 64, 64], max_len=33)
        got = run_attention(ctx, dev, q, io, H, {})
        want, bound, _, _ = R.attention(cache, tables, [33, 20, 33, 33], [1] * 4, q, io, H, {})
        assert (np.abs(got - want) <= bound).all()


def test_empty_calls(ctx):
    cache = R.Cache(F16, 2, 16, 2, 64)
    q = R.store(np.zeros((1, 4 * 64)), F32)
    announce("empty batch")
    dev = Dev(ctx, cache, np.zeros((0, 1)), [], [], starts=[0], n_rows=1, max_len=0)
    assert (run_attention(ctx, dev, q, F32, 4, {}) == -3.0).all()


@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
@pytest.mark.parametrize("new", [1, 33])
def test_large_scores(ctx, t, io, new):
    """Scores in the hundreds: one key takes all; nothing overflows on the way."""
    H, KH, hd, n = 4, 2, 64, 80
    rng = np.random.default_rng(5)
    cache = R.Cache(t, 8, 16, KH, hd, rng=rng)
    tables = tables_of(rng, [n], 16, 8)
    q = R.store(rng.standard_normal((new, H * hd)) * 400.0, io)
    announce(f"large scores {NAME[t]}/{NAME[io]} new={new}")
    got = run_attention(ctx, Dev(ctx, cache, tables, [n], [new]), q, io, H, {})
    want, bound, _, _ = R.attention(cache, tables, [n], [new], q, io, H, {})
    assert np.isfinite(got).all() and (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("t,io", [(F32, F32), (BF16, F32), (BF16, BF16)], ids=["f32-f32", "bf16-f32", "bf16-bf16"])
@pytest.mark.parametrize("new", [1, 40])
def test_scores_far_below_zero(ctx, t, io, new):
    """Equal scores of -3e32: every seen position has the same share, however low the scores are."""
    H, KH, hd, n = 4, 1, 8, 300
    rng = np.random.default_rng(23)
    cache = R.Cache(t, 20, 16, KH, hd, rng=rng, weight=True)
    cache.k[:] = R.store(np.full(cache.k.shape, -1e16), t)
    cache.weight[:] = 0.0
    tables = tables_of(rng, [n], 16, 20)
    q = R.store(np.full((new, H * hd), 1e16), io)
    announce(f"far below zero {NAME[t]}/{NAME[io]} new={new}")
    dev = Dev(ctx, cache, tables, [n], [new])
    got = run_attention(ctx, dev, q, io, H, {})
    v = np.stack([R.load(cache.v, t).reshape(-1)[cache.index(tables[0][j // 16], j % 16, 0)] for j in range(n)])
    eps = 2.0 ** -24 if io == F32 else 2.0 ** -8
    w = np.zeros(n)
    for r in range(new):
        seen = n - new + r + 1
        w[:seen] += H / seen
        want, size = v[:seen].astype(np.float64).mean(0), np.abs(v[:seen]).astype(np.float64).mean(0)
        # shares of exactly 1 to be summed and divided by; the output rounded once
        assert (np.abs(got[r] - want) <= (seen + 4) * 2.0 ** -24 * size + eps * np.abs(want)).all()
    got_w = np.array([dev.image("weight")[tables[0][j // 16], 0, j % 16] for j in range(n)])
    assert (np.abs(got_w - w) <= (new * H + 4) * 2.0 ** -23 * w).all()


def test_f32_rows_beyond_half_range(ctx):
    """F32 rows whose values pass a half's range, and tiny ones, over F16 and BF16 caches."""
    H, KH, hd, n = 4, 2, 64, 80
    for t in (F16, BF16):
        for new in (1, 33):
            for mag, scale in ((1e7, 1e-7), (1e-9, 1e9), (3e33, 1e-33)):
                rng = np.random.default_rng(6)
                cache = R.Cache(t, 8, 16, KH, hd, rng=rng)
                tables = tables_of(rng, [n], 16, 8)
                q = R.store(rng.standard_normal((new, H * hd)) * mag, F32)
                announce(f"range {NAME[t]} {mag} new={new}")
                got = run_attention(ctx, Dev(ctx, cache, tables, [n], [new]), q, F32, H, dict(scale=scale))
                want, bound, _, _ = R.attention(cache, tables, [n], [new], q, F32, H, dict(scale=scale))
                assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()


def test_calls_repeat_to_the_bit(ctx):
    """The same call gives the same bits, with weights, for single tokens and prompts."""
    for lens, news in (([3000, 50], [1, 1]), ([300, 90], [300, 20])):
        outs = []
        for _ in range(3):
            dev, got = check_attention(ctx, "repeat", (8, 2, 64), F16, F32, lens, news, weight=True, seed=12)
            outs.append((got, dev.image("weight")))
        for o in outs[1:]:
            assert np.array_equal(o[0], outs[0][0]) and np.array_equal(o[1], outs[0][1])


def test_offsets_past_32_bits(ctx):
    """A pool of more than 2^32 bytes and elements: the last pages are read and written as the first."""
    H, KH, hd, page = 4, 2, 64, 64
    pos_stride, row = KH * 2112, 2112  # a padded pool
    n_pages = (1 << 32) // (page * pos_stride) + 40
    bytes_ = n_pages * page * pos_stride * 2
    announce(f"pool of {bytes_ / 2**30:.1f} GiB each")
    k, v = ctx.alloc(bytes_), ctx.alloc(bytes_)
    _KEEP.extend([k, v])
    rng = np.random.default_rng(13)
    n, new = 200, 200
    tables = np.array([[n_pages - 1, 3, n_pages - 7, n_pages - 2]], np.int32)
    bufs = [up(ctx, tables), up(ctx, np.array([n], np.int32)), up(ctx, np.array([0, new], np.int32))]
    kv = mcpm.PagedKV(F16, n_pages, page, KH, hd, page * pos_stride, pos_stride, row, k.ptr, v.ptr, None)
    batch = mcpm.PagedBatch(1, new, new, n, 4, *[b.ptr for b in bufs])
    kn, vn = (R.store(rng.standard_normal((new, KH * hd)), F16) for _ in range(2))
    mcpm.check(ctx.lib.mcpm_paged_append(ctx.h, C.byref(kv), C.byref(batch), F16, up(ctx, kn).ptr, up(ctx, vn).ptr, KH * hd,
                                         None, 0, 0, 0.0))
    small = R.Cache(F16, 4, page, KH, hd)
    for j in range(n):
        for h in range(KH):
            small.k[small.index(j // page, j % page, h)] = kn[j, h * hd:(h + 1) * hd]
            small.v[small.index(j // page, j % page, h)] = vn[j, h * hd:(h + 1) * hd]
    q = R.store(rng.standard_normal((new, H * hd)), F16)
    od = up(ctx, q)
    for rows in (new, 1):
        batch = mcpm.PagedBatch(1, rows, rows, n, 4, bufs[0].ptr, bufs[1].ptr, up(ctx, np.array([0, rows], np.int32)).ptr)
        mcpm.check(ctx.lib.mcpm_paged_attention(ctx.h, od.ptr, H * hd, up(ctx, q).ptr, H * hd, F16, H, C.byref(kv),
                                                C.byref(batch), None))
        got = R.load(ctx.download(od, q.dtype, q.shape), F16).reshape(-1, H, hd)[:rows]
        want, bound, _, _ = R.attention(small, np.arange(4).reshape(1, 4), [n], [rows], q[:rows], F16, H, {})
        assert (np.abs(got - want) <= bound).all()


# -------------------------------------------------------------------- append

@pytest.mark.parametrize("t,io", TYPES, ids=IDS)
@pytest.mark.parametrize("heads", ["gqa4", "gqa8", "gqa5_80", "g20_8", "mqa256"])
@pytest.mark.parametrize("base", [0.0, 10000.0, 5e6])
def test_append(ctx, t, io, heads, base):
    """k rotated and v as it is at their positions, q in place; everything else as it was."""
    H, KH, hd = HEADS[heads]
    page, lens, news = 16, [40, 100000, 7, 1], [3, 20, 7, 1]
    rng = np.random.default_rng(14)
    cache = R.Cache(t, 60, page, KH, hd, "phd", 1, weight=True, rng=rng)
    cache.weight[:] = 1.0
    per = -(-max(lens) // page)
    tables = np.full((4, per), 59, np.int32)
    pages = iter(rng.permutation(58))
    for b, n in enumerate(lens):
        for j in range(n - news[b], n):
            if tables[b][j // page] == 59:
                tables[b][j // page] = next(pages)
    rows = sum(news)
    x = {n: R.store(rng.standard_normal((rows + 2, w * hd)) * 2, io) for n, w in (("k", KH), ("v", KH), ("q", H))}
    announce(f"append {heads} {NAME[t]}/{NAME[io]} base={base}")
    dev = Dev(ctx, cache, tables, lens, news, n_rows=rows + 2)
    qd = up(ctx, x["q"])
    mcpm.check(ctx.lib.mcpm_paged_append(ctx.h, C.byref(dev.kv), C.byref(dev.batch), io, up(ctx, x["k"]).ptr,
                                         up(ctx, x["v"]).ptr, KH * hd, qd.ptr, H * hd, H, base))
    got = {"k": R.load(dev.image("k"), t), "v": R.load(dev.image("v"), t), "q": R.load(ctx.download(qd, x["q"].dtype, x["q"].shape), io)}
    want = {"k": R.load(cache.k, t), "v": R.load(cache.v, t), "q": R.load(x["q"], io)}
    tol = {n: np.zeros_like(w) for n, w in want.items()}
    weight = cache.weight.copy()
    at = R.spans(lens, news)
    # a rotated element: two products and a sum in 32 bits, cos and sin rounded once each
    eps = 4 * 2.0 ** -24
    for b in range(4):
        for r in range(news[b]):
            pos, row = lens[b] - news[b] + r, at[b] + r
            kx = R.load(x["k"], io)[row].reshape(KH, hd)
            qx = R.load(x["q"], io)[row].reshape(H, hd)
            ky, qy = (R.rope(kx, pos, base), R.rope(qx, pos, base)) if base else (kx, qx)
            mag = lambda a: np.repeat(np.abs(a[:, 0::2]) + np.abs(a[:, 1::2]), 2, axis=1)  # noqa: E731
            for h in range(KH):
                i = cache.index(tables[b][pos // page], pos % page, h)
                want["k"][i], want["v"][i] = ky[h], R.load(x["v"], io)[row].reshape(KH, hd)[h]
                tol["k"][i] = (eps * mag(kx)[h] if base else 0) + R.HALF[t] * 1.01 * np.abs(ky[h]) + 2.0 ** -25
                tol["v"][i] = (R.HALF[t] * np.abs(want["v"][i]) + 2.0 ** -25) if t != io else 0
                weight[tables[b][pos // page], h, pos % page] = 0.0
            if base:
                want["q"][row] = qy.ravel()
                tol["q"][row] = (eps * mag(qx) + R.HALF[io] * 1.01 * np.abs(qy)).ravel() + 2.0 ** -25
    for n in want:
        bad = np.abs(got[n] - want[n]) > tol[n]
        assert not bad.any(), (n, bad.sum(), np.abs(got[n] - want[n])[bad].max())
    assert np.array_equal(dev.image("weight"), weight)


def test_append_bad_pages_and_negative_positions(ctx):
    """Nothing is stored for a page outside the pool or a position below 0; q of such a page is still rotated."""
    H, KH, hd, page = 4, 2, 64, 16
    rng = np.random.default_rng(15)
    cache = R.Cache(F16, 6, page, KH, hd, rng=rng)
    tables = np.array([[0, 6], [-1, 2], [3, 4]], np.int32)
    lens, news = [18, 4, 2], [3, 2, 4]  # positions 15..17, 2..3, -2..1
    k, v = (R.store(rng.standard_normal((9, KH * hd)), F32) for _ in range(2))
    q = R.store(rng.standard_normal((9, H * hd)), F32)
    announce("append bad pages")
    dev = Dev(ctx, cache, tables, lens, news)
    qd = up(ctx, q)
    mcpm.check(ctx.lib.mcpm_paged_append(ctx.h, C.byref(dev.kv), C.byref(dev.batch), F32, up(ctx, k).ptr, up(ctx, v).ptr,
                                         KH * hd, qd.ptr, H * hd, H, 10000.0))
    got = R.load(dev.image("v"), F16)
    want = R.load(cache.v, F16)
    for row, (p, o) in {0: (0, 15), 7: (3, 0), 8: (3, 1)}.items():
        for h in range(KH):
            want[cache.index(p, o, h)] = v[row, h * hd:(h + 1) * hd].astype(np.float16)
    assert np.array_equal(got, want)
    gq = ctx.download(qd, np.float32, q.shape).astype(np.float64)
    pos = [15, 16, 17, 2, 3, None, None, 0, 1]
    for r, p in enumerate(pos):
        w = R.rope(q[r].reshape(H, hd).astype(np.float64), p, 10000.0).ravel() if p is not None else q[r]
        assert np.abs(gq[r] - w).max() <= 2.0 ** -20


# --------------------------------------------------------------------- evict

def run_evict(ctx, cache, tables, lens, dst, budget, first, recent, max_len=None):
    dev = Dev(ctx, cache, tables, lens, max_len=max_len)
    n, KH = len(lens), cache.kvh
    kept, dl = up(ctx, np.full((n, KH, budget), -9, np.int32)), up(ctx, np.full(n, -9, np.int32))
    mcpm.check(ctx.lib.mcpm_paged_evict(ctx.h, C.byref(dev.kv), C.byref(dev.batch), budget, first, recent, up(ctx, dst).ptr,
                                        dst.shape[1], kept.ptr, dl.ptr))
    return dev, ctx.download(kept, np.int32, (n, KH, budget)), ctx.download(dl, np.int32, n)


def check_evict(ctx, name, t, KH, hd, page, lens, budget, first, recent, weights, order="phd", pad=0):
    rng = np.random.default_rng(16)
    per, pd = max(1, max(-(-n // page) for n in lens)), -(-budget // page)
    cache = R.Cache(t, (per + pd) * len(lens) + 1, page, KH, hd, order, pad, True, rng)
    perm = rng.permutation(cache.n_pages)
    tables = perm[:per * len(lens)].reshape(len(lens), per).astype(np.int32)
    dst = perm[per * len(lens):(per + pd) * len(lens)].reshape(len(lens), pd).astype(np.int32)
    cache.weight[:] = weights(rng, cache.weight.shape)
    announce(f"evict {name} {NAME[t]} {KH}x{hd} page={page} lens={lens} budget={budget} first={first} recent={recent}")
    dev, kept, dl = run_evict(ctx, cache, tables, lens, dst, budget, first, recent)
    want_k, want_v, want_w = cache.k.copy(), cache.v.copy(), cache.weight.copy()
    for b, n in enumerate(lens):
        assert dl[b] == min(n, budget)
        for h in range(KH):
            w = np.array([cache.weight[tables[b][j // page], h, j % page] for j in range(n)], np.float32)
            keep = R.evict_kept(w, n, budget, first, recent)
            assert np.array_equal(kept[b, h, :len(keep)], keep)
            assert (kept[b, h, len(keep):] == -1).all()
            for i, j in enumerate(keep):
                s, d = (tables[b][j // page], j % page), (dst[b][i // page], i % page)
                want_k[cache.index(*d, h)], want_v[cache.index(*d, h)] = cache.k[cache.index(*s, h)], cache.v[cache.index(*s, h)]
                want_w[d[0], h, d[1]] = cache.weight[s[0], h, s[1]]
    for n, w in (("k", want_k), ("v", want_v), ("weight", want_w)):
        g = dev.image(n)
        assert np.array_equal(g.view(np.uint8), w.view(np.uint8)), n


def heavy(rng, shape):
    return rng.exponential(size=shape).astype(np.float32) ** 3


def ties(rng, shape):
    return rng.integers(0, 3, shape).astype(np.float32) * 0.5


def odd_values(rng, shape):
    return rng.choice(np.array([0.0, -0.0, 1.0, -1.0, np.inf, -np.inf, np.nan, 1e-40, -1e-40, 3e38], np.float32), shape)


@pytest.mark.parametrize("weights", [heavy, ties, odd_values])
@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_evict(ctx, t, weights):
    check_evict(ctx, weights.__name__, t, 2, 64, 16, [200, 31, 32, 33, 1], 32, 2, 9, weights)


@pytest.mark.parametrize("budget,first,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 0, 64), (64, 64, 0), (64, 10, 54), (63, 0, 0),
                                                 (100, 4, 30)])
def test_evict_budgets(ctx, budget, first, recent):
    check_evict(ctx, "budget", F16, 3, 40, 8, [300, 65, 64, 0], budget, first, recent, heavy, order="hpd", pad=1)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 2049, 4300, 5000, 16500, 20001, 65700, 131500])
def test_evict_lengths(ctx, n):
    check_evict(ctx, "length", F16, 1, 8, 64, [n], n // 3, 4, 100, ties)
    check_evict(ctx, "length", F16, 1, 8, 64, [n], n // 3, 4, 100, heavy)


def test_evict_bad_pages(ctx):
    """A page outside the pool weighs nothing and is not copied; a destination outside it is not written."""
    rng = np.random.default_rng(17)
    cache = R.Cache(F16, 8, 16, 1, 64, weight=True, rng=rng)
    cache.weight[:] = rng.random(cache.weight.shape) + 0.5
    tables, dst = np.array([[0, 1 << 20, 2, 3]], np.int32), np.array([[5, -1]], np.int32)
    announce("evict bad pages")
    dev, kept, dl = run_evict(ctx, cache, tables, [64], dst, 32, 1, 1)
    w = np.array([cache.weight[tables[0][j // 16], 0, j % 16] if j // 16 != 1 else np.nan for j in range(64)], np.float32)
    keep = R.evict_kept(w, 64, 32, 1, 1)
    assert np.array_equal(kept[0, 0], keep)
    want = cache.k.copy()
    for i, j in enumerate(keep[:16]):
        if j // 16 != 1:
            want[cache.index(5, i, 0)] = cache.k[cache.index(tables[0][j // 16], j % 16, 0)]
    assert np.array_equal(dev.image("k"), want)


# -------------------------------------------------------------------- logits

def check_logits(ctx, name, n, V, stride, hist, rep, pres, freq, bias, allowed, x):
    """hist: a list of id lists; bias: a list of (id, value) lists; each of the rules may be None."""
    announce(f"logits {name} n={n} vocab={V}")
    img = np.full((n, stride), 77.0, np.float32)
    img[:, :V] = x
    ld = up(ctx, img)
    flat = lambda ls, dt: np.array([i for l in ls for i in l], dt)  # noqa: E731
    cat = lambda ls: np.cumsum([0] + [len(l) for l in ls]).astype(np.int32)  # noqa: E731
    words = (V + 31) // 32 + 1
    bits = None
    if allowed is not None:
        full = np.zeros((n, words * 32), bool)
        full[:, :V] = allowed
        bits = np.packbits(full, axis=1, bitorder="little").view(np.uint32)
    arr = [None if a is None else up(ctx, np.asarray(a, np.float32)) for a in (rep, pres, freq)]
    r = mcpm.LogitRules(n_seq=n, vocab=V, stride=stride, repetition=ptr(arr[0]), presence=ptr(arr[1]), frequency=ptr(arr[2]),
                        allowed=ptr(up(ctx, bits)), allowed_stride=words)
    if hist is not None:
        r.history, r.history_starts = up(ctx, flat(hist, np.int32)).ptr, up(ctx, cat(hist)).ptr
    if bias is not None:
        r.bias_ids, r.bias = up(ctx, flat([[i for i, _ in l] for l in bias], np.int32)).ptr, up(ctx, flat([[v for _, v in l] for l in bias], np.float32)).ptr
        r.bias_starts = up(ctx, cat(bias)).ptr
    mcpm.check(ctx.lib.mcpm_process_logits(ctx.h, ld.ptr, C.byref(r)))
    got = ctx.download(ld, np.float32, img.shape)
    assert (got[:, V:] == 77.0).all()
    for b in range(n):
        f = lambda a, d: d if a is None else float(np.float32(a[b]))  # noqa: E731
        h = hist[b] if hist is not None else []
        want = R.logits(img[b, :V], h, f(rep, 1.0), f(pres, 0.0), f(freq, 0.0),
                        [(i, float(np.float32(v))) for i, v in bias[b]] if bias is not None else [],
                        allowed[b] if allowed is not None else None)
        # a quotient or product, freq * c, two sums and the bias: a rounding of each
        c = np.bincount([i for i in h if 0 <= i < V], minlength=V)
        pen = np.abs(img[b, :V]) * max(f(rep, 1.0), 1 / f(rep, 1.0)) + f(freq, 0.0) * c + f(pres, 0.0)
        big = max([abs(v) for _, v in bias[b]], default=0) if bias is not None else 0
        fin = np.isfinite(want)
        assert np.array_equal(np.isnan(got[b, :V]), np.isnan(want))
        assert np.array_equal(got[b, :V][~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)])
        with np.errstate(invalid="ignore"):
            assert (np.abs(got[b, :V] - want)[fin] <= (6 * 2.0 ** -24 * (pen + big))[fin]).all()
        same = (c == 0) & ~np.isin(np.arange(V), [i for i, _ in bias[b]] if bias is not None else []) & (allowed[b] if allowed is not None else True)
        assert np.array_equal(got[b, :V][same].view(np.uint32), img[b, :V][same].view(np.uint32))


@pytest.mark.parametrize("V", [1, 31, 32, 33, 1000, 4095, 4096, 4097, 130560, 130561])
@pytest.mark.parametrize("n", [1, 5])
def test_logits(ctx, n, V):
    rng = np.random.default_rng(V + n)
    hist = [rng.integers(-2, V + 2, k).tolist() for k in rng.integers(0, 700, n)]
    hist[0] = [V - 1, 0, V - 1, V // 2] * 50 + [-5, V, 2 ** 31 - 1, -2 ** 31]
    bias = [[(int(i), float(v)) for i, v in zip(rng.integers(-1, V + 1, k), rng.standard_normal(k))] for k in rng.integers(0, 60, n)]
    bias[-1] = [(0, 5.0), (0, -2.5), (V - 1, 1.0), (0, 0.25)]
    check_logits(ctx, "all", n, V, V + 3, hist, rng.uniform(1, 1.5, n), rng.uniform(-1, 1, n), rng.uniform(0, 0.5, n), bias,
                 rng.random((n, V)) < 0.5, rng.standard_normal((n, V)) * 3)


@pytest.mark.parametrize("which", ["none", "history", "frequency", "bias", "allowed", "nothing_allowed"])
def test_logits_each_rule_alone(ctx, which):
    rng = np.random.default_rng(20)
    n, V = 3, 5000
    hist = [rng.integers(0, V, 300).tolist(), [], [7]] if which in ("history", "frequency") else None
    bias = [[], [(4999, 3.0)], [(i, 1.0) for i in range(50)]] if which == "bias" else None
    allowed = {"allowed": rng.random((n, V)) < 0.1, "nothing_allowed": np.zeros((n, V), bool)}.get(which)
    check_logits(ctx, which, n, V, V, hist, rng.uniform(1, 2, n) if which == "history" else None, None,
                 rng.uniform(0, 1, n) if which == "frequency" else None, bias, allowed, rng.standard_normal((n, V)))


def test_logits_odd_values(ctx):
    """Infinities and NaN in the logits, under each rule; a masked one is -inf whatever it was."""
    V = 400
    x = np.resize(np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-40, 3e38, -3e38], np.float32), (1, V))
    check_logits(ctx, "odd values", 1, V, V, [list(range(0, V, 2)) * 3], [1.25], [0.5], [0.125],
                 [[(i, 2.0) for i in range(100)]], (np.arange(V) % 7 != 3)[None], x)


# ----------------------------------------------------------- a run of them all

def test_serving_step(ctx):
    """Three conversations: prompts appended and attended, single tokens with weights, an eviction to shorter
    caches, more tokens on them; then the logits' rules and the sampler.  Each step against the definition,
    on the state that the steps before it left on the device."""
    H, KH, hd, page, t, io = 8, 2, 64, 16, F16, F32
    rng = np.random.default_rng(21)
    cache = R.Cache(t, 64, page, KH, hd, weight=True, rng=rng, fill=0.0)
    cache.weight[:] = 5.0  # a page's earlier owner left something
    free = iter(rng.permutation(64))
    tables = np.array([[next(free) for _ in range(8)] for _ in range(3)], np.int32)
    lens = [0, 0, 0]
    dev = Dev(ctx, cache, tables, [0, 0, 0], [1, 1, 1])

    def step(news, rules):
        rows = sum(news)
        for b in range(3):
            lens[b] += news[b]
        d = Dev.__new__(Dev)
        d.ctx, d.cache, d.k, d.v, d.w = ctx, cache, dev.k, dev.v, dev.w
        bufs = [up(ctx, tables), up(ctx, np.array(lens, np.int32)), up(ctx, np.array(R.spans(lens, news), np.int32))]
        d.kv, d.batch = dev.kv, mcpm.PagedBatch(3, rows, max(news), max(lens), tables.shape[1], *[b.ptr for b in bufs])
        q, k, v = (R.store(rng.standard_normal((rows, w * hd)), io) for w in (H, KH, KH))
        qd = up(ctx, q)
        mcpm.check(ctx.lib.mcpm_paged_append(ctx.h, C.byref(d.kv), C.byref(d.batch), io, up(ctx, k).ptr, up(ctx, v).ptr,
                                             KH * hd, qd.ptr, H * hd, H, 10000.0))
        cache.k, cache.v, cache.weight = d.image("k"), d.image("v"), d.image("weight")
        q = ctx.download(qd, np.float32, q.shape)
        got = run_attention(ctx, d, q, io, H, rules)
        want, bound, w, wb = R.attention(cache, tables, lens, news, q, io, H, rules)
        assert (np.abs(got - want) <= bound).all()
        assert (np.abs(d.image("weight") - cache.weight - w) <= wb + 2.0 ** -22 * (w + cache.weight)).all()
        cache.weight = d.image("weight")
        return got

    announce("serving step")
    step([70, 33, 90], dict(softcap=30.0))
    for _ in range(3):
        step([1, 1, 1], {})
    n_before = list(lens)
    dst = np.array([[next(free) for _ in range(8)] for _ in range(3)], np.int32)
    kept, dl = ctx.zeros(3 * KH * 48 * 4), ctx.zeros(12)
    _KEEP.extend([kept, dl])
    batch = mcpm.PagedBatch(3, 0, 0, max(lens), 8, up(ctx, tables).ptr, up(ctx, np.array(lens, np.int32)).ptr, None)
    mcpm.check(ctx.lib.mcpm_paged_evict(ctx.h, C.byref(dev.kv), C.byref(batch), 48, 4, 16, up(ctx, dst).ptr, 8, kept.ptr, dl.ptr))
    got = ctx.download(kept, np.int32, (3, KH, 48))
    for b in range(3):
        for h in range(KH):
            w = np.array([cache.weight[tables[b][j // page], h, j % page] for j in range(n_before[b])], np.float32)
            keep = R.evict_kept(w, n_before[b], 48, 4, 16)
            assert np.array_equal(got[b, h, :len(keep)], keep)
    tables = dst
    lens = ctx.download(dl, np.int32, 3).tolist()
    assert lens == [min(n, 48) for n in n_before]
    cache.k, cache.v, cache.weight = (ctx.download(b, a.dtype, a.shape) for b, a in ((dev.k, cache.k), (dev.v, cache.v), (dev.w, cache.weight)))
    out = step([1, 2, 1], {})
    step([1, 1, 1], dict(window=20))

    V = 5000
    x = (rng.standard_normal((1, V)) * 2).astype(np.float32) + out.ravel()[0].astype(np.float32)
    ld, tok = up(ctx, x), ctx.zeros(4)
    _KEEP.append(tok)
    top = np.argsort(-x[0])[:40]
    allowed = np.ones(((V + 31) // 32) * 32, bool)
    allowed[top[:5]] = False
    r = mcpm.LogitRules(n_seq=1, vocab=V, stride=V, history=up(ctx, top[5:10].astype(np.int32)).ptr,
                        history_starts=up(ctx, np.array([0, 5], np.int32)).ptr, presence=up(ctx, np.array([50.0], np.float32)).ptr,
                        allowed=up(ctx, np.packbits(allowed, bitorder="little")).ptr, allowed_stride=(V + 31) // 32)
    mcpm.check(ctx.lib.mcpm_process_logits(ctx.h, ld.ptr, C.byref(r)))
    mcpm.check(ctx.lib.mcpm_argmax(ctx.h, ld.ptr, V, tok.ptr))
    assert ctx.download(tok, np.int32, 1)[0] == top[10]
    host = ctx.download(ld, np.float32, V)
    for draw in (0.0, 0.3, 0.77, 0.999):
        mcpm.check(ctx.lib.mcpm_sample_device(ctx.h, ld.ptr, V, 0.7, 0.9, draw, tok.ptr))
        got = int(ctx.download(tok, np.int32, 1)[0])
        assert got not in top[:10]
        p = np.exp((host.astype(np.float64) - host.max()) / np.float64(np.float32(0.7)))
        assert p[got] > 0


def test_two_contexts(ctx):
    """Calls of two contexts between each other's do not share scratch."""
    other = mcpm.Context(0)
    try:
        H, KH, hd = 8, 2, 64
        rng = np.random.default_rng(22)
        made = []
        for c, n in ((ctx, 3000), (other, 2000)):
            cache = R.Cache(F16, 64, 64, KH, hd, weight=True, rng=rng)
            tables = tables_of(rng, [n], 64, 64)
            q = R.store(rng.standard_normal((1, H * hd)), F32)
            dev = Dev(c, cache, tables, [n], [1])
            made.append((c, cache, tables, n, q, dev, up(c, q), up(c, q * 0)))
        announce("two contexts")
        for _ in range(4):
            for c, cache, tables, n, q, dev, qd, od in made:
                mcpm.check(c.lib.mcpm_paged_attention(c.h, od.ptr, H * hd, qd.ptr, H * hd, F32, H, C.byref(dev.kv), C.byref(dev.batch), None))
        for c, cache, tables, n, q, dev, qd, od in made:
            got = c.download(od, np.float32, q.shape).reshape(1, H, hd)
            want, bound, _, _ = R.attention(cache, tables, [n], [1], q, F32, H, {})
            assert (np.abs(got - want) <= bound).all()
        other.sync()
        _KEEP.clear()
        made.clear()
    finally:
        other.close()
