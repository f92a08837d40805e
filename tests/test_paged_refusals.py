"""What the operators over many sequences refuse, and how their kernels map positions to memory: host code only.
The entry points check every argument before they look at the context, so a null context shows that the
arguments passed."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import mcpm
from conftest import ROOT

A = 1 << 20  # an aligned address that no check reads


def kv(**over):
    d = dict(type=mcpm.TYPE_F16, n_pages=8, page_size=16, n_kv_heads=2, head_dim=64, page_stride=16 * 128, pos_stride=128,
             head_stride=64, k=A, v=A, weight=None)
    return mcpm.PagedKV(**{**d, **over})


def batch(**over):
    d = dict(n_seq=2, n_rows=2, max_new=1, max_len=32, max_pages=2, pages=A, lens=A, starts=A)
    return mcpm.PagedBatch(**{**d, **over})


def attention(lib, kv_=None, batch_=None, rules=None, out=A, out_stride=512, q=A, q_stride=512, io=mcpm.TYPE_F32, heads=8):
    return lib.mcpm_paged_attention(None, out, out_stride, q, q_stride, io, heads, kv_ or kv(), batch_ or batch(), rules)


def append(lib, kv_=None, batch_=None, io=mcpm.TYPE_F32, k=A, v=A, stride=128, q=A, q_stride=512, heads=8, base=1e4):
    return lib.mcpm_paged_append(None, kv_ or kv(), batch_ or batch(), io, k, v, stride, q, q_stride, heads, base)


def evict(lib, kv_=None, batch_=None, budget=16, first=1, recent=4, dst=A + 64, max_dst=1, kept=A, lens=A + 128):
    return lib.mcpm_paged_evict(None, kv_ or kv(weight=A), batch_ or batch(), budget, first, recent, dst, max_dst, kept, lens)


def logits(lib, x=A, **over):
    d = dict(n_seq=2, vocab=1000, stride=1000)
    return lib.mcpm_process_logits(None, x, mcpm.LogitRules(**{**d, **over}))


def refused(lib, rc, code, words):
    msg = lib.mcpm_last_error().decode()
    assert rc == code and words in msg, (rc, msg)


def accepted(lib, rc):
    refused(lib, rc, mcpm.ERR_ARG, "null context")


def test_values_past_the_range_are_refused(lib):
    for rules in (mcpm.AttnRules(scale=2e38), mcpm.AttnRules(scale=-2e38), mcpm.AttnRules(softcap=2e38),
                  mcpm.AttnRules(scale=1e10, softcap=1e-30), mcpm.AttnRules(scale=float("nan"))):
        refused(lib, attention(lib, rules=rules), mcpm.ERR_ARG, "1e38")
    accepted(lib, attention(lib, rules=mcpm.AttnRules(scale=1e37, softcap=1e38)))
    many = batch(n_rows=1 << 30, max_new=1 << 30)
    refused(lib, attention(lib, batch_=many), mcpm.ERR_ARG, "max_new * n_heads")


def test_sound_calls_get_as_far_as_the_context(lib):
    for rc in (attention(lib), append(lib), evict(lib), logits(lib)):
        accepted(lib, rc)
    accepted(lib, attention(lib, rules=mcpm.AttnRules(softcap=30.0, window=5, docs=A, docs_stride=32)))
    accepted(lib, attention(lib, io=mcpm.TYPE_F16))
    accepted(lib, attention(lib, batch_=batch(n_seq=0, pages=None, lens=None, n_rows=0)))
    accepted(lib, attention(lib, batch_=batch(starts=None)))
    accepted(lib, append(lib, q=None, heads=0, base=0.0))
    accepted(lib, evict(lib, budget=16, first=0, recent=16))


CACHES = [
    (dict(type=mcpm.TYPE_Q8_0), mcpm.ERR_UNSUPPORTED, "cache type"),
    (dict(k=None), mcpm.ERR_ARG, "k and v"),
    (dict(v=A + 8), mcpm.ERR_ARG, "16-byte aligned"),
    (dict(page_size=24), mcpm.ERR_ARG, "power of two"),
    (dict(page_size=0), mcpm.ERR_ARG, "power of two"),
    (dict(page_size=1 << 17), mcpm.ERR_ARG, "power of two"),
    (dict(n_pages=0), mcpm.ERR_ARG, "n_pages"),
    (dict(head_dim=68), mcpm.ERR_ARG, "multiple of 8"),
    (dict(head_dim=264), mcpm.ERR_ARG, "up to 256"),
    (dict(head_dim=0), mcpm.ERR_ARG, "head_dim"),
    (dict(n_kv_heads=0), mcpm.ERR_ARG, "n_kv_heads"),
    (dict(pos_stride=132), mcpm.ERR_ARG, "strides"),
    (dict(head_stride=56), mcpm.ERR_ARG, "strides"),
    (dict(page_stride=-128), mcpm.ERR_ARG, "strides"),
    (dict(pos_stride=1 << 31), mcpm.ERR_ARG, "less than 2^31"),
    (dict(head_stride=1 << 31), mcpm.ERR_ARG, "less than 2^31"),
]


@pytest.mark.parametrize("over,code,words", CACHES)
def test_caches(lib, over, code, words):
    refused(lib, attention(lib, kv_=kv(**over)), code, words)
    refused(lib, append(lib, kv_=kv(**over)), code, words)
    refused(lib, evict(lib, kv_=kv(weight=A, **over)), code, words)


BATCHES = [
    (dict(n_seq=-1), "n_seq"),
    (dict(n_seq=70000), "n_seq"),
    (dict(max_len=-1), "max_len"),
    (dict(max_len=(1 << 30) + 1), "max_len"),
    (dict(max_pages=-1), "batch"),
    (dict(lens=None), "lens"),
    (dict(pages=None), "pages"),
]


@pytest.mark.parametrize("over,words", BATCHES)
def test_batches(lib, over, words):
    for rc in (attention(lib, batch_=batch(**over)), append(lib, batch_=batch(**over)), evict(lib, batch_=batch(**over))):
        refused(lib, rc, mcpm.ERR_ARG, words)


def test_rows(lib):
    for f in (attention, append):
        refused(lib, f(lib, batch_=batch(n_rows=-1)), mcpm.ERR_ARG, "rows")
        refused(lib, f(lib, batch_=batch(max_new=-1)), mcpm.ERR_ARG, "rows")
        refused(lib, f(lib, batch_=batch(starts=None, n_rows=1)), mcpm.ERR_ARG, "without starts")
        refused(lib, f(lib, q=A + 4), mcpm.ERR_ARG, "q rows")
        refused(lib, f(lib, q_stride=511), mcpm.ERR_ARG, "q rows")
        refused(lib, f(lib, q_stride=514), mcpm.ERR_ARG, "q rows")
        refused(lib, f(lib, io=mcpm.TYPE_BF16), mcpm.ERR_UNSUPPORTED, "F32 or of the cache's type")
        refused(lib, f(lib, io=7), mcpm.ERR_UNSUPPORTED, "F32 or of the cache's type")
        refused(lib, f(lib, kv_=kv(type=mcpm.TYPE_F32), io=mcpm.TYPE_F16), mcpm.ERR_UNSUPPORTED, "F32 or")
    refused(lib, attention(lib, q=None), mcpm.ERR_ARG, "q rows")
    refused(lib, attention(lib, out=None), mcpm.ERR_ARG, "out rows")
    refused(lib, attention(lib, out_stride=504), mcpm.ERR_ARG, "out rows")
    refused(lib, attention(lib, heads=7), mcpm.ERR_ARG, "n_heads")
    refused(lib, attention(lib, heads=0), mcpm.ERR_ARG, "n_heads")
    refused(lib, append(lib, k=None), mcpm.ERR_ARG, "k rows")
    refused(lib, append(lib, v=A + 2), mcpm.ERR_ARG, "v rows")
    refused(lib, append(lib, stride=120), mcpm.ERR_ARG, "k rows")
    refused(lib, append(lib, heads=0), mcpm.ERR_ARG, "n_heads")
    for base in (-1.0, float("nan"), float("inf")):
        refused(lib, append(lib, base=base), mcpm.ERR_ARG, "rope_base")


def test_rules(lib):
    for over in (dict(scale=float("nan")), dict(scale=float("inf")), dict(softcap=-1.0), dict(softcap=float("inf")),
                 dict(softcap=float("nan")), dict(window=-1)):
        refused(lib, attention(lib, rules=mcpm.AttnRules(**over)), mcpm.ERR_ARG, "softcap and window")
    refused(lib, attention(lib, rules=mcpm.AttnRules(docs=A, docs_stride=31)), mcpm.ERR_ARG, "docs_stride")


def test_evictions(lib):
    for over in (dict(budget=0), dict(first=-1), dict(recent=-1), dict(first=13, recent=4), dict(first=2 ** 31 - 1, recent=2 ** 31 - 1)):
        refused(lib, evict(lib, **over), mcpm.ERR_ARG, "budget")
    refused(lib, evict(lib, budget=17), mcpm.ERR_ARG, "less than budget")
    refused(lib, evict(lib, max_dst=0), mcpm.ERR_ARG, "less than budget")
    refused(lib, evict(lib, kv_=kv()), mcpm.ERR_ARG, "null weight")
    refused(lib, evict(lib, kv_=kv(weight=A + 4)), mcpm.ERR_ARG, "weight must be 16-byte aligned")
    refused(lib, attention(lib, kv_=kv(weight=A + 8)), mcpm.ERR_ARG, "weight must be 16-byte aligned")
    for over in (dict(dst=None), dict(kept=None), dict(lens=None)):
        refused(lib, evict(lib, **over), mcpm.ERR_ARG, "null weight, dst_pages")
    refused(lib, evict(lib, dst=A), mcpm.ERR_ARG, "memory of their own")
    refused(lib, evict(lib, lens=A), mcpm.ERR_ARG, "memory of their own")


def test_logit_rules(lib):
    for over in (dict(n_seq=-1), dict(n_seq=70000), dict(vocab=0), dict(vocab=2 ** 31 - 1, stride=1 << 40), dict(stride=999)):
        refused(lib, logits(lib, **over), mcpm.ERR_ARG, "vocab")
    refused(lib, logits(lib, x=None), mcpm.ERR_ARG, "null")
    for over in (dict(history=A), dict(history_starts=A), dict(bias=A), dict(bias=A, bias_ids=A), dict(bias_starts=A)):
        refused(lib, logits(lib, **over), mcpm.ERR_ARG, "come together")
    refused(lib, logits(lib, allowed=A, allowed_stride=31), mcpm.ERR_ARG, "allowed_stride")
    accepted(lib, logits(lib, allowed=A, allowed_stride=32, history=A, history_starts=A))


def test_null_descriptors(lib):
    assert lib.mcpm_paged_attention(None, A, 512, A, 512, 0, 8, None, batch(), None) == mcpm.ERR_ARG
    assert lib.mcpm_paged_attention(None, A, 512, A, 512, 0, 8, kv(), None, None) == mcpm.ERR_ARG
    assert lib.mcpm_process_logits(None, A, None) == mcpm.ERR_ARG


def test_positions_in_memory():
    """Lengths, rows, pages and element offsets as the kernels form them, run on the host: bad page numbers,
    lengths past every bound, starts out of order, offsets past 32 bits."""
    prog = os.path.join(ROOT, "tests", "cpp", "paged_check")
    assert os.path.exists(prog), "make -C tests/cpp"
    out = subprocess.run([prog], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "paged positions ok" in out.stdout
