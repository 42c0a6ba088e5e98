"""CPU: what the cache, attention and sampling entry points refuse, before
anything reaches a GPU."""
from __future__ import annotations

import ctypes

import pytest

from warp_route import _abi

FAKE = 0x10000  # aligned, never dereferenced
P = ctypes.c_void_p(FAKE)


def cache(**kw):
    f = dict(k=FAKE, v=FAKE, page_stride=2 * 16 * 64, head_stride=16 * 64, slot_stride=64, num_pages=4,
             num_kv_heads=2, page_size=16, head_dim=64, dtype=_abi.WR_DTYPE_BF16, reserved=0)
    f.update(kw)
    return _abi.PagedKv(*(f[n] for n, _ in _abi.PagedKv._fields_))


def rows(**kw):
    f = dict(ptr=FAKE, token_stride=512, head_stride=64)
    f.update(kw)
    return _abi.Rows(*(f[n] for n, _ in _abi.Rows._fields_))


def append(c=None, T=3, k=None, v=None, slots=P, pos=P, inv=P, rot=64, hq=4, q=None, q_out=None):
    lib = _abi.load()
    r = ctypes.byref
    return lib.wr_append_paged_kv(r(c or cache()), T, r(k or rows()), r(v or rows()), slots, pos, inv, rot, 0, hq,
                                  r(q) if q is not None else None, q_out, None)


def message():
    return _abi.load().wr_last_error_string().decode()


BAD_CACHES = [
    (dict(dtype=7), _abi.WR_ERR_INVALID, "dtype"),
    (dict(num_pages=0), _abi.WR_ERR_INVALID, "num_pages"),
    (dict(page_size=-1), _abi.WR_ERR_INVALID, "page_size"),
    (dict(num_kv_heads=0), _abi.WR_ERR_INVALID, "num_kv_heads"),
    (dict(head_dim=60), _abi.WR_ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=8), _abi.WR_ERR_UNSUPPORTED, "head_dim"),
    (dict(head_dim=264), _abi.WR_ERR_UNSUPPORTED, "head_dim"),
    (dict(k=0), _abi.WR_ERR_INVALID, "NULL"),
    (dict(v=FAKE + 2), _abi.WR_ERR_UNSUPPORTED, "aligned"),
    (dict(slot_stride=68), _abi.WR_ERR_UNSUPPORTED, "aligned"),
    (dict(page_stride=-64), _abi.WR_ERR_INVALID, "negative"),
]


@pytest.mark.parametrize("kw,status,word", BAD_CACHES)
def test_bad_caches(kw, status, word):
    assert append(cache(**kw)) == status and word in message()
    lib = _abi.load()
    d = _abi.AttnDesc(3, 3, 4, 2, 2, 0, 0.1)
    assert lib.wr_shared_prefix_attention_workspace_size(ctypes.byref(cache(**kw)), ctypes.byref(d), 0) == 0
    assert word in message()


@pytest.mark.parametrize("kw,status,word", [
    (dict(T=-1), _abi.WR_ERR_INVALID, "num_tokens"),
    (dict(rot=63), _abi.WR_ERR_INVALID, "rot_dim"),
    (dict(rot=66), _abi.WR_ERR_INVALID, "rot_dim"),
    (dict(pos=None), _abi.WR_ERR_INVALID, "positions"),
    (dict(inv=None), _abi.WR_ERR_INVALID, "positions"),
    (dict(slots=None), _abi.WR_ERR_INVALID, "slots"),
    (dict(k=rows(ptr=0)), _abi.WR_ERR_INVALID, "k must"),
    (dict(v=rows(ptr=FAKE + 8)), _abi.WR_ERR_UNSUPPORTED, "v and its strides"),
    (dict(k=rows(token_stride=515)), _abi.WR_ERR_UNSUPPORTED, "k and its strides"),
    (dict(q=rows()), _abi.WR_ERR_INVALID, "q and q_out"),
    (dict(q=rows(), q_out=P), _abi.WR_ERR_INVALID, "alias"),
    (dict(q=rows(ptr=FAKE + 4096), q_out=P, hq=0), _abi.WR_ERR_INVALID, "num_q_heads"),
    (dict(q=rows(ptr=FAKE + 4096), q_out=P, hq=20000), _abi.WR_ERR_UNSUPPORTED, "heads"),
])
def test_bad_appends(kw, status, word):
    assert append(**kw) == status and word in message()


def test_append_of_no_tokens_needs_no_gpu():
    assert append(T=0, k=rows(ptr=0), v=rows(ptr=0), slots=None, rot=0, pos=None, inv=None) == _abi.WR_OK


def attend(T=3, B=3, hq=4, width=2, prefix=0, q=None, tables=P, lens=P, q_start=None, pp=None, out=P, ws=P,
           ws_bytes=1 << 40, stride=2):
    lib = _abi.load()
    r = ctypes.byref
    d = _abi.AttnDesc(T, B, hq, width, stride, prefix, 0.1)
    return lib.wr_shared_prefix_attention(r(cache()), r(d), r(q or rows()), tables, lens, q_start, pp, out, None, ws,
                                          ws_bytes, None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(T=-1, B=-1), _abi.WR_ERR_INVALID, "num_tokens"),
    (dict(T=4), _abi.WR_ERR_INVALID, "q_start"),
    (dict(T=4, B=0, q_start=P), _abi.WR_ERR_INVALID, "num_seqs"),
    (dict(hq=3), _abi.WR_ERR_INVALID, "num_q_heads"),
    (dict(hq=0), _abi.WR_ERR_INVALID, "num_q_heads"),
    (dict(prefix=-1), _abi.WR_ERR_INVALID, "prefix_len"),
    (dict(prefix=5), _abi.WR_ERR_INVALID, "prefix_pages"),
    (dict(width=1 << 28), _abi.WR_ERR_UNSUPPORTED, "keys"),
    (dict(stride=-2), _abi.WR_ERR_INVALID, "table_stride"),
    (dict(q=rows(ptr=0)), _abi.WR_ERR_INVALID, "q must"),
    (dict(q=rows(ptr=FAKE + 2)), _abi.WR_ERR_UNSUPPORTED, "q and its strides"),
    (dict(tables=None), _abi.WR_ERR_INVALID, "block_tables"),
    (dict(lens=None), _abi.WR_ERR_INVALID, "context_lens"),
    (dict(out=None), _abi.WR_ERR_INVALID, "out"),
    (dict(out=ctypes.c_void_p(FAKE + 2)), _abi.WR_ERR_UNSUPPORTED, "out"),
    (dict(ws=None), _abi.WR_ERR_WORKSPACE, "workspace"),
    (dict(ws=ctypes.c_void_p(FAKE + 16)), _abi.WR_ERR_WORKSPACE, "aligned"),
    (dict(ws_bytes=100), _abi.WR_ERR_WORKSPACE, "too small"),
])
def test_bad_attention_calls(kw, status, word):
    assert attend(**kw) == status and word in message()


def test_attention_of_no_tokens_needs_no_gpu():
    assert attend(T=0, B=0) == _abi.WR_OK
    assert attend(T=0, B=2, q_start=P) == _abi.WR_OK


def test_attention_workspace_grows_with_the_batch():
    lib = _abi.load()

    def size(T, prefix, q_start=0):
        d = _abi.AttnDesc(T, T, 4, 2, 2, prefix, 0.1)
        return lib.wr_shared_prefix_attention_workspace_size(ctypes.byref(cache()), ctypes.byref(d), q_start)

    # partial results of the prefix for every row: fp32 sums and (m, l)
    assert size(64, 1000) >= size(64, 0) + 64 * 4 * (64 * 4 + 8)
    assert size(64, 0, 1) >= size(64, 0) + 64 * 4


def sample(rows_=2, vocab=10, dtype=_abi.WR_DTYPE_F32, logits=P, stride=10, u=P, s=True, ids=P):
    st = _abi.Sampling(1.0, 1.0, 0.0, 0, None, None, None, None)
    return _abi.load().wr_sample_tokens(rows_, vocab, dtype, logits, stride, u, ctypes.byref(st) if s else None, ids,
                                        None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(rows_=-1), _abi.WR_ERR_INVALID, "num_rows"),
    (dict(rows_=1 << 30), _abi.WR_ERR_INVALID, "num_rows"),
    (dict(vocab=0), _abi.WR_ERR_INVALID, "vocab"),
    (dict(vocab=262145), _abi.WR_ERR_UNSUPPORTED, "vocab"),
    (dict(dtype=9), _abi.WR_ERR_INVALID, "dtype"),
    (dict(stride=-1), _abi.WR_ERR_INVALID, "row_stride"),
    (dict(logits=None), _abi.WR_ERR_INVALID, "logits"),
    (dict(u=None), _abi.WR_ERR_INVALID, "uniforms"),
    (dict(s=False), _abi.WR_ERR_INVALID, "sampling"),
    (dict(ids=None), _abi.WR_ERR_INVALID, "ids"),
])
def test_bad_samples(kw, status, word):
    assert sample(**kw) == status and word in message()


def test_sample_of_no_rows_needs_no_gpu():
    assert sample(rows_=0, logits=None, u=None, ids=None) == _abi.WR_OK


def test_python_entry_points_refuse_what_is_not_on_a_gpu():
    import torch

    import warp_route

    c = torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="k_cache must be a CUDA tensor"):
        warp_route.append_paged_kv(k, k, c, c, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="k_cache must be a CUDA tensor"):
        warp_route.shared_prefix_attention(k, c, c, torch.zeros(3, 1, dtype=torch.int32),
                                           torch.zeros(3, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="logits must be a CUDA tensor"):
        warp_route.sample_tokens(torch.zeros(1, 10), torch.zeros(1))


def test_append_with_queries_of_no_heads():
    # an empty tensor's pointer is NULL: the heads are what is wrong with it
    assert append(q=rows(ptr=FAKE + 4096), q_out=None, hq=0) == _abi.WR_ERR_INVALID
    assert "num_q_heads must be positive" in message()


@pytest.mark.parametrize("kw", [dict(page_stride=0), dict(head_stride=0), dict(slot_stride=0)])
def test_append_into_an_expanded_cache(kw):
    """Heads (rows, pages) that are one memory cannot hold keys of their own."""
    assert append(cache(**kw)) == _abi.WR_ERR_INVALID and "strides" in message()
    # read, such a cache is as good as any; a dimension of one has no stride that counts
    d = _abi.AttnDesc(3, 3, 4, 2, 2, 0, 0.1)
    lib = _abi.load()
    assert lib.wr_shared_prefix_attention_workspace_size(ctypes.byref(cache(**kw)), ctypes.byref(d), 0) > 0
    one = dict(num_pages=1, num_kv_heads=1, page_size=1, page_stride=0, head_stride=0, slot_stride=0)
    assert append(cache(**one), T=0) == _abi.WR_OK


def test_prefix_waits_have_one_answer_for_a_warp():
    """k_attn_prefix branches on its waits around warp-wide instructions: each
    wait whose answer counts goes through a vote, and so does the word by
    which one warp tells the others that it gave up."""
    import os
    import re

    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(repo, "warp-route_b200", "csrc", "wr_attn_prefix.cu")) as f:
        text = f.read()
    lines = [ln.split("//")[0].strip() for ln in text.splitlines()]
    for ln in lines:
        if "mbar_wait(" in ln or "mbar_try_wait(" in ln or "wait_long(" in ln:
            dropped = ln.startswith("mbar_wait(")  # its answer is not used
            itself = re.match(r"(__device__|return mbar_wait\(bar, parity, abort, )", ln)
            assert dropped or itself or "__all_sync(0xffffffffu," in ln, ln
        if "*abort" in ln and not re.search(r"\*abort = 1;|volatile int\* abort", ln):
            assert "__any_sync(0xffffffffu, *abort)" in ln, ln
