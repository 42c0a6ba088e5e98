"""GPU: what the cache, attention and sampling entry points refuse of tensors,
with the argument's name in the message, before anything runs."""
from __future__ import annotations

import pytest
import torch

import warp_route

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _z(*shape, dtype=torch.bfloat16, device="cuda"):
    return torch.zeros(*shape, dtype=dtype, device=device)


def _append(**kw):
    a = dict(k=_z(3, 2, 64), v=_z(3, 2, 64), k_cache=_z(4, 2, 16, 64), v_cache=_z(4, 2, 16, 64),
             slots=_z(3, dtype=torch.int64))
    opt = dict(positions=None, inv_freq=None, q=None)
    for n, t in kw.items():
        (a if n in a else opt)[n] = t
    return warp_route.append_paged_kv(a["k"], a["v"], a["k_cache"], a["v_cache"], a["slots"], **opt)


@pytest.mark.parametrize("kw,word", [
    (lambda: dict(k=_z(3, 2, 64, dtype=torch.float32)), "k and k_cache must have the same dtype"),
    (lambda: dict(v=_z(3, 2, 32)), "v must have shape"),
    (lambda: dict(v=_z(2, 2, 64)), "v must have shape"),
    (lambda: dict(k=_z(3, 64, 2).transpose(1, 2)), "last dimension must be contiguous"),
    (lambda: dict(k=_z(3, 2, 66)[:, :, 1:65]), "16-byte aligned"),
    (lambda: dict(k_cache=_z(4, 2, 16, 64, dtype=torch.float16)), "float32 or bfloat16"),
    (lambda: dict(v_cache=_z(4, 2, 8, 64)), "v_cache must have k_cache's shape"),
    (lambda: dict(v_cache=_z(4, 16, 2, 64).transpose(1, 2)), "strides"),
    (lambda: dict(k_cache=_z(2, 16, 64)), "k_cache must have shape"),
    (lambda: dict(slots=_z(3, dtype=torch.int32)), "slots must be"),
    (lambda: dict(slots=_z(4, dtype=torch.int64)), "slots must have shape"),
    (lambda: dict(slots=_z(3, dtype=torch.int64, device="cpu")), "slots must be a CUDA tensor"),
    (lambda: dict(positions=_z(3, dtype=torch.int64)), "go together"),
    (lambda: dict(positions=_z(3, dtype=torch.int64), inv_freq=_z(33, dtype=torch.float32)), "rot_dim"),
    (lambda: dict(positions=_z(3, dtype=torch.int64), inv_freq=_z(8, dtype=torch.float64)), "inv_freq must be"),
    (lambda: dict(q=_z(2, 4, 64)), "q must have shape"),
])
def test_append(kw, word):
    with pytest.raises(RuntimeError, match=word):
        _append(**kw())


def _attend(**kw):
    a = dict(q=_z(3, 4, 64), k_cache=_z(4, 2, 16, 64), v_cache=_z(4, 2, 16, 64), t=_z(3, 2, dtype=torch.int32),
             lens=_z(3, dtype=torch.int32))
    opt = {}
    for n, t in kw.items():
        (a if n in a else opt)[n] = t
    return warp_route.shared_prefix_attention(a["q"], a["k_cache"], a["v_cache"], a["t"], a["lens"], **opt)


@pytest.mark.parametrize("kw,word", [
    (lambda: dict(q=_z(3, 3, 64)), "num_q_heads"),
    (lambda: dict(q=_z(3, 4, 64, dtype=torch.float32)), "q and k_cache must have the same dtype"),
    (lambda: dict(q=_z(2, 4, 64)), "one token a sequence"),
    (lambda: dict(t=_z(3, 2, dtype=torch.int64)), "block_tables must be"),
    (lambda: dict(t=_z(3, dtype=torch.int32)), "block_tables must have shape"),
    (lambda: dict(t=_z(2, 3, dtype=torch.int32).t()), "block_tables' last dimension"),
    (lambda: dict(lens=_z(2, dtype=torch.int32)), "context_lens must have shape"),
    (lambda: dict(q_start=_z(3, dtype=torch.int32)), "q_start must have shape"),
    (lambda: dict(prefix_len=5), "prefix_pages must be given"),
    (lambda: dict(prefix_len=17, prefix_pages=_z(1, dtype=torch.int32)), "too few"),
    (lambda: dict(prefix_len=-1), "prefix_len"),
    (lambda: dict(prefix_len=5, prefix_pages=_z(1, dtype=torch.int64)), "prefix_pages must be"),
])
def test_attention(kw, word):
    with pytest.raises(RuntimeError, match=word):
        _attend(**kw())


@pytest.mark.parametrize("kw,word", [
    (dict(logits=(10,)), "logits must have shape"),
    (dict(uniforms=(4,)), "uniforms must have shape"),
    (dict(top_k=((3,), torch.int64)), "top_k must be"),
    (dict(top_p=((3,), torch.float64)), "top_p must be"),
    (dict(min_p=((2,), torch.float32)), "min_p must have shape"),
    (dict(temperature=((3, 1), torch.float32)), "temperature must have shape"),
])
def test_sampling(kw, word):
    logits = _z(*kw.get("logits", (3, 10)), dtype=torch.float32)
    uniforms = _z(*kw.get("uniforms", (3,)), dtype=torch.float32)
    opt = {n: _z(*v[0], dtype=v[1]) for n, v in kw.items() if n not in ("logits", "uniforms")}
    with pytest.raises(RuntimeError, match=word):
        warp_route.sample_tokens(logits, uniforms, **opt)
    with pytest.raises(RuntimeError, match="float32 or bfloat16"):
        warp_route.sample_tokens(_z(3, 10, dtype=torch.float16), _z(3, dtype=torch.float32))


def test_append_with_queries_of_no_heads():
    """Refused: it must not return as if the keys had been written."""
    with pytest.raises(RuntimeError, match="num_q_heads must be positive"):
        _append(q=_z(3, 0, 64))
    # no tokens is another matter: nothing to write
    out = _append(k=_z(0, 2, 64), v=_z(0, 2, 64), slots=_z(0, dtype=torch.int64), q=_z(0, 4, 64))
    assert out.shape == (0, 4, 64)
