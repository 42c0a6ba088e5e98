"""GPU: append_paged_kv against a 64-bit form.

Tolerance: the angle's remainder (at most half a turn) is rounded to 24 bits
and sine and cosine to about 2 of their last places, so each is off by at most
2^-22 absolutely; two products and a sum add 3 * 2^-24 of their size; the
result is rounded once to the type.  With s = |x_i| + |x_j|:
error <= s * 2^-21 + half a step of the value (eps / 2).
"""
from __future__ import annotations

import pytest
import torch

import warp_route
from decode_reference import rotate

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _check(got, want, x, rot, dtype):
    half = torch.finfo(dtype).eps / 2
    s = x.double().abs()
    size = s.amax(-1, keepdim=True) * 2  # at least |x_i| + |x_j| of any pair
    err = (got.double() - want).abs()
    bound = size * 2.0 ** -21 + half * (want.abs() + size * 2.0 ** -21)
    assert (err <= bound).all(), (err - bound).max()
    assert torch.equal(got[..., rot:], x[..., rot:])  # the rest of the head as it was


def _case(T, hq, hk, d, page, pages, dtype, seed=0, layout="heads"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    qkv = torch.randn(T, (hq + 2 * hk) * d, generator=g, device="cuda").to(dtype)
    heads = qkv.view(T, hq + 2 * hk, d)
    shape = (pages, hk, page, d) if layout == "heads" else (pages, page, hk, d)
    kc = torch.randn(shape, generator=g, device="cuda").to(dtype)
    vc = torch.randn(shape, generator=g, device="cuda").to(dtype)
    if layout != "heads":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    return heads[:, :hq], heads[:, hq:hq + hk], heads[:, hq + hk:], kc, vc, g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hq,hk,d,rot,page,pages,far,interleaved,layout", [
    (1, 32, 8, 128, 128, 16, 4, 10, False, "heads"),
    (1, 1, 1, 16, 16, 1, 3, 1, True, "heads"),           # the smallest of everything
    (7, 6, 2, 80, 40, 16, 5, 1000000, False, "heads"),   # half a rotation is no whole chunk
    (37, 8, 8, 64, 64, 7, 9, 131072, False, "tokens"),   # pages of 7, token-major cache
    (130, 12, 2, 256, 128, 64, 3, 4096, True, "tokens"),
    (33, 4, 4, 96, 20, 32, 2, 999999, False, "heads"),
    (33, 4, 4, 96, 22, 32, 2, 999999, True, "heads"),    # ends inside a chunk
])
def test_append_matches_plain(T, hq, hk, d, rot, page, pages, far, interleaved, layout, dtype):
    q, k, v, kc, vc, g = _case(T, hq, hk, d, page, pages, dtype, layout=layout)
    n = pages * page
    slots = torch.randperm(n, generator=g, device="cuda")[:T]
    if slots.numel() < T:  # more tokens than slots: the rest has none
        slots = torch.cat([slots, torch.full((T - n,), -1, device="cuda", dtype=torch.int64)])
    if T > 3:
        slots[1] = -1          # padding
        slots[2] = n           # behind the cache: dropped
        slots[T - 1] = -2 ** 62
    positions = torch.randint(0, far, (T,), generator=g, device="cuda")
    inv = (1e6 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)).float()
    k0, v0 = kc.clone(), vc.clone()
    qr = warp_route.append_paged_kv(k, v, kc, vc, slots, positions=positions, inv_freq=inv, q=q,
                                    interleaved=interleaved)
    torch.cuda.synchronize()
    _check(qr, rotate(q, positions, inv, interleaved), q, rot, dtype)
    live = (slots >= 0) & (slots < n)
    at = slots[live]
    rows_k, rows_v = kc[at // page, :, at % page], vc[at // page, :, at % page]
    _check(rows_k, rotate(k, positions, inv, interleaved)[live], k[live], rot, dtype)
    assert torch.equal(rows_v, v[live])
    # every other slot as it was
    mask = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    mask[at // page, at % page] = False
    m = mask[:, None, :, None]
    assert torch.equal(torch.where(m, kc, 0), torch.where(m, k0, 0))
    assert torch.equal(torch.where(m, vc, 0), torch.where(m, v0, 0))


def test_append_without_rotation_or_queries():
    q, k, v, kc, vc, g = _case(5, 4, 2, 64, 16, 2, torch.bfloat16)
    slots = torch.arange(5, device="cuda") + 3
    assert warp_route.append_paged_kv(k, v, kc, vc, slots) is None
    assert torch.equal(kc[0, :, 3:8].transpose(0, 1), k) and torch.equal(vc[0, :, 3:8].transpose(0, 1), v)
    qr = warp_route.append_paged_kv(k, v, kc, vc, slots, q=q)  # no angles: a copy
    assert torch.equal(qr, q)


def test_append_no_tokens():
    q, k, v, kc, vc, _ = _case(0, 4, 2, 64, 16, 2, torch.bfloat16)
    k0 = kc.clone()
    e = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert warp_route.append_paged_kv(k, v, kc, vc, e) is None
    assert warp_route.append_paged_kv(k, v, kc, vc, e, q=q).shape == (0, 4, 64)
    assert torch.equal(kc, k0)


def test_append_in_a_cache_beyond_32_bits():
    """Offsets of more than 2^31 elements: pages far apart in one buffer."""
    hk, page, d, pages = 8, 64, 128, 33000  # 2.2e9 elements, 4.3 GB each
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    kc = torch.empty(pages, hk, page, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    k = torch.randn(2, hk, d, device="cuda").bfloat16()
    slots = torch.tensor([pages * page - 1, 5], device="cuda")
    warp_route.append_paged_kv(k, -k, kc, vc, slots)
    assert torch.equal(kc[-1, :, -1], k[0]) and torch.equal(vc[-1, :, -1], -k[0])
    assert torch.equal(kc[0, :, 5], k[1])


def test_append_in_a_graph_and_on_a_stream():
    q, k, v, kc, vc, g = _case(9, 4, 2, 64, 16, 4, torch.bfloat16)
    slots = torch.arange(9, device="cuda")
    pos = torch.arange(9, device="cuda")
    inv = torch.full((32,), 0.25, device="cuda")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        qr = warp_route.append_paged_kv(k, v, kc, vc, slots, positions=pos, inv_freq=inv, q=q)
    slots += 20  # the graph reads what is there when it runs
    graph.replay()
    torch.cuda.synchronize()
    _check(qr, rotate(q, pos, inv, False), q, 64, torch.bfloat16)
    at = slots
    assert torch.equal(vc[at // 16, :, at % 16], v)
