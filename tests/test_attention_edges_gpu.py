"""GPU: shared_prefix_attention where its tensor-core kernel for the prefix can
go wrong, against the 64-bit form with the tolerances of test_attention_gpu.

That kernel takes bf16 calls with more than 32 rows (tokens times query heads a
key head) for each key head and more than 64 MB of keys and values read again
for every 16 rows; it has one tile of 128 rows a CTA up to 128 rows and two
above.  Each case here says which of the two it is meant for, and the rule is
worked out from the sizes, so that a case that would not reach the kernel
fails rather than passes for nothing.
"""
from __future__ import annotations

import pytest
import torch

import warp_route
from test_attention_gpu import call, check, make

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def tiles(tokens, hq, hk, d, prefix):
    """Row tiles a CTA of the prefix's kernel, 0: it does not take the call."""
    rows = tokens * hq // hk
    again = -(-rows // 16) * hk * prefix * d * 4
    return 0 if rows <= 32 or again <= 64 << 20 else 1 if rows <= 128 else 2


@pytest.mark.parametrize("n,hq,hk,d,page,prefix,layout,want", [
    (33, 8, 8, 128, 16, 5600, "heads", 1),      # 33 rows a key head
    (17, 16, 8, 128, 32, 5471, "tokens", 1),    # 34
    (16, 32, 8, 128, 64, 5000, "heads", 1),     # a small batch
    (21, 48, 8, 128, 128, 2731, "heads", 1),    # 126, six heads a key head
    (127, 16, 16, 96, 16, 1409, "heads", 1),    # 127, columns behind the head
    (32, 32, 8, 128, 16, 2049, "heads", 1),     # 128: the tile is full; one key in the last unit
    (32, 32, 8, 72, 32, 3700, "tokens", 1),
    (60, 8, 4, 72, 256, 7400, "heads", 1),
    (64, 16, 8, 64, 16, 4097, "heads", 1),      # the same with heads of 64
    (43, 24, 8, 64, 64, 4000, "tokens", 2),     # 129
    (43, 24, 8, 128, 16, 2000, "heads", 2),     # 129
    (65, 16, 8, 128, 64, 1921, "tokens", 2),    # 130
    (51, 40, 8, 128, 32, 1025, "heads", 2),     # 255
    (64, 32, 8, 128, 16, 1151, "heads", 2),     # 256: both tiles full
    (64, 32, 8, 64, 16, 2304, "heads", 2),
    (257, 8, 8, 128, 16, 1023, "heads", 2),     # 257: a row of a second pair of tiles
    (520, 32, 8, 128, 16, 128, "heads", 2),     # one unit of 128 keys, whole
    (530, 32, 8, 128, 64, 127, "tokens", 2),    # ... and cut
    (520, 32, 8, 128, 128, 129, "heads", 2),    # ... and one key more
])
def test_edges_of_the_tiles(n, hq, hk, d, page, prefix, layout, want):
    assert tiles(n, hq, hk, d, prefix) == want
    s = make([(i * 29) % 40 for i in range(n)], [1] * n, hq, hk, d, page, prefix, torch.bfloat16, layout=layout, seed=n)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)
    again, _ = call(s, return_lse=True)
    assert torch.equal(out, again)


@pytest.mark.parametrize("prefix", [1, 2])
def test_a_prefix_of_one_key(prefix):
    """Two million rows behind one or two keys, no own keys: the outputs are
    the key's value, or a mean of two."""
    n, hk, d = 33000, 64, 128
    assert tiles(n, hk, hk, d, prefix) == 2
    if torch.cuda.mem_get_info()[0] < 16 << 30:
        pytest.skip("needs 16 GB")
    g = torch.Generator(device="cuda").manual_seed(prefix)
    kc = torch.full((3, hk, 16, d), float("nan"), device="cuda", dtype=torch.bfloat16)
    vc = torch.full_like(kc, float("nan"))
    kc[1, :, :prefix] = torch.randn(hk, prefix, d, generator=g, device="cuda").bfloat16()
    vc[1, :, :prefix] = torch.randn(hk, prefix, d, generator=g, device="cuda").bfloat16()
    q = torch.randn(n, hk, d, generator=g, device="cuda", dtype=torch.bfloat16)
    out, lse = warp_route.shared_prefix_attention(
        q, kc, vc, torch.zeros(n, 0, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"),
        prefix_pages=torch.tensor([1], dtype=torch.int32, device="cuda"), prefix_len=prefix, return_lse=True)
    k, v = kc[1, :, :prefix].double(), vc[1, :, :prefix].double()
    for lo in range(0, n, 3000):
        s = torch.einsum("nhd,hkd->nhk", q[lo:lo + 3000].double(), k) * d ** -0.5
        size = torch.einsum("nhd,hkd->nhk", q[lo:lo + 3000].double().abs(), k.abs()).amax(-1) * d ** -0.5
        es = (d + 8) * 2.0 ** -24 * size
        p = s.softmax(-1)
        ref, mass = torch.einsum("nhk,hkd->nhd", p, v), torch.einsum("nhk,hkd->nhd", p, v.abs())
        # as in test_attention_gpu: scores, weights in bf16, sums, the output rounded once
        bound = mass * (2.0 ** -8 * (1 + 2.0 ** -8) + 2 * es[..., None] + 2.0 ** -19 + 65 * 2.0 ** -24)
        bound = bound + 2.0 ** -8 * (ref.abs() + bound)
        assert ((out[lo:lo + 3000].double() - ref).abs() <= bound).all()
        want = torch.logsumexp(s, -1)
        assert ((lse[lo:lo + 3000].double() - want).abs()
                <= es + 2.0 ** -20 + 66 * 2.0 ** -24 + 2.0 ** -23 * want.abs()).all()


def test_prefix_pages_beyond_32_bits():
    """Pages whose offsets pass 2^32 bytes and 2^31 elements, read by tiles."""
    hk, page, d, pages, prefix, n = 8, 64, 128, 33000, 2100, 64
    assert tiles(n, 2 * hk, hk, d, prefix) == 1
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    g = torch.Generator(device="cuda").manual_seed(1)
    kc = torch.empty(pages, hk, page, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    tail = 40
    kc[-tail:].normal_(generator=g)
    vc[-tail:].normal_(generator=g)
    q = torch.randn(n, 2 * hk, d, generator=g, device="cuda").bfloat16()
    order = pages - tail + torch.randperm(tail, generator=g, device="cuda").int()
    t = order[-1:].expand(n, 1).contiguous()
    lens = (torch.arange(n, device="cuda") % 60).int()
    pp = order[:-(-prefix // page)].contiguous()
    out, lse = warp_route.shared_prefix_attention(q, kc, vc, t, lens, prefix_pages=pp, prefix_len=prefix,
                                                  return_lse=True)
    small = dict(q=q, k_cache=kc[-tail:].clone(), v_cache=vc[-tail:].clone(), tables=t - (pages - tail), lens=lens,
                 prefix_pages=pp - (pages - tail), prefix=prefix, q_start=None)
    del kc, vc
    check(small, out, lse)


def test_one_row_tile_with_scores_that_grow():
    """The running maximum moves by more than is tolerated without rescaling."""
    n, prefix = 16, 5000
    assert tiles(n, 32, 8, 128, prefix) == 1
    s = make([5] * n, [1] * n, 32, 8, 128, 16, prefix, torch.bfloat16)
    ramp = torch.linspace(0.05, 3.0, prefix, device="cuda")
    for i, p in enumerate(s["prefix_pages"].tolist()):
        rows = min(16, prefix - 16 * i)
        s["k_cache"][p, :, :rows] *= ramp[16 * i:16 * i + rows, None].to(torch.bfloat16)
    s["q"][::3] *= 4
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("hq,prefix,want", [(16, 5000, 1), (64, 3000, 2)])
def test_bad_pages_and_several_tokens_in_front_of_tiles(hq, prefix, want):
    nq = [i % 5 for i in range(24)]
    assert tiles(sum(nq), hq, 8, 128, prefix) == want
    s = make([(i * 53) % 200 + 9 for i in range(24)], nq, hq, 8, 128, 32, prefix, torch.bfloat16)
    s["prefix_pages"][3] = -1
    s["prefix_pages"][8:16] = 2 ** 31 - 1
    s["prefix_pages"][-1] = s["k_cache"].shape[0]
    out, lse = call(s, return_lse=True)
    check(s, out, lse)
    tail = torch.full_like(s["q"][:3], 7.0)  # tokens of no sequence
    more, ml = call(dict(s, q=torch.cat([s["q"], tail])), return_lse=True)
    assert not more[-3:].any() and (ml[-3:] == float("-inf")).all()
    check(s, more[:-3], ml[:-3])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,group,prefix", [(64, 8, 0), (128, 4, 0), (256, 3, 0), (96, 1, 70), (128, 20, 300),
                                            (128, 8, 10000)])
def test_later_keys_that_are_not_finite_against_the_plain_form(d, group, prefix, dtype):
    nq, lens = [1, 20, 7, 40, 33], [50, 20, 90, 47, 200]
    s = make(lens, nq, 2 * group, 2, d, 16, prefix, dtype)
    clean = call(s, return_lse=True)
    starts = [sum(nq[:i]) for i in range(6)]
    hit = torch.zeros(sum(nq), dtype=torch.bool, device="cuda")
    dirty = dict(s, k_cache=s["k_cache"].clone(), v_cache=s["v_cache"].clone())
    for b, back in ((1, 1), (2, 3), (3, 20), (4, 2)):
        for j in (lens[b] - back, lens[b] - 1):
            page = s["tables"][b, j // 16]
            dirty["k_cache"][page, :, j % 16] = float("nan")
            dirty["v_cache"][page, :, j % 16, ::3] = float("inf")
        hit[starts[b] + nq[b] - back:starts[b + 1]] = True
    out, lse = call(dirty, return_lse=True)
    # rows that see none of those keys: as if they were not there
    out[hit], lse[hit] = clean[0][hit], clean[1][hit]
    check(s, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hq,prefix,several", [(8, 0, False), (8, 0, True), (8, 70, False), (8, 70, True),
                                               (32, 5000, False), (32, 5000, True)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_stays_alone(bad, hq, prefix, several, dtype):
    """Rows share tiles of products: one token's query must not reach another's output."""
    nq = [3, 1, 4, 2, 7] if several else [1] * 17
    if prefix == 5000 and dtype == torch.bfloat16:
        assert tiles(sum(nq), hq, 8, 128, prefix) == 1
    s = make([(i * 31) % 90 + 7 for i in range(len(nq))], nq, hq, 8, 128, 16, prefix, dtype)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)
    q = s["q"].clone()
    q[5, ::2] = bad
    got, gl = call(dict(s, q=q), return_lse=True)
    keep = torch.ones(q.shape[:2], dtype=torch.bool, device="cuda")
    keep[5, ::2] = False
    assert torch.equal(got[keep], out[keep]) and torch.equal(gl[keep], lse[keep])
    assert torch.isnan(got[~keep]).all()
