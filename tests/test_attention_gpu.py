"""GPU: shared_prefix_attention against a 64-bit form.

Tolerances.  With u = eps / 2 of the type, M = sum_j p_j |v_j| (the reference
gives it) and n keys:
  * scores: sums of d products in fp32, |error| <= es = (d + 8) 2^-24 S with S
    the largest sum |q_i k_i| * scale of the row; a weight is then off by a
    factor 1 +- (es + 2^-20) (exponent's argument and its approximation);
  * weights rounded to bf16 for the second product: 2^-8 each, so 2^-8 M;
  * sums over the keys in fp32: (n / 16 + 64) 2^-24 M at most with the 16 keys
    of a unit added exactly enough (their 16 roundings are within the 64);
  * the output rounded once: u |out|.
fp32 has no rounding of the weights but sums key by key: (n + 64) 2^-24 M.
lse: es + 2^-20 + (n + 64) 2^-24, and its own rounding 2^-24 |lse|.
"""
from __future__ import annotations

import pytest
import torch

import warp_route
from decode_reference import attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def make(lens, nq, hq, hk, d, page, prefix, dtype, seed=0, layout="heads", spare=2, junk=float("nan")):
    """Inputs; slots that hold no key are filled with `junk`."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    counts = [-(-c // page) for c in lens]
    np_ = -(-prefix // page)
    total = np_ + sum(counts) + spare
    order = torch.randperm(total, generator=g, device="cuda").tolist()
    shape = (total, hk, page, d) if layout == "heads" else (total, page, hk, d)
    kc = torch.randn(shape, generator=g, device="cuda").to(dtype)
    vc = torch.randn(shape, generator=g, device="cuda").to(dtype)
    if layout != "heads":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    used = torch.zeros(total, page, dtype=torch.bool, device="cuda")
    pp, at = order[:np_], np_
    for i, p in enumerate(pp):
        used[p, :min(page, prefix - i * page)] = True
    wide = max(counts + [1])
    tables = torch.full((len(lens), wide), 10 ** 9, dtype=torch.int32)
    for b, c in enumerate(lens):
        for i in range(counts[b]):
            tables[b, i] = order[at]
            used[order[at], :min(page, c - i * page)] = True
            at += 1
    m = used[:, None, :, None]
    kc.copy_(torch.where(m, kc, torch.full_like(kc, junk)))
    vc.copy_(torch.where(m, vc, torch.full_like(vc, junk)))
    q = torch.randn(sum(nq), hq, d, generator=g, device="cuda").to(dtype)
    start = None
    if any(n != 1 for n in nq):
        start = torch.tensor([sum(nq[:i]) for i in range(len(nq) + 1)], dtype=torch.int32, device="cuda")
    return dict(q=q, k_cache=kc, v_cache=vc, tables=tables.cuda(),
                lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                prefix_pages=torch.tensor(pp, dtype=torch.int32, device="cuda") if prefix else None,
                prefix=prefix, q_start=start)


def call(s, **kw):
    return warp_route.shared_prefix_attention(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lens"],
                                              prefix_pages=s["prefix_pages"], prefix_len=s["prefix"],
                                              q_start=s["q_start"], **kw)


def check(s, out, lse=None, scale=None):
    q = s["q"]
    d = q.shape[2]
    scale = d ** -0.5 if scale is None else scale
    want, wl, mass, size = attention(q, s["k_cache"], s["v_cache"], s["tables"], s["lens"],
                                     s["prefix_pages"], s["prefix"], s["q_start"], scale)
    n = s["prefix"] + (int(s["lens"].max()) if s["lens"].numel() else 0)
    es = ((d + 8) * 2.0 ** -24 * size).unsqueeze(-1)
    if q.dtype == torch.bfloat16:
        bound = mass * (2.0 ** -8 * (1 + 2.0 ** -8) + 2 * es + 2.0 ** -19 + (n / 16 + 64) * 2.0 ** -24)
    else:
        bound = mass * (2 * es + 2.0 ** -19 + (n + 64) * 2.0 ** -24)
    bound = bound + torch.finfo(q.dtype).eps / 2 * (want.abs() + bound)
    err = (out.double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= bound).all(), f"over by {(err - bound).max():.3e}, error {err.max():.3e}"
    if lse is not None:
        none = wl == float("-inf")
        assert torch.equal(none, lse == float("-inf"))
        eb = es.squeeze(-1) + 2.0 ** -20 + (n + 64) * 2.0 ** -24 + 2.0 ** -23 * wl.abs()
        assert ((lse.double() - wl).abs() <= eb)[~none].all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,hq,hk,page,layout", [
    (128, 8, 2, 16, "heads"), (64, 4, 4, 32, "tokens"), (256, 6, 1, 16, "heads"), (96, 6, 2, 7, "tokens"),
    (16, 16, 1, 1, "heads"), (80, 5, 1, 64, "heads"), (248, 2, 2, 33, "heads"), (128, 40, 2, 16, "heads"),
])
@pytest.mark.parametrize("prefix", [0, 1, 37, 300])
def test_one_token_a_sequence(prefix, d, hq, hk, page, layout, dtype):
    s = make([1, 0, 15, 16, 17, 130, 64], [1] * 7, hq, hk, d, page, prefix, dtype, layout=layout)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,prefix", [([1], 0), ([5], 0), ([0], 3), ([2000], 0), ([1999], 1001), ([0], 0)])
def test_one_sequence(lens, prefix, dtype):
    s = make(lens, [1], 8, 2, 128, 16, prefix, dtype)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,lens,prefix", [
    ([3, 1, 4], [3, 1, 4], 0),           # prompts: the first token sees itself alone
    ([5, 2, 0, 9], [100, 2, 30, 40], 77),
    ([33, 17], [33, 200], 129),
    ([4], [2], 0),                       # more tokens than keys: the first rows see none
    ([4, 1], [2, 1], 20),
    ([0, 0], [5, 6], 10),                # nobody asks
])
def test_several_tokens_a_sequence(nq, lens, prefix, dtype):
    s = make(lens, nq, 6, 2, 128, 16, prefix, dtype)
    if sum(nq) == 0:
        s["q_start"] = torch.zeros(3, dtype=torch.int32, device="cuda")
        assert call(s).shape == (0, 6, 128)
        return
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("n,hq,hk,d,page,prefix,layout", [
    (70, 16, 2, 128, 16, 1000, "heads"),      # 560 rows: two tiles and a rest
    (17, 4, 2, 128, 16, 1, "heads"),          # 34 rows, one key
    (33, 2, 2, 64, 32, 127, "tokens"),
    (64, 2, 1, 128, 128, 128, "heads"),       # 128 rows, whole tiles of keys
    (65, 2, 1, 64, 256, 129, "heads"),        # pages larger than a tile
    (43, 6, 2, 128, 64, 4000, "tokens"),      # a group that does not divide a tile
    (256, 8, 8, 64, 16, 511, "heads"),
    (130, 48, 8, 128, 64, 2500, "heads"),
    (40, 4, 4, 128, 8, 300, "heads"),         # pages too small for TMA copies of tiles
    (40, 4, 4, 96, 16, 300, "heads"),
    (40, 4, 4, 128, 24, 300, "heads"),
    (700, 16, 2, 96, 16, 1500, "heads"),      # columns behind the head
    (300, 24, 2, 72, 32, 2000, "tokens"),
    (200, 32, 4, 128, 256, 2700, "heads"),    # enough bytes for the tensor cores
    (150, 32, 4, 64, 16, 6000, "tokens"),
    (90, 32, 16, 128, 32, 3100, "heads"),
    (60, 16, 8, 64, 64, 9000, "heads"),       # 120 rows a head: one tile
])
def test_many_rows_behind_a_prefix(n, hq, hk, d, page, prefix, layout):
    s = make([(i * 37) % 90 for i in range(n)], [1] * n, hq, hk, d, page, prefix, torch.bfloat16, layout=layout)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)
    again, _ = call(s, return_lse=True)
    assert torch.equal(out, again)


def test_scores_that_grow_along_the_prefix():
    """The running maximum moves by more than the kernels tolerate without
    rescaling, again and again, for some rows and not for others."""
    s = make([5] * 80, [1] * 80, 16, 8, 128, 16, 2000, torch.bfloat16)
    ramp = torch.linspace(0.05, 3.0, 2000, device="cuda")
    pages = s["prefix_pages"].long()
    for i, p in enumerate(pages.tolist()):
        rows = min(16, 2000 - 16 * i)
        s["k_cache"][p, :, :rows] *= ramp[16 * i:16 * i + rows, None].to(torch.bfloat16)
    s["q"][::3] *= 4
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


def test_bad_pages_hide_a_tile_of_the_prefix():
    s = make([9] * 50, [1] * 50, 256, 16, 128, 16, 500, torch.bfloat16)
    s["prefix_pages"][3] = -1
    s["prefix_pages"][8:16] = 2 ** 31 - 1   # a whole tile of 128 keys
    s["prefix_pages"][-1] = s["k_cache"].shape[0]
    out, lse = call(s, return_lse=True)
    check(s, out, lse)
    s["prefix_pages"][:] = -7               # nothing of the prefix is left
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


def test_several_tokens_and_many_rows():
    s = make([(i * 53) % 200 + 9 for i in range(24)], [i % 9 + 1 for i in range(24)], 64, 8, 128, 32, 1111,
             torch.bfloat16)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


def test_bad_pages_hide_their_keys():
    for dtype in (torch.bfloat16, torch.float32):
        s = make([100, 50, 16], [1, 1, 1], 8, 2, 128, 16, 70, dtype)
        s["tables"][0, 2] = -1
        s["tables"][1, 0] = 2 ** 30
        s["tables"][2, 0] = s["k_cache"].shape[0]
        s["prefix_pages"][1] = -5
        out, lse = call(s, return_lse=True)
        check(s, out, lse)


def test_lengths_beyond_the_table_and_below_zero():
    s = make([40, 40], [1, 1], 4, 2, 64, 16, 0, torch.bfloat16, junk=0.5)
    full = dict(s, lens=torch.tensor([48, 0], dtype=torch.int32, device="cuda"))
    out = call(dict(s, lens=torch.tensor([2 ** 31 - 1, -7], dtype=torch.int32, device="cuda")))
    assert torch.equal(out, call(full))


def test_tokens_of_no_sequence_get_zero():
    s = make([20, 30], [2, 3], 4, 2, 64, 16, 33, torch.bfloat16)
    q = torch.cat([s["q"], torch.full_like(s["q"][:3], 7.0)])
    out, lse = call(dict(s, q=q), return_lse=True)
    assert (out[5:] == 0).all() and (lse[5:] == float("-inf")).all()
    check(s, out[:5], lse[:5])


def test_strided_queries_and_tables():
    s = make([20, 30], [1, 1], 4, 2, 64, 16, 33, torch.bfloat16)
    want = call(s)
    wide = torch.zeros(2, 10, 64, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:7] = s["q"]
    t = torch.full((4, s["tables"].shape[1] + 3), -9, dtype=torch.int32, device="cuda")
    t[::2, :-3] = s["tables"]
    got = call(dict(s, q=wide[:, 3:7], tables=t[::2, :-3]))
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_other_scales(scale):
    s = make([60, 3], [1, 1], 4, 2, 128, 16, 21, torch.bfloat16)
    out, lse = call(s, scale=scale, return_lse=True)
    check(s, out, lse, scale=scale)


def test_large_scores_do_not_overflow():
    s = make([100], [1], 4, 2, 128, 16, 0, torch.float32)
    s["q"] *= 300
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


def test_same_result_every_time():
    for prefix, n in ((0, 1), (700, 9)):
        s = make([500 + 31 * i for i in range(n)], [1] * n, 8, 2, 128, 16, prefix, torch.bfloat16)
        first = call(s)
        for _ in range(5):
            assert torch.equal(call(s), first)


def test_graph_follows_lengths_and_two_graphs_share_nothing():
    s = make([64, 64, 64], [1, 1, 1], 8, 2, 128, 16, 100, torch.bfloat16, junk=0.25)
    r = make([30, 90], [1, 1], 8, 2, 128, 16, 0, torch.bfloat16, seed=1, junk=0.25)
    graphs, outs = [], []
    for x in (s, r):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            call(x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(call(x))
        graphs.append((g, st))
    s["lens"].copy_(torch.tensor([1, 33, 50], dtype=torch.int32))
    r["lens"].copy_(torch.tensor([29, 77], dtype=torch.int32))
    torch.cuda.synchronize()
    for _ in range(10):
        for g, st in graphs:
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], call(s)) and torch.equal(outs[1], call(r))
    check(s, outs[0])
    check(r, outs[1])


def test_cache_beyond_32_bits():
    hk, page, d, pages = 8, 64, 128, 33000  # offsets beyond 2^31 elements
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    kc = torch.empty(pages, hk, page, d, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    kc[-3:].normal_()
    vc[-3:].normal_()
    q = torch.randn(40, 16, d, device="cuda").bfloat16()
    t = torch.full((40, 1), pages - 1, dtype=torch.int32, device="cuda")
    pp = torch.tensor([pages - 2, pages - 3], dtype=torch.int32, device="cuda")
    lens = torch.full((40,), 50, dtype=torch.int32, device="cuda")
    got = warp_route.shared_prefix_attention(q, kc, vc, t, lens, prefix_pages=pp, prefix_len=100)
    kc, vc = kc[-3:].clone(), vc[-3:].clone()
    want = warp_route.shared_prefix_attention(q, kc, vc, t - (pages - 3), lens, prefix_pages=pp - (pages - 3),
                                              prefix_len=100)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_own_pages_at_all(dtype):
    s = make([0] * 5, [1] * 5, 8, 2, 128, 16, 75, dtype)
    s["tables"] = s["tables"][:, :0]
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,c,prefix", [(1, 40, 500), (7, 7, 33), (50, 130, 700), (3, 1, 18)])
def test_one_sequence_with_several_tokens_behind_a_prefix(n, c, prefix, dtype):
    s = make([c], [n], 6, 2, 128, 16, prefix, dtype)
    if n == 1:
        s["q_start"] = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


def test_pages_that_several_sequences_name():
    """A page may stand in several tables, several times, and in the prefix."""
    s = make([64, 64, 30], [1, 1, 1], 8, 2, 128, 16, 64, torch.bfloat16, junk=0.5)
    s["tables"][1] = s["tables"][0]
    s["tables"][0, 2] = s["tables"][0, 1]
    s["prefix_pages"][3] = s["tables"][2, 0]
    s["prefix_pages"][1] = s["prefix_pages"][0]
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


def test_two_calls_at_once():
    a = make([700 + 90 * i for i in range(20)], [1] * 20, 16, 2, 128, 16, 3000, torch.bfloat16)
    b = make([50] * 300, [1] * 300, 32, 4, 128, 16, 2048, torch.bfloat16, seed=3)
    want = [call(a), call(b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(6):
        for i, (s, st) in enumerate(zip((a, b), streams)):
            with torch.cuda.stream(st):
                got[i].append(call(s))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_many_sequences():
    n = 3000
    s = make([(i * 7) % 20 for i in range(n)], [1] * n, 2, 1, 64, 16, 40, torch.bfloat16)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 256),
                                     (torch.float32, 64), (torch.float32, 128), (torch.float32, 256)])
@pytest.mark.parametrize("group", [1, 5, 8])
def test_many_tokens_of_many_sequences(group, dtype, d):
    """More rows than the warps of a launch could leave unfinished, with rows
    of no sequence behind them; most units lie behind some row's own key."""
    hk = 4 if d > 64 else 8
    n = 2 + 60000 // (hk * group * 30)
    nq = [(i * 13) % 61 for i in range(n)]
    lens = [c + (i * 7) % 40 if i % 9 else c // 2 for i, c in enumerate(nq)]
    s = make(lens, nq, hk * group, hk, d, 16, 0, dtype, seed=group)
    tail = torch.randn(9, hk * group, d, device="cuda").to(dtype)
    s["q"] = torch.cat([s["q"], tail])
    out, lse = call(s, return_lse=True)
    check(s, out, lse)
    assert not out[-9:].any() and (lse[-9:] == float("-inf")).all()
    again = call(s)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_sequences_of_many_tokens(dtype):
    """Tiles cut by several ranges, of which the first rows see only a part."""
    nq, lens = [700, 1, 300, 700], [700, 900, 2500, 650]
    s = make(lens, nq, 16, 2, 128, 16, 0, dtype)
    out, lse = call(s, return_lse=True)
    check(s, out, lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,group,prefix", [(64, 8, 0), (128, 4, 0), (256, 3, 0), (96, 1, 70), (128, 20, 300)])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_later_keys_that_are_not_finite(bad, d, group, prefix, dtype):
    """Keys and values of a sequence's last tokens: no row before them sees
    them, whatever they hold."""
    nq, lens = [1, 20, 7, 40, 33], [50, 20, 90, 47, 200]
    s = make(lens, nq, 2 * group, 2, d, 16, prefix, dtype)
    clean, lse = call(s, return_lse=True)
    check(s, clean, lse)
    hit = torch.zeros(sum(nq), dtype=torch.bool, device="cuda")
    starts = [sum(nq[:i]) for i in range(6)]
    # 3 late keys of each longer sequence: in the last unit, and one before it
    for b, back in ((1, 1), (2, 3), (3, 20), (4, 2)):
        for j in (lens[b] - back, lens[b] - 1):
            page = s["tables"][b, j // 16]
            s["k_cache"][page, :, j % 16] = bad
            s["v_cache"][page, :, j % 16, ::3] = bad
        hit[starts[b] + nq[b] - back:starts[b + 1]] = True
    out, got = call(s, return_lse=True)
    assert torch.isfinite(out[~hit]).all() and torch.isfinite(got[~hit]).all()
    # only the order of a unit's sums, and the rounding of its weights, differ
    tol = (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -14)
    assert ((out[~hit].double() - clean[~hit].double()).abs() <= tol * (1 + clean[~hit].double().abs())).all()
    assert torch.equal(got[~hit], lse[~hit])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_value_that_is_not_finite_reaches_who_sees_it(dtype):
    nq, lens = [20], [20]
    s = make(lens, nq, 4, 2, 128, 16, 0, dtype)
    s["v_cache"][s["tables"][0, 0], :, 9, 5] = float("inf")
    out = call(s)
    assert torch.isfinite(out[:9]).all()
    seen = out[9:, :, 5]
    assert (seen == float("inf")).all()
    rest = torch.ones(128, dtype=torch.bool, device="cuda")
    rest[5] = False
    assert torch.isfinite(out[:, :, rest]).all()
