"""GPU: sample_tokens against a 64-bit form, token by token.

The tokens have to be equal.  The kernel holds weights in whole numbers of
2^-45 of the largest, the reference in 64-bit floating point: with V values
their running sums differ by at most V * 2^-46, which moves a border past the
given number in a row with probability about 2 V * V * 2^-46 at most
(V = 50000: 7e-5) were all weights equal to the largest, and far less for
weights that fall off; the seeds are fixed, so a pass is a pass.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

import warp_route
from decode_reference import sample

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def _f(v, r):
    return float(v[r]) if isinstance(v, torch.Tensor) else float(np.float32(v))


def check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    ids = warp_route.sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert ids.dtype == torch.int64 and ids.shape == (logits.shape[0],)
    got = ids.cpu().numpy()
    x = logits.double().cpu().numpy()
    un = u.cpu().numpy()
    for r in range(x.shape[0]):
        k = int(top_k[r]) if isinstance(top_k, torch.Tensor) else top_k
        want = sample(x[r], un[r], _f(temperature, r), k, _f(top_p, r), _f(min_p, r))
        assert got[r] == want, (r, got[r], want, x[r].max())
    return ids


def rows(n, v, dtype=torch.float32, seed=0, spread=2.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = (torch.randn(n, v, generator=g, device="cuda") * spread).to(dtype)
    return x, torch.rand(n, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [1, 2, 5, 2047, 2048, 2049, 32000, 50001, 131072])
@pytest.mark.parametrize("kw", [
    dict(), dict(temperature=0.0), dict(temperature=0.3), dict(top_k=1), dict(top_k=7), dict(top_k=1000),
    dict(top_p=0.0), dict(top_p=0.5), dict(top_p=0.999), dict(min_p=0.05), dict(min_p=1.0),
    dict(temperature=1.7, top_k=50, top_p=0.9, min_p=0.01), dict(temperature=0.6, top_k=40000, top_p=0.97),
])
def test_matches_plain(v, kw, dtype):
    x, u = rows(5, v, dtype, seed=v)
    check(x, u, **kw)


@pytest.mark.parametrize("n", [1, 18, 19, 200])
def test_rows_with_settings_of_their_own(n):
    x, u = rows(n, 30011, seed=n)
    r = torch.arange(n, device="cuda")
    check(x, u, temperature=torch.where(r % 4 == 0, 0.0, 0.5 + (r % 5) / 4).float(),
          top_k=torch.where(r % 3 == 0, 0, r * 7 + 1).int(),
          top_p=torch.where(r % 2 == 0, 1.0, 0.05 + (r % 9) / 10).float(),
          min_p=torch.where(r % 5 == 1, 0.1, 0.0).float())


@pytest.mark.parametrize("u", [0.0, 1e-30, 0.25, 0.5, 1 - 2.0 ** -24])
def test_ends_of_the_uniform_numbers(u):
    x, _ = rows(3, 5003)
    check(x, torch.full((3,), u, device="cuda"))
    check(x, torch.full((3,), u, device="cuda"), top_p=0.7)


@pytest.mark.parametrize("kw", [dict(top_k=k) for k in (1, 2, 3, 2500, 4999, 5000)] +
                         [dict(top_p=p) for p in (0.0, 1e-4, 0.5, 0.7501, 1.0)] +
                         [dict(top_k=3000, top_p=0.3), dict(temperature=0.0), dict(min_p=1.0)])
def test_equal_values_go_by_index(kw):
    u = torch.tensor([0.0, 0.3, 0.77, 0.9999], device="cuda")
    check(torch.full((4, 5000), 1.25, device="cuda"), u, **kw)
    x = torch.zeros(4, 5000, device="cuda")
    x[:, ::3] = 2.0   # two values, each many times
    x[:, 1] = -0.0
    check(x, u, **kw)


def test_ties_across_the_border_of_a_large_row():
    x, u = rows(4, 100000, torch.bfloat16, seed=3)
    for k in (10, 100, 1000, 30000):
        check(x, u, top_k=k)
    for p in (0.1, 0.6, 0.95):
        check(x, u, top_p=p)
    check((x.float() / 4).round().bfloat16(), u, top_k=777, top_p=0.8)


def test_top_p_stays_within_what_top_k_cut():
    """Equal values across the border of top_k: top_p must not bring back the
    ones that top_k cut off, whichever of its ways it takes."""
    u = torch.tensor([0.0, 0.4, 0.6, 0.9999], device="cuda")
    for v in (300, 5000, 50000):
        x, _ = rows(4, v, torch.bfloat16, seed=v)
        x[:, 11::v // 7] = 12.5
        for k in (1, 2, 5):
            for p in (0.1, 0.5, 0.99):
                check(x, u, top_k=k, top_p=p)
        x[:, ::2] = 13.0  # more equal ones than are sorted
        for k in (1, 20, v // 3):
            check(x, u, top_k=k, top_p=0.9)


def test_infinities_and_nan():
    inf, nan = float("inf"), float("nan")
    x, u = rows(6, 3001)
    x[0] = -inf                      # nothing to sample
    x[1, 100:] = -inf
    x[2, ::2] = nan
    x[3, 7] = inf
    x[3, 2000] = inf                 # these two alone, evenly
    x[4] = nan
    x[5, :3000] = -inf               # one value left
    for kw in (dict(), dict(top_k=50), dict(top_p=0.9), dict(temperature=0.0), dict(top_k=500, top_p=0.5, min_p=0.1)):
        ids = check(x, u, **kw)
        assert ids[0] == -1 and ids[4] == -1 and ids[5] == 3000
    lowest = torch.full((2, 40), torch.finfo(torch.float32).min, device="cuda")
    lowest[1, 5] = torch.finfo(torch.float32).max
    check(lowest, u[:2])
    check(lowest, u[:2], top_p=0.5)
    check(lowest, u[:2], top_k=30, top_p=0.5)


def test_strided_and_unaligned_rows():
    x, u = rows(4, 4003)
    base = torch.zeros(4, 4100, device="cuda")
    for off in (0, 1, 4):
        v = base[:, off:off + 4003]
        v.copy_(x)
        check(v, u, top_k=20)
    b = base.bfloat16()[:, 3:3 + 4003]
    check(b, u, top_p=0.8)
    check(x[:1].expand(4, -1), u)


def test_largest_vocabulary_and_no_rows():
    x, u = rows(2, 262144, seed=9)
    check(x, u, top_p=0.9)
    check(x, u, top_k=5000)
    assert warp_route.sample_tokens(x[:0], u[:0]).shape == (0,)


def test_in_a_graph():
    x, u = rows(3, 20000)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ids = warp_route.sample_tokens(x, u, top_k=40, top_p=0.9)
    for seed in (1, 2):
        y, w = rows(3, 20000, seed=seed)
        x.copy_(y)
        u.copy_(w)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids, check(y, w, top_k=40, top_p=0.9))


def test_frequencies_follow_the_probabilities():
    """65536 evenly spaced numbers hit each kept token as often as its share
    says, to within one (sums of shares move each end by at most one)."""
    n = 65536
    x = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5, -3.0], device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    ids = warp_route.sample_tokens(x.expand(n, -1), u, top_k=5)
    share = torch.softmax(torch.where(x == -3.0, float("-inf"), x).double(), 0)
    count = torch.bincount(ids, minlength=6).double()
    assert ((count - share * n).abs() <= 1.0 + 1e-6).all()


def test_two_calls_at_once_and_again():
    a, ua = rows(64, 60000, torch.bfloat16, seed=1)
    b, ub = rows(7, 131072, seed=2)
    want = [warp_route.sample_tokens(a, ua, top_p=0.9), warp_route.sample_tokens(b, ub, top_k=60, top_p=0.8)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(8):
        with torch.cuda.stream(streams[0]):
            got.append((0, warp_route.sample_tokens(a, ua, top_p=0.9)))
        with torch.cuda.stream(streams[1]):
            got.append((1, warp_route.sample_tokens(b, ub, top_k=60, top_p=0.8)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i, g in got)


def test_many_rows():
    x, u = rows(5000, 300, seed=8)
    check(x, u, top_k=30, top_p=0.9)


@pytest.mark.parametrize("shift", [-1e6, -3000.0, 3000.0, 1e6])
def test_logits_far_from_zero(shift):
    """Only differences count: far from zero they are coarse, not wrong."""
    x, u = rows(4, 20000, seed=4)
    check(x + shift, u, top_p=0.9)
    check(x + shift, u, top_k=77)
    check((x + shift), u, temperature=0.7, min_p=0.02)


@pytest.mark.parametrize("t", [1e-30, 1e-3, 50.0, 1e30, float("inf")])
def test_extreme_temperatures(t):
    x, u = rows(4, 20000, seed=5)
    check(x, u, temperature=t)
    check(x, u, temperature=t, top_k=100, top_p=0.7)
    check(x, u, temperature=t, top_p=0.7)


def _edge_rows(dtype):
    """Rows with a value just inside a bin's end: 1024 even bins over the
    row's span R have their first edge at R / 1024 below the maximum, and the
    product (max - x) * (1024 / R) comes out as 1 - 2^-24 for some of them."""
    kept = []
    for n in range(1, 4000):
        span = np.float32(n / 8)
        x = np.float32(-n / 8192)
        y = np.float32(-x) * np.float32(np.float32(1024) / span)
        if y == np.nextafter(np.float32(1), np.float32(0)):
            r = torch.tensor([0.0, float(x), -float(span)])
            if torch.equal(r.to(dtype).float(), r):
                kept.append(r)
    return torch.stack(kept).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_at_the_end_of_a_bin(dtype):
    """Every pass of top_p has to put such a value into the same bin."""
    x = _edge_rows(dtype)
    assert x.shape[0] >= (500 if dtype == torch.float32 else 20)
    assert (x.float() == torch.tensor([0.0, -41 / 8192, -5.125], device="cuda")).all(1).any()
    for u in (0.0, 0.3, 0.7, 1 - 2.0 ** -24):
        uu = torch.full((x.shape[0],), u, device="cuda")
        for p in (0.3, 0.5, 0.6, 0.9):
            check(x, uu, top_p=p)
    check(x, uu, top_p=0.6, top_k=2)


@pytest.mark.parametrize("v", [700, 6000, 40000])
def test_values_at_the_end_of_a_bin_before_a_full_one(v):
    """The next bin holds few values, more than one CTA sorts, or most of the row."""
    u = torch.tensor([0.0, 0.31, 0.68, 1 - 2.0 ** -24], device="cuda")
    x = torch.full((4, v), -5.125, device="cuda")
    for i in range(4):
        g = torch.Generator(device="cuda").manual_seed(i)
        at = torch.randperm(v, generator=g, device="cuda")
        x[i, at[:2]] = torch.tensor([0.0, -41 / 8192], device="cuda")
        # from the second bin's first value to its last
        n = v // 2
        x[i, at[2:2 + n]] = -(41 / 8192) * (1.01 + 0.98 * torch.arange(n, device="cuda") / n)
    for p in (0.5 / v, 1.5 / v, 2.5 / v, 0.2, 0.5, 0.97, 0.999):
        check(x, u, top_p=p)
    check(x.bfloat16(), u, top_p=0.4)
    check(x, u, top_p=0.4, top_k=v // 3)


@pytest.mark.parametrize("kw", [dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.4), dict(top_k=900, top_p=0.9)])
@pytest.mark.parametrize("t", [1e36, 1e38, float("inf")])
def test_the_largest_finite_logits(t, kw):
    """Only an infinite maximum leaves the finite values without weight."""
    big = torch.finfo(torch.float32).max
    x = big * (1 - torch.rand(6, 1000, device="cuda", generator=torch.Generator("cuda").manual_seed(1)) / 100)
    x[:, 17] = big
    x[1, ::2] = -big  # a span beyond the type
    x[2, 3] = float("inf")
    u = torch.tensor([0.1, 0.3, 0.5, 0.7, 0.9, 0.99], device="cuda")
    check(x, u, temperature=t, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masks_of_the_lowest_value(dtype):
    """Masked logits are the type's lowest finite value: all others share one
    of the even bins, and masked ones only come in where nothing else is left."""
    x, u = rows(5, 30000, dtype, seed=2)
    low = torch.finfo(dtype).min
    x[0, ::2] = low
    x[1, 40:] = low
    x[2, :-3] = low
    x[3] = low
    for kw in (dict(), dict(top_k=7), dict(top_k=20000), dict(top_p=0.8), dict(top_k=5000, top_p=0.3),
               dict(top_p=0.9, temperature=2.5), dict(min_p=0.1), dict(temperature=0.0)):
        ids = check(x, u, **kw)
        if kw.get("top_k") != 20000:
            assert ids[1] < 40 and ids[2] >= 30000 - 3
