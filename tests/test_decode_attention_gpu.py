"""GPU: the decode stack with attention in front of its MoE layers, the cache
it fills, and tokens sampled from its output, run together as a decode loop
would: a prompt shared by all sequences enters the cache, then every sequence
goes on from it with its own tokens.
"""
from __future__ import annotations

import pytest
import torch

import warp_route
from decode_reference import attention, rotate
from warp_route import synthetic
from warp_route.decode import MoEStack, StackAttention, StackContext, StackLayer

pytestmark = pytest.mark.gpu

HQ, HK, D, PAGE = 8, 2, 64, 16


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")


def build(tokens, dtype, layers=2, prefix=37, pages=40, seed=5):
    E, H, I, K = synthetic.SHAPES["tiny"]
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    inv = (1e4 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)).float()
    ls = []
    for i in range(layers):
        L = synthetic.make_layer(E, H, I, K, dtype=dtype, seed=seed + i, device="cuda")
        a = StackAttention(normal((HQ + 2 * HK) * D, H, std=H ** -0.5), normal(H, HQ * D, std=(HQ * D) ** -0.5), HQ, HK,
                           normal(pages, HK, PAGE, D, std=1), normal(pages, HK, PAGE, D, std=1), inv)
        a.k_cache.fill_(float("nan"))  # nothing has been written yet
        a.v_cache.fill_(float("nan"))
        ls.append(StackLayer(L.gate_w, L.weight_buf, attention=a))
    shared = -(-prefix // PAGE)
    ctx = StackContext.empty(tokens, 4, "cuda", torch.arange(shared, dtype=torch.int32, device="cuda") + 3, prefix)
    head = normal(1000, H, std=H ** -0.5)
    stack = MoEStack(ls, E, H, I, K, tokens, context=ctx, head=head)
    # the shared prompt: its keys and values into every layer's cache
    slots = torch.arange(prefix, device="cuda") + 3 * PAGE
    pos = torch.arange(prefix, device="cuda")
    for L in ls:
        kv = normal(prefix, 2 * HK, D, std=1)
        warp_route.append_paged_kv(kv[:, :HK], kv[:, HK:], L.attention.k_cache, L.attention.v_cache, slots,
                                   positions=pos, inv_freq=inv)
    own = torch.arange(tokens * 4, dtype=torch.int32, device="cuda").view(tokens, 4) + 3 + shared
    ctx.block_tables.copy_(own)
    return stack, normal, H


def advance(ctx, n):
    """Context of every sequence's n-th own token (from 0)."""
    T = ctx.slots.shape[0]
    page = ctx.block_tables[:, n // PAGE].long()
    ctx.slots.copy_(page * PAGE + n % PAGE)
    ctx.positions.fill_(ctx.prefix_len + n)
    ctx.context_lens.fill_(n + 1)
    if T > 2:  # one sequence has ended: padding
        ctx.slots[T - 1] = -1
        ctx.context_lens[T - 1] = 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens", [1, 5])
def test_decode_loop(tokens, dtype):
    stack, normal, H = build(tokens, dtype)
    A, ctx = stack.layers[0].attention, stack.context
    embed = normal(1000, H, std=1)
    x = normal(tokens, H, std=1)
    stack.capture()
    keys = torch.isfinite(A.k_cache).all(-1).sum().item()
    assert keys == 37 * HK  # capturing with no sequence taking part writes nothing
    for n in range(20):  # beyond a page
        advance(ctx, n)
        before = A.k_cache.clone()
        xs = x.view(stack.x_in.shape)
        # layer 0's attention on its own, from the operators' parts
        qkv = torch.nn.functional.linear(x, A.wqkv).view(tokens, -1, D)
        out = stack.step(xs).clone()
        torch.cuda.synchronize()
        live = ctx.slots >= 0
        at = ctx.slots[live]
        want = rotate(qkv[:, HQ:HQ + HK], ctx.positions, A.inv_freq, False)[live]
        got = A.k_cache[at // PAGE, :, at % PAGE].double()
        # one rounding and the angle's own error, see test_kvcache_gpu
        u = torch.finfo(dtype).eps / 2
        size = qkv.double().abs().amax() * 2
        assert ((got - want).abs() <= u * want.abs() + size * 2.0 ** -20).all()
        before[at // PAGE, :, at % PAGE] = A.k_cache[at // PAGE, :, at % PAGE]
        assert torch.equal(torch.nan_to_num(before), torch.nan_to_num(A.k_cache))
        # the graph's step is the eager one, which is the layers' composition
        assert torch.equal(stack.eager(xs), out)
        h = xs
        for i in range(len(stack.layers)):
            h = stack.attention(i, h)
            nxt = torch.empty_like(h)
            stack.layer(i, h, nxt)
            h = nxt
        assert torch.equal(h, out) and torch.isfinite(out).all()
        # attention against the cache's content in 64 bits (its bound, see
        # test_attention_gpu, is below 2^-7 of the largest value here in bf16)
        q = rotate(qkv[:, :HQ], ctx.positions, A.inv_freq, False).to(dtype)
        ref, _, mass, _ = attention(q, A.k_cache, A.v_cache, ctx.block_tables, ctx.context_lens, ctx.prefix_pages,
                                    ctx.prefix_len, None, D ** -0.5)
        mine = warp_route.shared_prefix_attention(q, A.k_cache, A.v_cache, ctx.block_tables, ctx.context_lens,
                                                  prefix_pages=ctx.prefix_pages, prefix_len=ctx.prefix_len)
        tol = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -14
        assert ((mine.double() - ref).abs() <= tol * mass + 1e-6).all()
        u01 = torch.rand(tokens, device="cuda").clamp(max=1 - 2.0 ** -24)
        ids = stack.sample(out, u01, temperature=0.8, top_k=20, top_p=0.9)
        logits = torch.nn.functional.linear(out.view(tokens, H), stack.head)
        kept = logits.topk(20, 1).values[:, -1]
        picked = logits.gather(1, ids[:, None])[:, 0]
        assert (picked >= kept).all() and ((ids >= 0) & (ids < 1000)).all()
        x = embed[ids].contiguous()
    stack.close()


def test_stack_without_attention_is_as_before():
    E, H, I, K = synthetic.SHAPES["tiny"]
    L = synthetic.make_layer(E, H, I, K, dtype=torch.bfloat16, seed=1, device="cuda")
    x = torch.randn(4, H, device="cuda").bfloat16()
    stack = MoEStack([StackLayer(L.gate_w, L.weight_buf)], E, H, I, K, 4)
    nxt = torch.empty_like(x)
    warp_route.moe_decode_layer(x, L.gate_w, L.weight_buf, E, H, I, K, next_x=nxt)
    assert torch.equal(stack.step(x), nxt)
    with pytest.raises(ValueError, match="head"):
        stack.sample(nxt, torch.rand(4, device="cuda"))
    stack.close()


def test_attention_without_a_context_is_refused():
    stack, _, _ = build(2, torch.bfloat16, layers=1)
    with pytest.raises(ValueError, match="context"):
        MoEStack(stack.layers, stack.E, stack.H, stack.I, stack.K, 2)
    with pytest.raises(ValueError, match="tokens"):
        MoEStack(stack.layers, stack.E, stack.H, stack.I, stack.K, 3, context=stack.context)


def test_a_captured_step_refuses_another_prefix_or_context():
    """The graph holds prefix_len by value and the tensors by address: a step
    with others must not run on the old ones."""
    stack, normal, H = build(3, torch.bfloat16, prefix=37)
    ctx, A = stack.context, stack.layers[1].attention
    x = normal(3, H, std=1)
    advance(ctx, 0)
    first = stack.step(x).clone()
    ctx.prefix_len = 20
    with pytest.raises(ValueError, match="prefix_len"):
        stack.step(x)
    ctx.prefix_len = 37
    assert torch.equal(stack.step(x), first)
    for field in ("slots", "positions", "context_lens", "block_tables", "prefix_pages"):
        old = getattr(ctx, field)
        setattr(ctx, field, old.clone())
        with pytest.raises(ValueError, match="in place"):
            stack.step(x)
        setattr(ctx, field, old)
    caches = A.k_cache, A.v_cache
    A.k_cache = A.k_cache.clone()
    with pytest.raises(ValueError, match="caches"):
        stack.step(x)
    A.k_cache = caches[0]
    assert torch.equal(stack.step(x), first)
    # released, it captures the new prefix
    stack.close()
    ctx.prefix_len = 20
    ctx.slots = ctx.slots.clone()
    shorter = stack.step(x).clone()
    assert torch.equal(shorter, stack.eager(x)) and not torch.equal(shorter, first)
    stack.close()


def test_capture_writes_no_cache():
    """The warm-up runs on whatever input is there: it must not reach slots
    that the context already names."""
    stack, normal, H = build(3, torch.bfloat16)
    x = normal(3, H, std=1)
    advance(stack.context, 0)
    stack.eager(x)
    stack.x_in.zero_()  # as another step's input would be
    slots = stack.context.slots.clone()
    before = [t.clone() for L in stack.layers for t in (L.attention.k_cache, L.attention.v_cache)]
    stack.capture()
    torch.cuda.synchronize()
    after = [t for L in stack.layers for t in (L.attention.k_cache, L.attention.v_cache)]
    assert all(torch.equal(torch.nan_to_num(a), torch.nan_to_num(b)) for a, b in zip(after, before))
    assert torch.equal(stack.context.slots, slots)
    assert torch.equal(stack.step(x), stack.eager(x))
    stack.close()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_the_stack_samples_the_plain_forms_tokens(dtype):
    from decode_reference import sample

    stack, normal, H = build(4, dtype)
    for n in range(6):
        advance(stack.context, n)
        out = stack.step(normal(4, H, std=1))
        u = torch.rand(4, device="cuda", generator=torch.Generator("cuda").manual_seed(n))
        for kw in (dict(), dict(temperature=0.8, top_k=20, top_p=0.9), dict(top_p=0.5, min_p=0.02)):
            ids = stack.sample(out, u, **kw)
            logits = torch.nn.functional.linear(out.view(4, H), stack.head).double().cpu().numpy()
            full = dict(dict(temperature=1.0, top_k=0, top_p=1.0, min_p=0.0), **kw)
            full = {k: v if k == "top_k" else float(torch.tensor(v)) for k, v in full.items()}
            assert ids.tolist() == [sample(logits[r], u[r].item(), **full) for r in range(4)]
    stack.close()
