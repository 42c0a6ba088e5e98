"""GPU: waits of the prefix's tensor-core kernel that run out.

The library is linked once more, with that kernel built so that each wait that
its work hangs on gives up at once (the waits for copies and products still in
flight keep their whole limit).  A call must then end by itself with NaN in
every row that the prefix belongs to, and leave the GPU as it was: the same
call of the usual library gives the same result before and after.  Nothing
faults or hangs: no wait is endless, and no product is issued without its
operands.
"""
from __future__ import annotations

import ctypes
import os
import subprocess

import pytest
import torch

import build as wr_build
from warp_route import _abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def gives_up(tmp_path_factory):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    d = tmp_path_factory.mktemp("give_up")

    def compiled(source, *flags):
        obj = str(d / (source + ".o"))
        subprocess.run([wr_build.NVCC] + wr_build.NVCC_FLAGS + [*flags, "-c", os.path.join(wr_build.CSRC, source),
                                                                "-o", obj], check=True)
        return obj

    objs = []
    for source in wr_build.KERNEL_SOURCES:  # the usual library's objects, but for one
        usual = os.path.join(wr_build.OBJ_DIR, source + ".o")
        if source == "wr_attn_prefix.cu":
            objs.append(compiled(source, "-DWR_PREFIX_WAIT_NS=0"))
        else:
            objs.append(usual if os.path.exists(usual) else compiled(source))
    lib = str(d / "libgive_up.so")
    subprocess.run([wr_build.NVCC] + wr_build.ARCH + ["-shared", "-o", lib] + objs + ["-lcudart"], check=True)
    return _abi.load(lib)


def call(lib, q, kc, vc, tables, lens, pages, prefix):
    T, hq, d = q.shape
    p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
    cache = _abi.PagedKv(kc.data_ptr(), vc.data_ptr(), kc.stride(0), kc.stride(1), kc.stride(2), kc.shape[0],
                         kc.shape[1], kc.shape[2], d, _abi.WR_DTYPE_BF16, 0)
    desc = _abi.AttnDesc(T, T, hq, tables.shape[1], tables.stride(0), prefix, d ** -0.5)
    rows = _abi.Rows(q.data_ptr(), q.stride(0), q.stride(1))
    need = lib.wr_shared_prefix_attention_workspace_size(ctypes.byref(cache), ctypes.byref(desc), 0)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    lse = torch.zeros(T, hq, device="cuda")
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    st = lib.wr_shared_prefix_attention(ctypes.byref(cache), ctypes.byref(desc), ctypes.byref(rows), p(tables),
                                        p(lens), None, p(pages), p(out), p(lse), p(ws), need, stream)
    assert st == _abi.WR_OK, lib.wr_last_error_string()
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("n,hq,hk,d,page,prefix", [
    (40, 64, 8, 128, 16, 1600),   # two row tiles a CTA
    (16, 32, 8, 128, 64, 5003),   # one; a prefix that ends inside a page
    (60, 16, 8, 64, 64, 9000),    # heads of 64, more stages
])
def test_waits_that_run_out(gives_up, n, hq, hk, d, page, prefix):
    g = torch.Generator(device="cuda").manual_seed(n)
    pages = -(-prefix // page)
    kc = torch.randn(pages + n, hk, page, d, generator=g, device="cuda").bfloat16()
    vc = torch.randn(pages + n, hk, page, d, generator=g, device="cuda").bfloat16()
    q = torch.randn(n, hq, d, generator=g, device="cuda").bfloat16()
    tables = (pages + torch.arange(n, dtype=torch.int32, device="cuda"))[:, None].contiguous()
    lens = torch.full((n,), 9, dtype=torch.int32, device="cuda")
    pp = torch.arange(pages, dtype=torch.int32, device="cuda")
    args = (q, kc, vc, tables, lens, pp, prefix)
    usual = _abi.load()
    before, lse = call(usual, *args)
    assert torch.isfinite(before).all() and torch.isfinite(lse).all()
    for _ in range(3):
        out, s = call(gives_up, *args)
        assert torch.isnan(out).all() and torch.isnan(s).all()
    after, again = call(usual, *args)
    assert torch.equal(before, after) and torch.equal(lse, again)
