"""Argument checks of the packed-set operators without a GPU. The checks come before any device
call, so a host program with a context of its own reaches every refusal (and every call that has
nothing to do) on the CPU; the Python wrappers refuse tensors before they reach the library."""
import os
import shutil
import subprocess

import pytest
import torch

from conftest import ROOT

PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <cstring>
#include "tb_common.cuh"

static int failed = 0;
static tb_ctx ctx;
static void want(const char* what, tb_status got, tb_status exp) {
    if (got != exp) { std::printf("%s: got %d, want %d (%s)\n", what, (int)got, (int)exp, ctx.last_error.c_str()); failed = 1; }
}
alignas(16) static char mem[256];
// addresses that nothing reads: the arrays are 1 MB apart
static char* at(int i, int more = 0) { return reinterpret_cast<char*>((intptr_t)(i + 1) << 20) + more; }

static tb_attention_params attn() {
    tb_attention_params p;
    std::memset(&p, 0, sizeof p);
    p.q = at(0); p.k = at(1); p.v = at(2); p.out = at(3);
    p.q_offsets = p.k_offsets = (const int32_t*)mem;
    p.nq = 10; p.nk = 20; p.nset = 2; p.heads = 4; p.kv_heads = 2; p.head_dim = 64;
    p.q_row = p.out_row = 256; p.k_row = p.v_row = 128; p.q_head = p.k_head = p.v_head = p.out_head = 64;
    p.scale = 0.125f; p.dtype = TB_BF16; p.out_dtype = TB_BF16;
    return p;
}
static tb_rope_params rope() {
    tb_rope_params p;
    std::memset(&p, 0, sizeof p);
    p.x = at(0); p.out = at(1); p.coords = (const int32_t*)mem; p.n = 10;
    p.x_row = p.out_row = 256; p.x_head = p.out_head = 64; p.coord_stride = 4; p.axes = 3;
    p.sections[0] = p.sections[1] = p.sections[2] = 10;
    p.heads = 4; p.head_dim = 64; p.theta = 1e4; p.dtype = TB_BF16;
    return p;
}
#define ATTN(change, exp) do { tb_attention_params p = attn(); change; want(#change, tb_attention(&ctx, &p), exp); } while (0)
#define ROPE(change, exp) do { tb_rope_params p = rope(); change; want(#change, tb_rope(&ctx, &p), exp); } while (0)

int main() {
    want("null context", tb_attention(nullptr, nullptr), TB_ERR_INVALID_ARG);
    want("null parameters", tb_attention(&ctx, nullptr), TB_ERR_INVALID_ARG);
    ATTN(p.nq = 0, TB_OK);
    ATTN(p.nset = 0, TB_OK);
    ATTN(p.dtype = (tb_dtype)9, TB_ERR_INVALID_ARG);
    ATTN(p.out_dtype = TB_F16, TB_ERR_UNSUPPORTED);
    ATTN(p.nq = -1, TB_ERR_INVALID_ARG);
    ATTN(p.nk = -1, TB_ERR_INVALID_ARG);
    ATTN(p.heads = 0, TB_ERR_INVALID_ARG);
    ATTN(p.heads = 3, TB_ERR_INVALID_ARG);
    ATTN(p.kv_heads = 0, TB_ERR_INVALID_ARG);
    ATTN(p.heads = 130, TB_ERR_UNSUPPORTED);
    ATTN(p.head_dim = 60, TB_ERR_UNSUPPORTED);
    ATTN(p.head_dim = 136, TB_ERR_UNSUPPORTED);
    ATTN(p.head_dim = 0, TB_ERR_UNSUPPORTED);
    ATTN(p.nset = -1, TB_ERR_INVALID_ARG);
    ATTN(p.k_offsets = nullptr, TB_ERR_INVALID_ARG);
    ATTN((p.k_offsets = p.q_offsets = nullptr), TB_ERR_INVALID_ARG);
    ATTN(p.nset = 65537, TB_ERR_TOO_LARGE);
    ATTN(p.nk = (int64_t)1 << 31, TB_ERR_TOO_LARGE);
    ATTN(p.scale = 0.f, TB_ERR_INVALID_ARG);
    ATTN(p.scale = -1.f, TB_ERR_INVALID_ARG);
    ATTN(p.scale = NAN, TB_ERR_INVALID_ARG);
    ATTN(p.scale = INFINITY, TB_ERR_INVALID_ARG);
    ATTN(p.q_row = 0, TB_ERR_INVALID_ARG);
    ATTN(p.k_row = -128, TB_ERR_INVALID_ARG);
    ATTN(p.v_head = 60, TB_ERR_INVALID_ARG);
    ATTN(p.out_row = 128, TB_ERR_INVALID_ARG);
    ATTN(p.out_head = 32, TB_ERR_INVALID_ARG);
    ATTN(p.q = nullptr, TB_ERR_INVALID_ARG);
    ATTN(p.v = nullptr, TB_ERR_INVALID_ARG);
    ATTN(p.out = nullptr, TB_ERR_INVALID_ARG);
    ATTN(p.k = mem + 8, TB_ERR_INVALID_ARG);
    ATTN(p.out = (void*)p.q, TB_ERR_INVALID_ARG);
    ATTN(p.out = at(0, 512 * 9), TB_ERR_INVALID_ARG);                       // q's last row
    ATTN(p.out = at(0, -512 * 9 - 496), TB_ERR_INVALID_ARG);                // out's last row ends in q's first
    ATTN((p.k_row = p.v_row = 256, p.out = at(2, 512 + 240)), TB_ERR_INVALID_ARG);   // into v's head 1
    ATTN(p.scale = 3e38f, TB_ERR_INVALID_ARG);

    want("null context", tb_rope(nullptr, nullptr), TB_ERR_INVALID_ARG);
    want("null parameters", tb_rope(&ctx, nullptr), TB_ERR_INVALID_ARG);
    ROPE(p.n = 0, TB_OK);
    ROPE(p.n = -1, TB_ERR_INVALID_ARG);
    ROPE(p.heads = 0, TB_ERR_INVALID_ARG);
    ROPE(p.dtype = (tb_dtype)7, TB_ERR_INVALID_ARG);
    ROPE(p.head_dim = 60, TB_ERR_UNSUPPORTED);
    ROPE(p.head_dim = 264, TB_ERR_UNSUPPORTED);
    ROPE(p.layout = (tb_rope_layout)2, TB_ERR_INVALID_ARG);
    ROPE(p.freqs = (tb_rope_freqs)2, TB_ERR_INVALID_ARG);
    ROPE(p.axes = 0, TB_ERR_INVALID_ARG);
    ROPE(p.axes = 5, TB_ERR_INVALID_ARG);
    ROPE(p.coord_stride = 2, TB_ERR_INVALID_ARG);
    ROPE(p.theta = 0, TB_ERR_INVALID_ARG);
    ROPE(p.theta = NAN, TB_ERR_INVALID_ARG);
    ROPE(p.sections[1] = 0, TB_ERR_INVALID_ARG);
    ROPE(p.sections[1] = 13, TB_ERR_INVALID_ARG);
    ROPE(p.sections[1] = INT32_MAX, TB_ERR_INVALID_ARG);
    ROPE(p.x = nullptr, TB_ERR_INVALID_ARG);
    ROPE(p.x = mem + 4, TB_ERR_INVALID_ARG);
    ROPE(p.x_row = 260, TB_ERR_INVALID_ARG);
    ROPE(p.out_row = 192, TB_ERR_INVALID_ARG);
    ROPE((p.out = (void*)p.x, p.out_row = 512), TB_ERR_INVALID_ARG);
    ROPE(p.n = (int64_t)1 << 31, TB_ERR_TOO_LARGE);
    ROPE(p.out = at(0, 512), TB_ERR_INVALID_ARG);                           // one row on
    ROPE((p.n = 1, p.out = at(0, 16)), TB_ERR_INVALID_ARG);
    want("rows side by side", tb_rows_overlap({at(0), 10, 512, 256}, {at(0, 256), 10, 512, 256}) ? TB_ERR_INVALID_ARG : TB_OK, TB_OK);
    want("rows behind", tb_rows_overlap({at(0), 10, 512, 512}, {at(0, 5120), 10, 512, 512}) ? TB_ERR_INVALID_ARG : TB_OK, TB_OK);
    want("rows before", tb_rows_overlap({at(0, 5120), 10, 512, 512}, {at(0), 10, 512, 512}) ? TB_ERR_INVALID_ARG : TB_OK, TB_OK);
    want("columns meet", tb_rows_overlap({at(0), 10, 512, 272}, {at(0, 256), 10, 512, 256}) ? TB_OK : TB_ERR_INVALID_ARG, TB_OK);
    want("row past the edge", tb_rows_overlap({at(0, 512), 1, 0, 256}, {at(0, 272), 2, 512, 256}) ? TB_OK : TB_ERR_INVALID_ARG, TB_OK);

    const size_t need = tb_group_norm_workspace_bytes(&ctx, 10000, 32, 4, 1);
    auto gn = [&](const void* x, tb_dtype dt, const int32_t* off, int nset, int64_t n, int c, int groups, float eps, int act,
                  tb_dtype od, void* out, void* ws, size_t wb) {
        return tb_group_norm(&ctx, x, dt, off, nset, n, c, groups, nullptr, nullptr, eps, (tb_epilogue)act, od, out, ws, wb);
    };
    const int32_t* off = (const int32_t*)mem;
    void* out = at(5);
    want("gn no rows", gn(mem, TB_F32, off, 1, 0, 32, 4, 1e-5f, 0, TB_F32, out, nullptr, 0), TB_OK);
    want("gn no sets", gn(mem, TB_F32, off, 0, 100, 32, 4, 1e-5f, 0, TB_F32, out, nullptr, 0), TB_OK);
    want("gn dtype", gn(mem, (tb_dtype)5, off, 1, 100, 32, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn out dtype", gn(mem, TB_F16, off, 1, 100, 32, 4, 1e-5f, 0, TB_BF16, out, mem, need), TB_ERR_UNSUPPORTED);
    want("gn c", gn(mem, TB_F32, off, 1, 100, 20, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn wide", gn(mem, TB_F32, off, 1, 100, 4096, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn groups", gn(mem, TB_F32, off, 1, 100, 32, 5, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn no groups", gn(mem, TB_F32, off, 1, 100, 32, 0, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn sets without a table", gn(mem, TB_F32, nullptr, 2, 100, 32, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn act", gn(mem, TB_F32, off, 1, 100, 32, 4, 1e-5f, 3, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn eps", gn(mem, TB_F32, off, 1, 100, 32, 4, -1.f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn eps nan", gn(mem, TB_F32, off, 1, 100, 32, 4, NAN, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn too many sets", gn(mem, TB_F32, off, 65537, 100, 32, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_TOO_LARGE);
    want("gn null", gn(nullptr, TB_F32, off, 1, 100, 32, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn alignment", gn(mem + 4, TB_F32, off, 1, 100, 32, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn in place", gn(mem, TB_F16, off, 1, 100, 32, 4, 1e-5f, 0, TB_F32, mem, mem, need), TB_ERR_INVALID_ARG);
    want("gn overlap", gn(at(5, 64), TB_F32, off, 1, 100, 32, 4, 1e-5f, 0, TB_F32, out, mem, need), TB_ERR_INVALID_ARG);
    want("gn workspace", gn(mem, TB_F32, off, 1, 10000, 32, 4, 1e-5f, 0, TB_F32, out, nullptr, 0), TB_ERR_INVALID_ARG);
    want("gn small workspace", gn(mem, TB_F32, off, 1, 10000, 32, 4, 1e-5f, 0, TB_F32, out, mem, need - 1), TB_ERR_INVALID_ARG);
    std::printf(failed ? "failed\n" : "refusals ok\n");
    return failed;
}
"""


def test_refusals_of_the_library(tb, tmp_path):
    from trellis_cpp_b200 import _lib, build
    if not os.path.exists(build.NVCC) and not shutil.which(build.NVCC):
        pytest.skip("nvcc not found")
    libdir = os.path.dirname(_lib.LIB_PATH)
    (tmp_path / "refuse.cu").write_text(PROGRAM)
    b = subprocess.run([build.NVCC, "-std=c++17", "-I", os.path.join(ROOT, "include"), "-I", build.CSRC,
                        str(tmp_path / "refuse.cu"), "-o", str(tmp_path / "refuse"), "-L", libdir, "-ltb_sparse",
                        "-Xlinker", "-rpath=" + libdir], capture_output=True, text=True)
    assert b.returncode == 0, b.stderr
    r = subprocess.run([str(tmp_path / "refuse")], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "refusals ok" in r.stdout, r.stdout + r.stderr


def test_wrappers_refuse_host_tensors(tb):
    from trellis_cpp_b200 import ops
    q = torch.zeros((4, 2, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ops.attention(q, q, q)
    with pytest.raises(ValueError):
        ops.rope(q, torch.zeros((4, 3), dtype=torch.int32), (10, 10, 10))
    with pytest.raises(ValueError):
        ops.group_norm(q.view(4, 128), 8)
