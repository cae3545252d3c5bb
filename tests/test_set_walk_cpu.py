"""The walk over packed sets that finds the attention kernel's tiles, on the CPU: the header's own
code on 32 threads with the warp's exchanges as barriers, for numbers that rise, fall and come in any
order, against a plain list of the pieces. The order in which a running CTA is given further tiles is
not promised to rise."""
import shutil
import subprocess

import pytest

PROGRAM = r"""
#include <algorithm>
#include <barrier>
#include <cstdint>
#include <cstdio>
#include <random>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
enum { TB_DEVERR_BAD_OFFSETS = 4 };
static std::barrier<> meet(32);
static thread_local int lane_;
static uint64_t slot[32];
static uint64_t exchange(uint64_t v, int from) {
    slot[lane_] = v;
    meet.arrive_and_wait();
    const uint64_t y = slot[from];
    meet.arrive_and_wait();
    return y;
}
template <class T> T __shfl_sync(unsigned, T v, int src) { return (T)exchange((uint64_t)v, src); }
template <class T> T __shfl_up_sync(unsigned, T v, int d) { return (T)exchange((uint64_t)v, lane_ >= d ? lane_ - d : lane_); }
static uint32_t __ballot_sync(unsigned, bool p) {
    slot[lane_] = p;
    meet.arrive_and_wait();
    uint32_t y = 0;
    for (int i = 0; i < 32; ++i) y |= (uint32_t)(slot[i] & 1) << i;
    meet.arrive_and_wait();
    return y;
}
static int __ffs(uint32_t v) { return __builtin_ffs((int)v); }
static int atomicCAS(int* p, int cmp, int v) { return __sync_val_compare_and_swap(p, cmp, v); }
#include "tb_set_walk.cuh"

int main() {
    std::mt19937 rng(7);
    int failed = 0;
    for (int test = 0; test < 6; ++test) {
        const int nset = test == 0 ? 1 : test == 1 ? 31 : 33 + 40 * test, unit = test % 2 ? 128 : 64;
        std::vector<int32_t> q{5}, k{3};
        struct Want { int q0, nq, k0, nk; uint32_t at, of; };
        std::vector<Want> want;
        for (int s = 0; s < nset; ++s) {
            const int a = rng() % 3 ? (int)(rng() % 400) : 0, b = rng() % 4 ? (int)(rng() % 300) : 0;
            const uint32_t of = (uint32_t)((a + unit - 1) / unit);
            for (uint32_t i = 0; i < of; ++i) want.push_back({q.back(), a, k.back(), b, i, of});
            q.push_back(q.back() + a);
            k.push_back(k.back() + b);
        }
        const int64_t nq = q.back() + 9, nk = k.back();
        std::vector<uint32_t> order(want.size());
        for (size_t i = 0; i < order.size(); ++i) order[i] = (uint32_t)i;
        std::vector<uint32_t> calls = order;                            // rising, falling, any
        calls.insert(calls.end(), order.rbegin(), order.rend());
        std::shuffle(order.begin(), order.end(), rng);
        calls.insert(calls.end(), order.begin(), order.end());
        calls.push_back((uint32_t)want.size());                         // behind the last, then a real one
        calls.push_back(0);
        std::vector<int> bad(32, 0);
        int err = 0;
        std::vector<std::thread> lanes;
        for (int l = 0; l < 32; ++l)
            lanes.emplace_back([&, l] {
                lane_ = l;
                tbpk::SetWalk walk;
                for (uint32_t number : calls) {
                    tbpk::SetWalk::Piece p;
                    const bool found = walk.find(q.data(), k.data(), nset, nq, nk, unit, number, l, &err, p);
                    if (found != (number < want.size())) { bad[l]++; continue; }
                    if (!found) continue;
                    const Want& w = want[number];
                    bad[l] += p.q0 != w.q0 || p.nq != w.nq || p.k0 != w.k0 || p.nk != w.nk || p.at != w.at || p.of != w.of;
                }
            });
        for (auto& t : lanes) t.join();
        for (int l = 0; l < 32; ++l) failed += bad[l];
        if (failed || err) { std::printf("test %d: %d wrong of %zu, err %d\n", test, failed, calls.size(), err); return 1; }
    }
    std::printf("walk ok\n");
    return 0;
}
"""


def test_numbers_in_any_order(tb, tmp_path):
    from trellis_cpp_b200 import build
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("g++ not found")
    (tmp_path / "walk.cpp").write_text(PROGRAM)
    b = subprocess.run([gxx, "-std=c++20", "-O1", "-pthread", "-I", build.CSRC, str(tmp_path / "walk.cpp"), "-o",
                        str(tmp_path / "walk")], capture_output=True, text=True)
    assert b.returncode == 0, b.stderr
    r = subprocess.run([str(tmp_path / "walk")], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "walk ok" in r.stdout, r.stdout + r.stderr
