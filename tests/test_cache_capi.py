"""Refusals of the 16-bit cache's entry points, their workspaces, code objects and C++ launchers; no
GPU: every check comes before the first HIP call, and calls that are accepted run only where no GPU
could read their made-up pointers."""
import os
import re
import shutil
import subprocess

import pytest
import torch

import kernelfoundry_amd as kf
from tests.test_launcher_workspace import HIP, INCLUDE
from tests.test_serve_capi import FAKE, _strides, lib  # noqa: F401


def append(lib, K=FAKE, V=FAKE, strides=None, Kp=FAKE, Vp=FAKE, w=None, table=FAKE, starts=FAKE, lens=FAKE, n=2, T=4,  # noqa: F811
           H_kv=2, D=128, ps=16, mp=4, np_=8, flags=0):
    return lib.kf_kv_append(K, V, _strides(strides), Kp, Vp, w, table, starts, lens, n, T, H_kv, D, ps, mp, np_, flags, None)


def attend(lib, Q=FAKE, strides=None, Kp=FAKE, Vp=FAKE, table=FAKE, starts=FAKE, lens=FAKE, O=FAKE, n=2, T=4, H_q=8,  # noqa: F811
           H_kv=2, D=128, ps=16, mp=64, np_=8, flags=0, ws=FAKE, ws_bytes=1 << 50):
    return lib.kf_attn_paged(Q, _strides(strides), Kp, Vp, table, starts, lens, O, None, None, n, T, H_q, H_kv, D, ps, mp,
                             np_, flags, ws, ws_bytes, None)


def weigh(lib, Q=FAKE, strides=None, Kp=FAKE, w=FAKE, table=FAKE, starts=FAKE, lens=FAKE, lse=FAKE, n=2, T=4, H_q=8,  # noqa: F811
          H_kv=2, D=128, ps=16, mp=4, np_=8, flags=0, ws=FAKE, ws_bytes=1 << 50):
    return lib.kf_kv_weigh(Q, _strides(strides), Kp, w, table, starts, lens, lse, n, T, H_q, H_kv, D, ps, mp, np_, flags, ws,
                           ws_bytes, None)


def evict(lib, Kp=FAKE, Vp=FAKE, w=FAKE, table=FAKE, lens=FAKE, budgets=FAKE, kept=FAKE, n=2, H_kv=2, D=128, ps=16,  # noqa: F811
          mp=4, np_=8, recent=3, ws=FAKE, ws_bytes=1 << 50):
    return lib.kf_kv_evict(Kp, Vp, w, table, lens, budgets, kept, n, H_kv, D, ps, mp, np_, recent, ws, ws_bytes, None)


CALLS = (append, attend, weigh, evict)
no_gpu = pytest.mark.skipif(torch.cuda.is_available(), reason="an accepted call would run on addresses that are not real")


@no_gpu
def test_accepted_calls_reach_the_launch(lib):  # noqa: F811
    for call in CALLS:
        assert call(lib) == kf.KF_ERR_HIP, call
    for call in (append, attend, weigh):
        assert call(lib, flags=kf.KF_BF16) == kf.KF_ERR_HIP, call
    assert append(lib, strides=[768, 128, 768, 128], w=FAKE + 4) == kf.KF_ERR_HIP
    assert attend(lib, strides=[0, 0]) == kf.KF_ERR_HIP
    assert attend(lib, mp=4, ws=None, ws_bytes=0) == kf.KF_ERR_HIP      # so few keys that no tile is cut
    assert evict(lib, recent=2 ** 31 - 1) == kf.KF_ERR_HIP


@pytest.mark.parametrize("D", [0, 8, 16, 32, 80, 96, 192, 512, -128])
def test_head_dims(lib, D):  # noqa: F811
    for call in CALLS:
        assert call(lib, D=D) == kf.KF_ERR_HEAD_DIM, call
    assert kf.paged_attn_workspace_bytes(2, 4, 8, 2, D, 16, 64) == 0
    assert kf.evict_workspace_bytes(2, 2, D, 16, 64) == 0


def test_sizes(lib):  # noqa: F811
    for call in (attend, weigh):
        for H_q, H_kv in ((8, 3), (0, 2), (8, 0), (-8, 2), (2, 8), (8, -2)):
            assert call(lib, H_q=H_q, H_kv=H_kv) == kf.KF_ERR_GQA
    top = 2 ** 31 - 1
    for call in CALLS:
        for kw in (dict(n=0), dict(n=-1), dict(ps=8), dict(ps=24), dict(ps=1 << 21), dict(mp=0), dict(np_=0),
                   dict(ps=1 << 20, mp=4096)):
            assert call(lib, **kw) == kf.KF_ERR_SIZE, (call, kw)
        if call is not append:      # indexes that rounding up to a tile would take past an int
            assert call(lib, mp=top // 16) == kf.KF_ERR_SIZE, call
        if call is not evict:
            for kw in (dict(T=0), dict(T=-1), dict(T=top, H_kv=1), dict(T=1 << 30)):
                assert call(lib, **kw) == kf.KF_ERR_SIZE, (call, kw)
    assert append(lib, H_kv=0) == kf.KF_ERR_SIZE and evict(lib, H_kv=0) == kf.KF_ERR_SIZE
    assert evict(lib, recent=-1) == kf.KF_ERR_SIZE
    # Grids of more threads than a launch can number.
    assert append(lib, T=1 << 27, H_kv=8, D=256) == kf.KF_ERR_SIZE
    assert evict(lib, n=1 << 22, H_kv=1) == kf.KF_ERR_SIZE


def test_flags(lib):  # noqa: F811
    for f in (64, kf.KF_ROPE_INTERLEAVED, kf.KF_ATTN_OUT_F16 | kf.KF_ATTN_OUT_BF16, -1):
        assert attend(lib, flags=f) == kf.KF_ERR_FLAGS, f
    for f in (2, 4, 8, 32, 64, -1):
        assert weigh(lib, flags=f) == kf.KF_ERR_FLAGS, f
    for f in (1, 2, 8, 32, 64):
        assert append(lib, flags=f) == kf.KF_ERR_FLAGS, f


def test_null_and_misaligned_pointers(lib):  # noqa: F811
    names = {append: ("K", "V", "Kp", "Vp", "table", "starts", "lens"), attend: ("Q", "Kp", "Vp", "table", "starts", "lens", "O"),
             weigh: ("Q", "Kp", "w", "table", "starts", "lens", "lse"),
             evict: ("Kp", "Vp", "w", "table", "lens", "budgets", "kept")}
    for call, some in names.items():
        for name in some:
            assert call(lib, **{name: None}) == kf.KF_ERR_NULL, (call, name)
            assert call(lib, **{name: FAKE + 2}) == kf.KF_ERR_ALIGN, (call, name)
        for name in set(some) & {"Q", "K", "V", "Kp", "Vp", "O"}:
            assert call(lib, **{name: FAKE + 8}) == kf.KF_ERR_ALIGN, (call, name)
    assert append(lib, w=FAKE + 2) == kf.KF_ERR_ALIGN


def test_strides(lib):  # noqa: F811
    for call, n in ((append, 4), (attend, 2), (weigh, 2)):
        for i in range(n):
            s = [1024] * n
            s[i] = 1020
            assert call(lib, strides=s) == kf.KF_ERR_ALIGN
            s[i] = -1024
            assert call(lib, strides=s) == kf.KF_ERR_SIZE


def test_workspaces(lib):  # noqa: F811
    need = kf.paged_attn_workspace_bytes(2, 4, 8, 2, 128, 16, 64)
    assert need > 0 and need % 256 == 0
    assert attend(lib, ws=None) == attend(lib, ws_bytes=need - 1) == kf.KF_ERR_WORKSPACE
    assert attend(lib, ws=FAKE + 16) == kf.KF_ERR_ALIGN
    assert kf.paged_attn_workspace_bytes(2, 4, 8, 3, 128, 16, 64) == 0
    # A share for every workgroup, however many sequences.
    assert kf.paged_attn_workspace_bytes(1 << 26, 1 << 26, 8, 2, 128, 16, 64) == need
    # Tiles enough for the device, or few keys: none is cut.
    assert kf.paged_attn_workspace_bytes(8, 1 << 15, 32, 8, 128, 16, 1024) == 0
    assert kf.paged_attn_workspace_bytes(8, 8, 32, 8, 128, 16, 4) == 0
    need = kf.weigh_workspace_bytes(1, 2048, 32, 8, 128, 16, 256)
    assert need > 0 and need % 256 == 0 and kf.weigh_workspace_bytes(64, 64, 32, 8, 128, 16, 256) == 0
    many = dict(n=1, T=2048, H_q=32, H_kv=8, mp=256)
    assert weigh(lib, ws=None, **many) == weigh(lib, ws_bytes=need - 1, **many) == kf.KF_ERR_WORKSPACE
    assert weigh(lib, ws=FAKE + 16, **many) == kf.KF_ERR_ALIGN
    need = kf.evict_workspace_bytes(2, 2, 128, 16, 4)
    assert need == 256 + 2 * 2 * 64 * 4
    assert evict(lib, ws=None) == evict(lib, ws_bytes=need - 1) == kf.KF_ERR_WORKSPACE
    assert evict(lib, ws=FAKE + 16) == kf.KF_ERR_ALIGN


def test_python_entries_refuse_cpu_tensors():
    h = torch.float16
    Q, K = torch.zeros(4, 8, 128, dtype=h), torch.zeros(4, 2, 128, dtype=h)
    pages, w = torch.zeros(2, 2, 16, 128, dtype=h), torch.zeros(2, 2, 16)
    starts, lens, table = (torch.tensor(x, dtype=torch.int32) for x in ([0, 4], [4], [[1]]))
    for call in (lambda: kf.kv_append(K, K, pages, pages, table, starts, lens),
                 lambda: kf.attn_paged(Q, pages, pages, table, starts, lens),
                 lambda: kf.kv_weigh(Q, pages, w, table, starts, lens, torch.zeros(4, 8)),
                 lambda: kf.kv_evict(pages, pages, w, table, lens, lens)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_no_kernel_uses_scratch(tmp_path):
    tools = "/opt/rocm/llvm/bin"
    objcopy, bundler, readelf = (os.path.join(tools, t) for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-readelf"))
    if not all(os.path.exists(t) for t in (objcopy, bundler, readelf)):
        pytest.skip("ROCm LLVM tools not found")
    fat = tmp_path / "fatbin"
    subprocess.run([objcopy, "--dump-section", f".hip_fatbin={fat}", kf.LIB_PATH], check=True)
    blob, found = fat.read_bytes(), {}
    at = [m.start() for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", blob)]
    for k, (a, b) in enumerate(zip(at, at[1:] + [len(blob)])):
        part, co = tmp_path / f"part{k}", tmp_path / f"{k}.co"
        part.write_bytes(blob[a:b])
        subprocess.run([bundler, "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950", f"--input={part}",
                        f"--output={co}"], check=True)
        notes = subprocess.run([readelf, "--notes", str(co)], capture_output=True, text=True, check=True).stdout
        for block in re.split(r"\n\s+- \.agpr_count:", notes)[1:]:
            name = re.search(r"\.name:\s+(\S+)", block).group(1)
            found[name] = (int(re.search(r"\.private_segment_fixed_size:\s+(\d+)", block).group(1)),
                           int(re.search(r"\.vgpr_spill_count:\s+(\d+)", block).group(1)))
    mine = {n: v for n, v in found.items() if re.search("kf_attn_paged|kf_kv_append|kf_kv_weigh|kf_kv_evict", n)}
    assert {re.search(r"kf_[a-z0-9_]+?_kernel", n).group(0) for n in mine} >= {
        "kf_attn_paged_kernel", "kf_attn_paged_merge_kernel", "kf_kv_append_kernel", "kf_kv_weigh_kernel",
        "kf_kv_weigh_merge_kernel", "kf_kv_evict_select_kernel", "kf_kv_evict_move_kernel"}
    assert not {n: v for n, v in mine.items() if v != (0, 0)}


MAIN = r"""
#include "kf/flash_attn.hpp"
#include <cstdio>
static int status = KF_OK;
static size_t need = 4096, ws_bytes;
static void* ws_seen;
static long long seen[32];
static int count;
static void note(long long v) { seen[count++] = v; }
template <class... A> static int take(A... a) { count = 0; (note((long long)a), ...); return status; }
#define P(x) (long long)(uintptr_t)(x)
extern "C" {
int kf_last_hip_error(void) { return 2; }
int kf_kv_append(const void* K, const void* V, const int64_t* s, void* Kp, void* Vp, float* w, const int* t, const int* b,
                 const int* l, int n, int T, int hk, int D, int ps, int mp, int np, int f, void* st) {
    return take(P(K), P(V), P(s), P(Kp), P(Vp), P(w), P(t), P(b), P(l), n, T, hk, D, ps, mp, np, f, P(st));
}
size_t kf_attn_paged_workspace_bytes(int, int, int, int, int, int, int) { return need; }
int kf_attn_paged(const void* Q, const int64_t* s, const void* Kp, const void* Vp, const int* t, const int* b, const int* l,
                  void* O, float* m, float* u, int n, int T, int hq, int hk, int D, int ps, int mp, int np, int f, void* ws,
                  size_t have, void* st) {
    if (need && (!ws || have < need)) return KF_ERR_WORKSPACE;
    ws_seen = ws;
    ws_bytes = have;
    return take(P(Q), P(s), P(Kp), P(Vp), P(t), P(b), P(l), P(O), P(m), P(u), n, T, hq, hk, D, ps, mp, np, f, P(st));
}
size_t kf_kv_weigh_workspace_bytes(int, int, int, int, int, int, int) { return need; }
int kf_kv_weigh(const void* Q, const int64_t* s, const void* Kp, float* w, const int* t, const int* b, const int* l,
                const float* e, int n, int T, int hq, int hk, int D, int ps, int mp, int np, int f, void* ws, size_t have,
                void* st) {
    if (need && (!ws || have < need)) return KF_ERR_WORKSPACE;
    ws_seen = ws;
    ws_bytes = have;
    return take(P(Q), P(s), P(Kp), P(w), P(t), P(b), P(l), P(e), n, T, hq, hk, D, ps, mp, np, f, P(st));
}
size_t kf_kv_evict_workspace_bytes(int, int, int, int, int) { return need; }
int kf_kv_evict(void* Kp, void* Vp, float* w, const int* t, const int* l, const int* m, int* k, int n, int hk, int D, int ps,
                int mp, int np, int r, void* ws, size_t have, void* st) {
    if (!ws || have < need) return KF_ERR_WORKSPACE;
    ws_seen = ws;
    ws_bytes = have;
    return take(P(Kp), P(Vp), P(w), P(t), P(l), P(m), P(k), n, hk, D, ps, mp, np, r, P(st));
}
}
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
template <class T> T* p(long n) { return reinterpret_cast<T*>(n); }
static bool run(int a, int b, long long first) {
    for (int i = a; i <= b; ++i) if (seen[i] != first + (i - a)) return false;
    return true;
}
int main() {
    hipStream_t s1 = p<S>(901), s2 = p<S>(902);
    typedef uint16_t H;
    REQUIRE(kf::kv_append(p<H>(1), p<H>(2), p<int64_t>(3), p<H>(4), p<H>(5), p<float>(6), p<int>(7), p<int>(8), p<int>(9), 10,
                          11, 12, 13, 14, 15, 16, 17, s1) == hipSuccess);
    REQUIRE(run(0, 16, 1) && seen[17] == 901 && count == 18);
    auto weigh = [&](hipStream_t s) {
        return kf::kv_weigh(p<H>(1), p<int64_t>(2), p<H>(3), p<float>(4), p<int>(5), p<int>(6), p<int>(7), p<float>(8), 9, 10, 11,
                            12, 13, 14, 15, 16, 17, s);
    };
    auto attend = [&](hipStream_t s) {
        return kf::attn_paged(p<H>(1), p<int64_t>(2), p<H>(3), p<H>(4), p<int>(5), p<int>(6), p<int>(7), p<void>(8), 11, 12, 13,
                              14, 15, 16, 17, 18, 19, s, p<float>(9), p<float>(10));
    };
    auto evict = [&](hipStream_t s) {
        return kf::kv_evict(p<H>(1), p<H>(2), p<float>(3), p<int>(4), p<int>(5), p<int>(6), p<int>(7), 8, 9, 10, 11, 12, 13, 14, s);
    };
    // During a capture no workspace can be had: refused, nothing allocated.
    g_capturing = true;
    REQUIRE(attend(s1) == hipErrorStreamCaptureUnsupported && evict(s1) == hipErrorStreamCaptureUnsupported && g_mallocs == 0);
    REQUIRE(weigh(s1) == hipErrorStreamCaptureUnsupported && g_mallocs == 0);
    g_capturing = false;
    REQUIRE(attend(s1) == hipSuccess && run(0, 18, 1) && seen[19] == 901 && g_mallocs == 1 && ws_bytes >= need);
    void* first = ws_seen;
    REQUIRE(evict(s1) == hipSuccess && run(0, 13, 1) && seen[14] == 901 && ws_seen == first && g_mallocs == 1);
    REQUIRE(weigh(s1) == hipSuccess && run(0, 16, 1) && seen[17] == 901 && count == 18 && ws_seen == first && g_mallocs == 1);
    REQUIRE(evict(s2) == hipSuccess && ws_seen != first && g_mallocs == 2);     // streams share none
    g_capturing = true;
    REQUIRE(attend(s1) == hipSuccess && ws_seen == first);                      // captured with what there is
    g_capturing = false;
    need = 8192;
    REQUIRE(attend(s1) == hipSuccess && ws_seen != first && ws_bytes >= 8192);
    for (int i = 0; i < g_frees; ++i) REQUIRE(g_freed[i] != first);             // a graph holds it
    need = 0;                                                                   // a call that is not cut
    REQUIRE(attend(p<S>(903)) == hipSuccess && ws_seen == nullptr);
    REQUIRE(weigh(p<S>(903)) == hipSuccess && ws_seen == nullptr);
    status = KF_ERR_SIZE;
    REQUIRE(kf::kv_append(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, 0, 0, 0,
                          s1) == hipErrorInvalidValue);
    puts("ok");
    return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not installed")
def test_launchers(tmp_path):
    (tmp_path / "hip").mkdir()
    (tmp_path / "hip" / "hip_runtime.h").write_text(HIP)
    (tmp_path / "main.cpp").write_text(MAIN)
    exe = tmp_path / "main"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", f"-I{tmp_path}", f"-I{INCLUDE}", str(tmp_path / "main.cpp"),
                    "-o", str(exe)], check=True, capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
