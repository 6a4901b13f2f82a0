"""The C++ launchers of the serving entry points (kf/flash_attn.hpp), on the
host against a stand-in HIP runtime and C ABI: arguments arrive in their
places, statuses become hipError_t values, and attn_decode_kv4 brings the
workspace that it cannot do without, kept per stream and never grown during a
capture."""
import os
import shutil
import subprocess

import pytest

from tests.test_launcher_workspace import HIP, INCLUDE

MAIN = r"""
#include "kf/flash_attn.hpp"
#include <cstdio>
#include <cstring>
static int status = KF_OK;
static size_t need = 4096;
static void* ws_seen;
static size_t ws_bytes;
static long long seen[32];
static int count;
static void note(long long v) { seen[count++] = v; }
template <class... A> static int take(A... a) { count = 0; (note((long long)a), ...); return status; }
#define P(x) (long long)(uintptr_t)(x)
extern "C" {
int kf_last_hip_error(void) { return 2; }
int kf_attn_packed(const void* Q, const void* K, const void* V, void* O, float* m, float* l, const int64_t* s,
                   const int* qs, const int* ks, int n, int tq, int tk, int hq, int hk, int D, int f, void* st) {
    return take(P(Q), P(K), P(V), P(O), P(m), P(l), P(s), P(qs), P(ks), n, tq, tk, hq, hk, D, f, P(st));
}
int kf_qk_norm_rope(const void* Q, const void* K, void* Qo, void* Ko, const int64_t* s, const void* qw, const void* kw,
                    const int* pos, const double* fr, int T, int hq, int hk, int D, int rot, float eps, float scale,
                    int f, void* st) {
    return take(P(Q), P(K), P(Qo), P(Ko), P(s), P(qw), P(kw), P(pos), P(fr), T, hq, hk, D, rot, eps * 1000, scale, f, P(st));
}
int kf_kv4_append(const void* K, const void* V, const int64_t* s, void* Kp, void* Vp, const int* t, const int* b,
                  const int* l, int n, int T, int hk, int D, int ps, int mp, int np, int f, void* st) {
    return take(P(K), P(V), P(s), P(Kp), P(Vp), P(t), P(b), P(l), n, T, hk, D, ps, mp, np, f, P(st));
}
int kf_kv4_read(const void* Kp, const void* Vp, const int* t, const int* b, const int* l, void* K, void* V, int n, int T,
                int hk, int D, int ps, int mp, int np, int f, void* st) {
    return take(P(Kp), P(Vp), P(t), P(b), P(l), P(K), P(V), n, T, hk, D, ps, mp, np, f, P(st));
}
size_t kf_attn_decode_kv4_workspace_bytes(int, int, int, int, int, int, int) { return need; }
int kf_attn_decode_kv4(const void* Q, const void* Kp, const void* Vp, const int* t, const int* l, void* O, float* m,
                       float* s, int B, int q, int hq, int hk, int D, int ps, int mp, int np, int f, void* ws, size_t n,
                       void* st) {
    if (!ws || n < need) return KF_ERR_WORKSPACE;
    ws_seen = ws;
    ws_bytes = n;
    return take(P(Q), P(Kp), P(Vp), P(t), P(l), P(O), P(m), P(s), B, q, hq, hk, D, ps, mp, np, f, P(st));
}
}
#define REQUIRE(x) do { if (!(x)) { printf("line %d: %s\n", __LINE__, #x); return 1; } } while (0)
template <class T> T* p(long n) { return reinterpret_cast<T*>(n); }
// Arguments a .. b of the last call are consecutive numbers from `first`.
static bool run(int a, int b, long long first) {
    for (int i = a; i <= b; ++i) if (seen[i] != first + (i - a)) return false;
    return true;
}
int main() {
    hipStream_t s1 = p<S>(901), s2 = p<S>(902);
    REQUIRE(kf::attn_packed(p<uint16_t>(1), p<uint16_t>(2), p<uint16_t>(3), p<void>(4), p<int64_t>(7), p<int>(8), p<int>(9),
                            10, 11, 12, 13, 14, 15, 16, s1, p<float>(5), p<float>(6)) == hipSuccess);
    REQUIRE(run(0, 15, 1) && seen[16] == 901 && count == 17);
    REQUIRE(kf::qk_norm_rope(p<uint16_t>(1), p<uint16_t>(2), p<uint16_t>(3), p<uint16_t>(4), p<int64_t>(5), p<uint16_t>(6),
                             p<uint16_t>(7), p<int>(8), p<double>(9), 10, 11, 12, 13, 14, 0.015f, 16.0f, 17, s1) == hipSuccess);
    REQUIRE(run(0, 13, 1) && run(15, 16, 16) && seen[17] == 901);
    REQUIRE(kf::kv4_append(p<uint16_t>(1), p<uint16_t>(2), p<int64_t>(3), p<uint8_t>(4), p<uint8_t>(5), p<int>(6), p<int>(7),
                           p<int>(8), 9, 10, 11, 12, 13, 14, 15, 16, s1) == hipSuccess);
    REQUIRE(run(0, 15, 1) && seen[16] == 901);
    REQUIRE(kf::kv4_read(p<uint8_t>(1), p<uint8_t>(2), p<int>(3), p<int>(4), p<int>(5), p<uint16_t>(6), p<uint16_t>(7), 8, 9,
                         10, 11, 12, 13, 14, 15, s1) == hipSuccess);
    REQUIRE(run(0, 14, 1) && seen[15] == 901);
    auto decode = [&](hipStream_t s) {
        return kf::attn_decode_kv4(p<uint16_t>(1), p<uint8_t>(2), p<uint8_t>(3), p<int>(4), p<int>(5), p<void>(6), 9, 10, 11,
                                   12, 13, 14, 15, 16, 17, s, p<float>(7), p<float>(8));
    };
    // During a capture no workspace can be had: refused, nothing allocated.
    g_capturing = true;
    REQUIRE(decode(s1) == hipErrorStreamCaptureUnsupported && g_mallocs == 0);
    g_capturing = false;
    REQUIRE(decode(s1) == hipSuccess && run(0, 16, 1) && seen[17] == 901);
    REQUIRE(g_mallocs == 1 && ws_bytes >= need);
    void* first = ws_seen;
    REQUIRE(decode(s1) == hipSuccess && ws_seen == first && g_mallocs == 1);
    REQUIRE(decode(s2) == hipSuccess && ws_seen != first && g_mallocs == 2);    // streams share none
    g_capturing = true;
    REQUIRE(decode(s1) == hipSuccess && ws_seen == first);                      // captured with what there is
    g_capturing = false;
    need = 8192;
    REQUIRE(decode(s1) == hipSuccess && ws_seen != first && ws_bytes >= 8192);
    for (int i = 0; i < g_frees; ++i) REQUIRE(g_freed[i] != first);             // a graph holds it
    g_memory = 0;
    need = 1 << 20;
    REQUIRE(decode(s1) == hipErrorOutOfMemory);
    need = 0;                                                                   // sizes that the entry refuses
    status = KF_ERR_SIZE;
    REQUIRE(kf::kv4_read(p<uint8_t>(1), p<uint8_t>(2), nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, 0, 0, 0, s1) ==
            hipErrorInvalidValue);
    status = KF_ERR_HIP;
    REQUIRE(kf::kv4_append(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, 0, 0, 0, 0, 0, s1) ==
            hipErrorOutOfMemory);
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
