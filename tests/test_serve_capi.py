"""Refusals of the serving entry points (packed attention, norm and rotary
positions, 4-bit cache), sizes and helpers; no GPU: every check comes before
the first HIP call and the fake device pointers are never dereferenced."""
import ctypes
import math
import os
import re
import subprocess

import pytest
import torch

import kernelfoundry_amd as kf

FAKE = 0x10000


@pytest.fixture(scope="module")
def lib():
    return kf.load_library()


def _strides(values):
    return (ctypes.c_int64 * len(values))(*values) if values else None


def packed(lib, Q=FAKE, K=FAKE, V=FAKE, O=FAKE, strides=None, qs=FAKE, ks=FAKE, n=2, tq=10, tk=10, H_q=8, H_kv=2,
           D=128, flags=0):
    return lib.kf_attn_packed(Q, K, V, O, None, None, _strides(strides), qs, ks, n, tq, tk, H_q, H_kv, D, flags, None)


def rope(lib, Q=FAKE, K=FAKE, Qo=FAKE, Ko=FAKE, strides=None, qw=None, kw=None, pos=FAKE, fr=FAKE, T=4, H_q=8,
         H_kv=2, D=128, rot=128, flags=0):
    return lib.kf_qk_norm_rope(Q, K, Qo, Ko, _strides(strides), qw, kw, pos, fr, T, H_q, H_kv, D, rot, 1e-6, 1.0,
                               flags, None)


def append(lib, K=FAKE, V=FAKE, strides=None, Kp=FAKE, Vp=FAKE, table=FAKE, starts=FAKE, lens=FAKE, n=2, T=4,
           H_kv=2, D=128, ps=16, mp=4, np_=8, flags=0):
    return lib.kf_kv4_append(K, V, _strides(strides), Kp, Vp, table, starts, lens, n, T, H_kv, D, ps, mp, np_, flags,
                             None)


def read(lib, Kp=FAKE, Vp=FAKE, table=FAKE, starts=FAKE, lens=FAKE, K=FAKE, V=FAKE, n=2, T=4, H_kv=2, D=128, ps=16,
         mp=4, np_=8, flags=0):
    return lib.kf_kv4_read(Kp, Vp, table, starts, lens, K, V, n, T, H_kv, D, ps, mp, np_, flags, None)


def decode(lib, Q=FAKE, Kp=FAKE, Vp=FAKE, table=FAKE, lens=FAKE, O=FAKE, B=2, q=1, H_q=8, H_kv=2, D=128, ps=16,
           mp=4, np_=8, flags=0, ws=FAKE, ws_bytes=1 << 40):
    return lib.kf_attn_decode_kv4(Q, Kp, Vp, table, lens, O, None, None, B, q, H_q, H_kv, D, ps, mp, np_, flags, ws,
                                  ws_bytes, None)


def test_valid_calls_reach_the_first_hip_call(lib):
    """On a host without a GPU an accepted call fails only at its launch."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are fakes")
    for call in (packed, rope, append, read, decode):
        assert call(lib) == kf.KF_ERR_HIP
    assert packed(lib, strides=[1536, 128, 1536, 128, 1536, 128]) == kf.KF_ERR_HIP
    assert packed(lib, strides=[0] * 6) == kf.KF_ERR_HIP
    assert rope(lib, rot=0, pos=None, fr=None) == kf.KF_ERR_HIP
    assert rope(lib, D=16, rot=16) == kf.KF_ERR_HIP


@pytest.mark.parametrize("D", [0, 8, 16, 32, 80, 96, 192, 512, -128])
def test_head_dims(lib, D):
    for call in (packed, append, read, decode):
        assert call(lib, D=D) == kf.KF_ERR_HEAD_DIM, call
    if D != 16:
        assert rope(lib, D=D) == kf.KF_ERR_HEAD_DIM
    assert lib.kf_kv4_page_bytes(16, D) == 0


@pytest.mark.parametrize("H_q,H_kv", [(8, 3), (0, 2), (8, 0), (-8, 2), (2, 8), (8, -2)])
def test_head_counts(lib, H_q, H_kv):
    assert packed(lib, H_q=H_q, H_kv=H_kv) == kf.KF_ERR_GQA
    assert decode(lib, H_q=H_q, H_kv=H_kv) == kf.KF_ERR_GQA


def test_sizes(lib):
    big = 1 << 30
    for kw in (dict(n=0), dict(n=-1), dict(tq=0), dict(tk=0), dict(tq=-5), dict(tq=big), dict(tk=big)):
        assert packed(lib, **kw) == kf.KF_ERR_SIZE, kw
    assert packed(lib, H_q=1 << 20, H_kv=1, tq=1, tk=1 << 12) == kf.KF_ERR_SIZE
    # Indexes that rounding up to a tile would take past an int.
    top = 2 ** 31 - 1
    assert packed(lib, tq=top // 8) == kf.KF_ERR_SIZE
    assert packed(lib, tk=top // 4) == kf.KF_ERR_SIZE
    assert rope(lib, T=top) == kf.KF_ERR_SIZE
    # Grids of more threads than a launch can number.
    assert rope(lib, T=1 << 27, H_q=1, H_kv=1) == kf.KF_ERR_SIZE
    assert packed(lib, n=1 << 24, tq=1 << 24, H_q=2, H_kv=2) == kf.KF_ERR_SIZE
    for call in (append, read):
        assert call(lib, T=top, H_kv=1) == kf.KF_ERR_SIZE
    assert decode(lib, B=1, H_q=1, H_kv=1, mp=top // 16) == kf.KF_ERR_SIZE
    for kw in (dict(T=0), dict(T=-1), dict(H_q=0), dict(H_kv=0), dict(rot=-16), dict(rot=8), dict(rot=144),
               dict(rot=24)):
        assert rope(lib, **kw) == kf.KF_ERR_SIZE, kw
    for call in (append, read):
        for kw in (dict(n=0), dict(T=0), dict(H_kv=0), dict(ps=8), dict(ps=24), dict(mp=0), dict(np_=0),
                   dict(ps=1 << 20, mp=4096), dict(T=big)):
            assert call(lib, **kw) == kf.KF_ERR_SIZE, (call, kw)
    for kw in (dict(B=0), dict(q=0), dict(ps=8), dict(ps=48), dict(mp=0), dict(np_=0), dict(q=9),
               dict(H_q=66), dict(ps=1 << 20, mp=4096), dict(B=1 << 20, mp=1 << 16)):
        assert decode(lib, **kw) == kf.KF_ERR_SIZE, kw


def test_flags(lib):
    both = kf.KF_ATTN_OUT_F16 | kf.KF_ATTN_OUT_BF16
    for call in (packed, decode):
        for f in (64, kf.KF_ROPE_INTERLEAVED, both, -1):
            assert call(lib, flags=f) == kf.KF_ERR_FLAGS, (call, f)
    for f in (1, 2, 4, 8, 64):
        assert rope(lib, flags=f) == kf.KF_ERR_FLAGS
    for call in (append, read):
        for f in (1, 8, kf.KF_ROPE_INTERLEAVED, 64):
            assert call(lib, flags=f) == kf.KF_ERR_FLAGS


def test_null_and_misaligned_pointers(lib):
    pointers = {packed: ("Q", "K", "V", "O", "qs", "ks"), rope: ("Q", "K", "Qo", "Ko", "pos", "fr"),
                append: ("K", "V", "Kp", "Vp", "table", "starts", "lens"),
                read: ("K", "V", "Kp", "Vp", "table", "starts", "lens"),
                decode: ("Q", "Kp", "Vp", "table", "lens", "O")}
    for call, names in pointers.items():
        for name in names:
            assert call(lib, **{name: None}) == kf.KF_ERR_NULL, (call, name)
            assert call(lib, **{name: FAKE + 2}) == kf.KF_ERR_ALIGN, (call, name)
    for name in ("qw", "kw"):
        assert rope(lib, **{name: FAKE + 8}) == kf.KF_ERR_ALIGN
    assert rope(lib, fr=FAKE + 4) == kf.KF_ERR_ALIGN


def test_strides(lib):
    for call, n in ((packed, 6), (rope, 8), (append, 4)):
        for i in range(n):
            s = [1024] * n
            s[i] = 1020
            assert call(lib, strides=s) == kf.KF_ERR_ALIGN
            s[i] = -1024
            assert call(lib, strides=s) == kf.KF_ERR_SIZE


def test_packed_key_strides(lib):
    top = 1 << 28
    for i in range(6):
        s = [1024] * 6
        s[i] = top + 8
        assert (packed(lib, strides=s) == kf.KF_ERR_SIZE) == (i in (2, 4)), i


@pytest.mark.parametrize("token,head,ok", [(1024, 128, True), (128, 512, True), (2048, 136, True), (0, 128, False),
                                           (1024, 0, False), (1016, 128, False), (120, 512, False), (128, 504, False),
                                           (1 << 62, 128, True), (1 << 62, 1 << 62, False)])
def test_rope_outputs_are_not_broadcast(lib, token, head, ok):
    """4 tokens of 8 heads of 128: rows that overlap would be written twice."""
    if torch.cuda.is_available() and ok:
        pytest.skip("the pointers are fakes")
    s = [1024, 128, 256, 128, token, head, 256, 128]
    assert rope(lib, strides=s) == (kf.KF_ERR_HIP if ok else kf.KF_ERR_SIZE)
    s = [1024, 128, 1024, 128, 1024, 128, token, head]
    assert rope(lib, strides=s, H_kv=8) == (kf.KF_ERR_HIP if ok else kf.KF_ERR_SIZE)
    # Strides of a single token or head do not count.
    if not torch.cuda.is_available():
        assert rope(lib, strides=[1024, 128, 0, 0, 1024, 128, 0, 0], T=1, H_kv=1) == kf.KF_ERR_HIP


def test_decode_workspace(lib):
    need = kf.kv4_workspace_bytes(2, 1, 8, 2, 128, 16, 4)
    assert need > 0 and need % 256 == 0
    assert decode(lib, ws=None) == kf.KF_ERR_WORKSPACE
    assert decode(lib, ws_bytes=need - 1) == kf.KF_ERR_WORKSPACE
    assert decode(lib, ws=FAKE + 16) == kf.KF_ERR_ALIGN
    assert kf.kv4_workspace_bytes(2, 9, 8, 2, 128, 16, 4) == 0    # 36 rows per KV head
    assert kf.kv4_workspace_bytes(2, 1, 8, 2, 96, 16, 4) == 0
    # Two partials a wave, of R rows of D + 2 floats, and 16 bytes a head; a
    # small capacity has no more workgroups than its stages fill.
    stages = 2 * 2 * (4 * 16 // 32)
    assert need == 2 * stages * 4 * 128 * 4 + 2 * 256 + 256
    big = [kf.kv4_workspace_bytes(64, q, 8, 2, 128, 16, 4096) for q in (1, 2, 4, 8)]
    assert big == sorted(big)


def test_page_bytes(lib):
    for D in (64, 128, 256):
        for ps in (16, 32, 1 << 20):
            assert kf.kv4_page_bytes(ps, D) == ps * (D // 2 + D // 32)
    for ps in (0, 8, 17, 24, 1 << 21, -16):
        with pytest.raises(ValueError):
            kf.kv4_page_bytes(ps, 128)


def test_every_code_object_keeps_out_of_scratch(tmp_path):
    """The kernels of the serving operators, in the library's second code
    object: no private segment, no spilled vector registers."""
    tools = "/opt/rocm/llvm/bin"
    objcopy, bundler, readelf = (os.path.join(tools, t) for t in
                                 ("llvm-objcopy", "clang-offload-bundler", "llvm-readelf"))
    if not all(os.path.exists(t) for t in (objcopy, bundler, readelf)):
        pytest.skip("ROCm LLVM tools not found")
    fat = tmp_path / "fatbin"
    subprocess.run([objcopy, "--dump-section", f".hip_fatbin={fat}", kf.LIB_PATH], check=True)
    blob, kernels = fat.read_bytes(), {}
    magic = b"__CLANG_OFFLOAD_BUNDLE__"
    at = [m.start() for m in re.finditer(magic, blob)]
    assert len(at) == 2
    for k, (a, b) in enumerate(zip(at, at[1:] + [len(blob)])):
        part, co = tmp_path / f"part{k}", tmp_path / f"{k}.co"
        part.write_bytes(blob[a:b])
        subprocess.run([bundler, "--unbundle", "--type=o", "--targets=hipv4-amdgcn-amd-amdhsa--gfx950",
                        f"--input={part}", f"--output={co}"], check=True)
        notes = subprocess.run([readelf, "--notes", str(co)], capture_output=True, text=True, check=True).stdout
        for block in re.split(r"\n\s+- \.agpr_count:", notes)[1:]:
            name = re.search(r"\.name:\s+(\S+)", block).group(1)
            kernels[name] = (int(re.search(r"\.private_segment_fixed_size:\s+(\d+)", block).group(1)),
                             int(re.search(r"\.vgpr_spill_count:\s+(\d+)", block).group(1)))
    mine = {n: v for n, v in kernels.items()
            if re.search("kf_attn_packed|kf_qk_norm_rope|kf_kv4|kf_attn_decode_kv4", n)}
    assert {re.search(r"kf_[a-z0-9_]+?_kernel", n).group(0) for n in mine} >= {
        "kf_attn_packed_kernel", "kf_qk_norm_rope_kernel", "kf_kv4_append_kernel", "kf_kv4_read_kernel",
        "kf_attn_decode_kv4_kernel"}
    assert not {n: v for n, v in mine.items() if v != (0, 0)}


def test_python_entries_refuse_cpu_tensors_and_bad_shapes():
    h = torch.float16
    Q, K = torch.zeros(4, 8, 128, dtype=h), torch.zeros(4, 2, 128, dtype=h)
    starts, lens = torch.tensor([0, 4], dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    pages, table = torch.zeros(2, 2, 16 * 68, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        kf.attn_packed(Q, K, K, starts)
    with pytest.raises(ValueError, match="GPU"):
        kf.qk_norm_rope(Q, K, None, None)
    with pytest.raises(ValueError, match="GPU"):
        kf.kv4_append(K, K, pages, pages, table, starts, lens)
    with pytest.raises(ValueError, match="GPU"):
        kf.kv4_read(pages, pages, table, starts, lens, 4, 128)
    with pytest.raises(ValueError, match="GPU"):
        kf.attn_decode_kv4(Q[:, :, None], pages, pages, table, lens)
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        kf.kv4_read(pages, pages, table, starts, lens, 4, 128, out_dtype=torch.float32)


# ---------------------------------------------------------------------------
# Frequencies.
# ---------------------------------------------------------------------------
def test_rope_freqs_plain_and_linear():
    f, s = kf.rope_freqs(64, 500.0)
    assert f.dtype == torch.float64 and f.shape == (32,) and s == 1.0
    for i in (0, 1, 31):
        assert float(f[i]) == pytest.approx(500.0 ** (-2 * i / 64), rel=1e-14)
    g, s = kf.rope_freqs(64, 500.0, scaling="linear", factor=8.0)
    assert s == 1.0 and torch.allclose(g * 8, f, rtol=1e-14, atol=0)


def test_rope_freqs_ntk_keeps_the_highest_and_interpolates_the_lowest():
    f, _ = kf.rope_freqs(128)
    g, s = kf.rope_freqs(128, scaling="ntk", factor=4.0)
    assert s == 1.0 and float(g[0]) == 1.0
    assert float(g[-1] * 4) == pytest.approx(float(f[-1]), rel=1e-12)
    assert (g[1:] < f[1:]).all()


def test_rope_freqs_yarn_by_turns():
    f, _ = kf.rope_freqs(128)
    g, s = kf.rope_freqs(128, scaling="yarn", factor=16.0, original_len=4096)
    assert s == pytest.approx(1 + 0.1 * math.log(16), rel=1e-14)
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and (turns >= 32).any()
    low = turns <= 1
    assert low.any() and torch.allclose(g[low], f[low] / 16, rtol=1e-14, atol=0)
    mid = ~low & (turns < 32)
    share = (turns[mid] - 1) / 31
    assert torch.allclose(g[mid], f[mid] * share + f[mid] / 16 * (1 - share), rtol=1e-13, atol=0)


@pytest.mark.parametrize("kw", [dict(rot=0), dict(rot=-2), dict(rot=7), dict(scaling="other"),
                                dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0),
                                dict(scaling="yarn", factor=2.0, original_len=64, beta_fast=1.0),
                                dict(rot=2, scaling="ntk", factor=2.0)])
def test_rope_freqs_refusals(kw):
    with pytest.raises(ValueError):
        kf.rope_freqs(**{"rot": 64, **kw})
