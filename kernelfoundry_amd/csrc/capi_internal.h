// capi_internal.h -- what the two translation units of the C ABI share
// (attn_capi.hip defines it; none of it is exported).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "kf/attn.h"

namespace kf {
struct AttnParams;
}

namespace kf_capi __attribute__((visibility("hidden"))) {

constexpr size_t kWsAlign = 256;

struct DeviceShape {
    int cus;
    int xcds;
};

// CU and XCD counts of the device current on the calling thread, cached per
// device; the MI355X defaults when no device is visible.
DeviceShape current_device_shape();

// Keeps e for kf_last_hip_error(); returns KF_ERR_HIP.
int hip_fail(hipError_t e);

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }
inline bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

// Paged geometry: page_size a power of two in [16, 2^20], positive counts,
// key capacity max_pages_per_seq * page_size within int.  Returns the
// status and, on success, log2(page_size) and the capacity.
int paged_geometry(int page_size, int max_pages_per_seq, int num_pages, int* shift, int* cap);

// Waves per KV head of the ragged decode's merge, and its launch
// (kf_attn_ragged_merge_kernel, D = 64, 128 or 256; prm.merge_waves waves).
int ragged_merge_waves(int R, int n_groups, int D);
hipError_t merge_ragged(int D, int n_groups, const kf::AttnParams& prm, hipStream_t stream);

}  // namespace kf_capi
