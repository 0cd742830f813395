// fa_launch.h - host-side launch plumbing shared by the kernel translation units
// and the C ABI (fa_api.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include "../../include/fa.h"

namespace fa {

struct FwdArgs {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;
  int B, H, Hkv, S, D;
  float scale_log2;
  void* stream;
};

struct BwdArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* o;
  const void* d_o;
  const float* lse;
  void* dq;
  void* dk;
  void* dv;
  int B, H, Hkv, S, D;
  float scale_log2;
  float sm_scale;
  void* stream;
  // the (query tile, query head) pairs of a key tile are split over `nsplit`
  // workgroups, each writing fp32 partial dK / dV ([B*Hkv*nsplit, S, D] each) that a
  // reduction pass adds up; nsplit = 1: one workgroup, no workspace
  float* wsk;
  float* wsv;
  int nsplit;
  // [2, B*H, S] fp32: -LSE/c and -Delta of every query row, written by the dQ
  // kernel (then launched first) for the dK/dV kernel; null: dK/dV runs first, with
  // the terms written into dQ's own buffer by a row-terms pass (dQ overwrites them
  // last), or, with form_delta, formed by the dK/dV kernel in every key tile
  float* rowb;
  bool form_delta;
  // the grid leaves the GPU idle: dQ, and dK / dV where it is not split, in one launch
  bool small;
};

// rows [B, heads, N, D] with strides, and their norm and rotation, as the C ABI takes them
typedef ::fa_rows Rows;
typedef ::fa_rotation RotaryArgs;
constexpr int kMaxAxes = 3;

struct QkArgs {          // norm and rotation of q and k, forward or backward
  Rows q, k;             // inputs
  Rows gq, gk;           // backward: gradients of the outputs
  Rows oq, ok;           // outputs: y, or the gradients of q and k
  RotaryArgs rot;
  int B, H, Hkv, N;
  int heads;             // heads a workgroup takes one after another (q's or k's, never both)
  int blocks;            // backward: workgroups per chunk of heads
  float* part;           // backward: fp32 partial weight gradients [chunk, blocks][D]
  void* dwq;
  void* dwk;
  void* stream;
};

struct AppendArgs {
  Rows q, k, v, oq;      // oq: the turned queries (q.data null: none)
  RotaryArgs rot;
  ::fa_paged_cache cache;
  const int* past;
  const int* fresh;      // new tokens of each sequence; null: N
  int B, H, N, D;
  int heads;             // query heads a workgroup takes one after another
  void* stream;
};

struct PagedArgs {
  Rows q, o;
  ::fa_paged_cache cache;
  const int* past;
  const int* fresh;
  float* lse;            // [B, H, N]; null: none
  float* part;           // partial rows of a split, null: none
  int B, H, N, D;
  int nsplit;
  float scale_log2;
  void* stream;
};

// keys per dK/dV workgroup (4 waves x 32 keys), for the split heuristics on the host
constexpr int kDkdvKeys = 128;

typedef int (*FwdFn)(const FwdArgs&);
typedef int (*BwdFn)(const BwdArgs&);

// (fa_rotary.hip, fa_paged.hip; arguments checked by fa_api.hip)
int qk_norm_rotary(int dtype, int D, const QkArgs& a);
int qk_norm_rotary_bwd(int dtype, int D, const QkArgs& a);
size_t qk_norm_rotary_workspace(int B, int H, int Hkv, int N, int D);
int paged_append(int dtype, const AppendArgs& a);
int paged_attention(int dtype, PagedArgs a, size_t workspace_bytes);
int paged_attention_exact(int dtype, PagedArgs a, int block_rows, int parts, size_t workspace_bytes);
size_t paged_attention_workspace(int B, int H, int Hkv, int N, int D, long long keys);

// Raise the dynamic LDS limit of a kernel once (needed above 64 KB).  The
// static local makes the first call per kernel instance thread-safe.
template <int SMEM>
inline bool smem_attr(const void* kern) {
  if (SMEM <= 65536) return true;
  return hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, SMEM) == hipSuccess;
}

// CU count of the current device, read once per device and kept (the launch paths ask
// on every call, and a short call is bound by host time).  A failed query is answered
// with 256 (an MI355X) and leaves the HIP error state as the query left it: nothing here
// clears an error the caller's own work left behind.
constexpr int kMaxDevices = 64;
inline int cu_count() {
  static std::atomic<int> cus_of[kMaxDevices];
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 256;
  int cus = cus_of[dev].load(std::memory_order_relaxed);
  if (cus > 0) return cus;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus <= 0) return 256;
  cus_of[dev].store(cus, std::memory_order_relaxed);
  return cus;
}

// Grid of a kernel whose workgroups walk their share of `items` work items: the item
// count rounded up to a multiple of 8 (workgroups reach the 8 XCDs in turn), capped
// at the workgroups the device runs at once (its CUs times the kernel's occupancy
// per_cu, rounded down to a multiple of 8).
inline int resident_grid(int items, int per_cu) {
  const int all = (items + 7) / 8 * 8;
  if (per_cu <= 0) return all;
  const int resident = cu_count() * per_cu / 8 * 8;
  return resident >= 8 && resident < all ? resident : all;
}

// Workgroups of `kern` (launched with `threads` threads) that one CU holds at once;
// 0 if the runtime cannot tell (the callers keep the answer per kernel).
inline int occupancy_per_cu(const void* kern, int threads) {
  int per_cu = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kern, threads, 0) != hipSuccess) return 0;
  return per_cu;
}

// Whether a launch's threads stay below the runtime's 2^32.
inline bool grid_fits(long long workgroups, int threads) { return workgroups <= 0xffffffffLL / threads; }

#define set_smem_once(kern, SMEM)                                   \
  ([&]() {                                                          \
    static const bool ok_ = ::fa::smem_attr<SMEM>(kern);            \
    return ok_;                                                     \
  }())

}  // namespace fa

#define FA_HIDDEN __attribute__((visibility("hidden")))

// Per-slice dispatch tables, one translation unit per (element type, D).
extern "C" {
FA_HIDDEN fa::FwdFn fa_fwd_table_f16_32(int bm, int bn, int gh, int lse);
FA_HIDDEN fa::FwdFn fa_fwd_table_f16_64(int bm, int bn, int gh, int lse);
FA_HIDDEN fa::FwdFn fa_fwd_table_f16_128(int bm, int bn, int gh, int lse);
FA_HIDDEN fa::FwdFn fa_fwd_table_bf16_32(int bm, int bn, int gh, int lse);
FA_HIDDEN fa::FwdFn fa_fwd_table_bf16_64(int bm, int bn, int gh, int lse);
FA_HIDDEN fa::FwdFn fa_fwd_table_bf16_128(int bm, int bn, int gh, int lse);
FA_HIDDEN fa::BwdFn fa_bwd_table_f16_32(int bm, int bn);
FA_HIDDEN fa::BwdFn fa_bwd_table_f16_64(int bm, int bn);
FA_HIDDEN fa::BwdFn fa_bwd_table_f16_128(int bm, int bn);
FA_HIDDEN fa::BwdFn fa_bwd_table_bf16_32(int bm, int bn);
FA_HIDDEN fa::BwdFn fa_bwd_table_bf16_64(int bm, int bn);
FA_HIDDEN fa::BwdFn fa_bwd_table_bf16_128(int bm, int bn);
}
