// Shared by the paged-cache kernels (paged.hip) and the packed Gated DeltaNet
// kernels (delta.hip): the three element types, their matrix instructions, and
// the host-side checks of packed sequences.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "sw_backend.h"
#include "sw_device.h"

namespace sw {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));

constexpr int kSeqs = 128;  // sequences of one launch: their bounds travel as kernel arguments

// 16 bytes of eight 16-bit values in the matrix instructions of their type:
// 16x16x32: lane l gives A[l % 16][8 (l / 16) + j] and B[8 (l / 16) + j][l % 16],
//           holds D[4 (l / 16) + i][l % 16];
// 32x32x16: lane l gives A[l % 32][8 (l / 32) + j] and B[8 (l / 32) + j][l % 32],
//           holds D[8 (i / 4) + 4 (l / 32) + i % 4][l % 32].
// Any order of the contraction index serves, as long as A and B agree on it.
template <class T>
struct Mat16;
template <>
struct Mat16<_Float16> {
  static __device__ __forceinline__ v4f mul16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v16f mul32(v4u a, v4u b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  }
};
template <>
struct Mat16<__bf16> {
  static __device__ __forceinline__ v4f mul16(v4u a, v4u b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v16f mul32(v4u a, v4u b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  }
};

// two fp32 values rounded to nearest into one register of T
template <class T>
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
  typedef T v2t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(unsigned, v2t{(T)lo, (T)hi});
}

// sigmoid of a gate: exp overflows to inf for far negative ones, which gives 0
__device__ __forceinline__ float gate_sigmoid(float g) { return 1.0f / (1.0f + expf(-g)); }

// A barrier that waits for this wave's LDS accesses alone: __syncthreads would also
// wait for loads in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Rows of 16-byte chunks in LDS without padding: chunk c of row r lies at c ^
// chunk_xor(r).  For CPR chunks a row: bit by bit a sum of row bits, so that rows which
// differ by a constant differ by a constant here too; chosen so that 16 rows of a
// fragment of 32 or 16 columns, taken in the hardware's groups of 16 lanes, and the
// rows that a transposing load takes together lie in distinct banks.
template <int CPR>
__host__ __device__ constexpr int chunk_xor(int r) {
  return CPR == 8 ? ((r & 2) << 1) | ((r >> 1) & 2) | ((r >> 3) & 1)
                  : ((r & 3) << 2) | (((r >> 1) ^ (r >> 2)) & 2) | ((r >> 3) & 1);
}

// The last i with first[i] <= x among n + 1 ascending bounds in kernel arguments,
// x < first[n]: every lane compares its own entries, so one load finds it.
__device__ __forceinline__ int find_span(const int *first, int n, int x) {
  const int lane = threadIdx.x & 63;
  int found = 0;
  for (int i0 = 0; i0 < n; i0 += 64) {
    const int i = i0 + lane;
    found += __builtin_popcountll(__ballot(i < n && first[i] <= x));
  }
  return found - 1;
}

// x / d for 0 <= x < 2^31 by one multiplication: with 2^(l-1) < d <= 2^l and
// m = floor(2^32 (2^l - d) / d) + 1, x / d = (hi(m x) + x) >> l.
struct FastDiv {
  unsigned m;
  int l, d;
};
inline FastDiv fast_div(int d) {
  int l = 0;
  while ((1ll << l) < d) l++;
  return {(unsigned)((((1ull << l) - (unsigned long long)d) << 32) / (unsigned long long)d + 1), l, d};
}
__device__ __forceinline__ int div_by(const FastDiv &f, int x) {
  return (int)((__umulhi(f.m, (unsigned)x) + (unsigned)x) >> f.l);
}

// The caller's device stays current; the context's is current in between.
struct OnDevice {
  int before = -1;
  explicit OnDevice(const ColiCuda *ctx) {
    int now = -1;
    if (hipGetDevice(&now) == hipSuccess && now != ctx->device && hipSetDevice(ctx->device) == hipSuccess) before = now;
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
  OnDevice(const OnDevice &) = delete;
  OnDevice &operator=(const OnDevice &) = delete;
};

// ensure_scratch for sizes that creep up from call to call: where the slot has to grow,
// which waits for the stream, it grows to `room`, or to what is needed if that cannot be had.
inline int ensure_room(ColiCuda *ctx, Scratch which, size_t bytes, size_t room, const char *where) {
  if (ctx->scratch_cap[which] >= bytes) return 0;
  if (room > bytes) {
    if (!ensure_scratch(ctx, which, room, where)) return 0;
    (void)hipGetLastError();
  }
  return ensure_scratch(ctx, which, bytes, where);
}

inline int type_bytes(int type) { return type == COLI_TYPE_F32 ? 4 : type == COLI_TYPE_F16 || type == COLI_TYPE_BF16 ? 2 : 0; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace sw
