// The gated delta rule on packed sequences (coli_cuda_delta_prompt) and on single
// tokens (coli_cuda_delta_step): what k_gdn_recur does inside the Gated DeltaNet
// layer, for prompts of any length.
//
//   S <- e^g S;  d = beta (v - S^T k);  S <- S + k d^T;  o = S^T q
// with k and q brought to unit length (and q times key_dim^-1/2),
// g = -e^A_log softplus(a + dt_bias), beta = sigmoid(b), S [key_dim][value_dim] fp32.
//
// Prompts go in chunks of 64 tokens.  With G the running sum of g within a chunk and
// S0 the state before it, the rule's d of all the chunk's tokens solve
//   (1 + A) d = beta (v - e^G k S0),   A[t][s] = beta_t e^(G_t - G_s) k_t . k_s, s < t,
// and then
//   o = e^G q S0 + P d,                P[t][s] = e^(G_t - G_s) q_t . k_s, s <= t,
//   S = e^G_63 S0 + sum_t e^(G_63 - G_t) k_t d_t^T.
// What does not need S0 (the inverse of 1 + A, times beta; P; the factors) is formed
// for all chunks at once (k_delta_chunk), the rest walks a sequence's chunks
// (k_delta_scan).  Every exponent is a sum of g over tokens s+1 .. t, never positive,
// taken as a difference of 64-bit running sums, which keeps it however far G has run.
// All products are fp32, or bf16 parts that make up fp32 (kTri below).
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdlib.h>
#include <string.h>

#include "sw_delta_plan.h"
#include "sw_serve.h"

namespace sw {
namespace {

constexpr int kKey = 128;   // largest key_dim
constexpr int kSlice = 32;  // value columns of a k_delta_scan workgroup

// fp32 values as sums of three bf16 ones: 8 bits each, the rest exactly 24 (a bf16
// value is one of them, an fp16 value two).  Products of such sums on the bf16 matrix
// cores, without the terms below 2^-24, are fp32 products in all but rounding, at 3
// (one factor bf16) to 6 instructions of 16 cycles where the fp32 matrix cores take 8
// of 32 for the same tile.
constexpr int kTri = 12 * 256;  // elements of a 64 x 64 lower triangle in 16 x 16 tiles, two of them zero
// Outputs of 16-bit types take two parts a factor, terms down to 2^-16 of a product: far
// below bf16's rounding, 2^-8 of the result, and below fp16's, 2^-11, unless the result
// is less than about a thirtieth of the products it sums; states always all three.
// One (chunk, value head) record of k_delta_chunk: the inverse of 1 + A times beta as
// three bf16 triangles, P as one for each part that outputs take; then per token e^G |k|^-1, e^G |q|^-1 key_dim^-1/2
// and e^(G_63 - G) |k|^-1, then e^G_63, in fp32.  A triangle's row tiles are
// [16 rows][32 columns], twice, then [16][64], twice (zero above the diagonal): a lane
// has its matrix operand of 32 columns in one load.
template <class T>
struct Rec {
  static constexpr int kParts = sizeof(T) == 4 ? 3 : 2;  // of a factor of the outputs
  static constexpr int kInv = 0, kP = 3 * kTri * 2, kX = kP + kParts * kTri * 2, kQ = kX + kChunk * 4, kR = kQ + kChunk * 4,
                       kEnd = kR + kChunk * 4, kBytes = kEnd + 16;
  static_assert(kBytes % 16 == 0, "records are 16-byte aligned");
};
__device__ __forceinline__ constexpr int tri_at(int i, int row) {  // element of row tile i's row, column 0
  return i < 2 ? 512 * i + 32 * row : 1024 * (i - 1) + 64 * row;
}

struct DeltaArgs {
  const void *q, *k, *v;
  void *out;
  const float *a, *b, *a_log, *dt_bias;
  const float *state;
  float *state_out;
  char *rec;
  long long q_stride, k_stride, v_stride;
  int kh, vh, dk, dv, seqs;
  int chunk_first;  // first chunk of each sequence in this pass
  int chunks;       // chunks of a sequence in one pass, at most
  int begin[kSeqs], rows[kSeqs], slot[kSeqs];
  int chunk0[kSeqs + 1];  // records of sequence s: chunk0[s] .. chunk0[s + 1] - 1
};

// The next bf16 part of two values, packed, and what is left of them: one conversion
// for both, whose halves are fp32 values as they stand.
__device__ __forceinline__ unsigned next_part(float &x, float &y) {
  const unsigned b = pack2<__bf16>(x, y);
  x -= __uint_as_float(b << 16);
  y -= __uint_as_float(b & 0xffff0000u);
  return b;
}
// x as three bf16 values, packed two by two
__device__ __forceinline__ void split3(const float (&x)[4], v2u (&p)[3]) {
  float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int k = 0; k < 3; k++) {
    p[k][0] = next_part(r[0], r[1]);
    p[k][1] = next_part(r[2], r[3]);
  }
}
template <class T>
constexpr int planes_of() {
  return sizeof(T) == 4 ? 3 : __is_same(T, __bf16) ? 1 : 2;
}

// Eight elements from 16-byte aligned memory.
template <class T>
__device__ __forceinline__ void load8(float (&x)[8], const T *p) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = ((const float4 *)p)[0], b = ((const float4 *)p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    typedef T v8t __attribute__((ext_vector_type(8)));
    const v8t a = *(const v8t *)p;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (float)a[e];
  }
}

// log decay of a token, floored where e^g has long been 0 in fp32, so that sums of it
// stay finite; a NaN stays
__device__ __forceinline__ float log_decay(float a_exp, float a, float dt) {
  const float g = -a_exp * softplus_ref(a + dt);
  return g < -128.0f ? -128.0f : g;
}

// ---------------------------------------------------------------------------
// single tokens
// ---------------------------------------------------------------------------
// One wave a (row, value head, 32 value columns): lane (r, c) = (lane / 8, lane % 8)
// holds 16 state rows x 4 columns, loaded as 16-byte pieces, eight lanes a 128-byte
// line.  The state is read and written once: HBM-bound; 16 rows of 64 heads x 128 x
// 128 (134 MB) 24 us, 5.6 TB/s, stored past the caches (31.5 us in calls one after
// another without that: the next call's reads waited for this one's writes).  S may be
// updated in place.
struct StepArgs {
  const void *q, *k, *v;
  void *out;
  const float *a, *b, *a_log, *dt_bias;
  const float *state;
  float *state_out;
  long long q_stride, k_stride, v_stride;
  int kh, vh, dk, dv, row0;
  int slot[kSeqs];
};
template <class T>
__global__ __launch_bounds__(256) void k_delta_step(StepArgs g) {
  __shared__ __align__(16) float s_q[4][kKey], s_k[4][kKey];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane >> 3, c = lane & 7;
  const int nsp = g.dv / 32, unit = blockIdx.x * 4 + wave;
  const int t = blockIdx.y;
  if (unit >= g.vh * nsp) return;  // no barrier below
  const int h = unit / nsp, j = (unit % nsp) * 32 + 4 * c, hk = h / (g.vh / g.kh);
  const size_t row = (size_t)g.row0 + t;
  const size_t at = ((size_t)g.slot[t] * g.vh + h) * g.dk * g.dv + j;
  float4 S[16];
#pragma unroll
  for (int m = 0; m < 16; m++) {
    const int i = 16 * r + m;
    S[m] = i < g.dk ? *(const float4 *)(g.state + at + (size_t)i * g.dv) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const T *qp = (const T *)g.q + row * g.q_stride + (size_t)hk * g.dk, *kp = (const T *)g.k + row * g.k_stride + (size_t)hk * g.dk;
  const float q0 = 2 * lane < g.dk ? (float)qp[2 * lane] : 0.f, q1 = 2 * lane < g.dk ? (float)qp[2 * lane + 1] : 0.f;
  const float k0 = 2 * lane < g.dk ? (float)kp[2 * lane] : 0.f, k1 = 2 * lane < g.dk ? (float)kp[2 * lane + 1] : 0.f;
  const T *vp = (const T *)g.v + row * g.v_stride + (size_t)h * g.dv + j;
  const float v[4] = {(float)vp[0], (float)vp[1], (float)vp[2], (float)vp[3]};
  const float beta = sigmoid_ref(g.b[row * g.vh + h]);
  const float decay = expf(log_decay(expf(g.a_log[h]), g.a[row * g.vh + h], g.dt_bias[h]));
  const float qn = 1.f / sqrtf(wave_sum_dpp(__builtin_fmaf(q0, q0, q1 * q1)) + 1e-6f) * (1.f / sqrtf((float)g.dk));
  const float kn = 1.f / sqrtf(wave_sum_dpp(__builtin_fmaf(k0, k0, k1 * k1)) + 1e-6f);
  float *sq = s_q[wave], *sk = s_k[wave];
  *(float2 *)(sq + 2 * lane) = make_float2(q0 * qn, q1 * qn);
  *(float2 *)(sk + 2 * lane) = make_float2(k0 * kn, k1 * kn);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  float kk[16], mem[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int m = 0; m < 16; m += 4) *(float4 *)(kk + m) = *(const float4 *)(sk + 16 * r + m);
#pragma unroll
  for (int m = 0; m < 16; m++) {
    S[m].x *= decay, S[m].y *= decay, S[m].z *= decay, S[m].w *= decay;
    mem[0] = __builtin_fmaf(S[m].x, kk[m], mem[0]);
    mem[1] = __builtin_fmaf(S[m].y, kk[m], mem[1]);
    mem[2] = __builtin_fmaf(S[m].z, kk[m], mem[2]);
    mem[3] = __builtin_fmaf(S[m].w, kk[m], mem[3]);
  }
  float d[4], o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < 4; e++) {
#pragma unroll
    for (int x = 8; x < 64; x <<= 1) mem[e] += __shfl_xor(mem[e], x);
    d[e] = (v[e] - mem[e]) * beta;
  }
#pragma unroll
  for (int m = 0; m < 16; m++) {
    const float q = sq[16 * r + m];
    S[m].x = __builtin_fmaf(kk[m], d[0], S[m].x);
    S[m].y = __builtin_fmaf(kk[m], d[1], S[m].y);
    S[m].z = __builtin_fmaf(kk[m], d[2], S[m].z);
    S[m].w = __builtin_fmaf(kk[m], d[3], S[m].w);
    o[0] = __builtin_fmaf(S[m].x, q, o[0]);
    o[1] = __builtin_fmaf(S[m].y, q, o[1]);
    o[2] = __builtin_fmaf(S[m].z, q, o[2]);
    o[3] = __builtin_fmaf(S[m].w, q, o[3]);
  }
#pragma unroll
  for (int m = 0; m < 16; m++) {
    const int i = 16 * r + m;
    if (i < g.dk) __builtin_nontemporal_store(__builtin_bit_cast(v4f, S[m]), (v4f *)(g.state_out + at + (size_t)i * g.dv));
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
#pragma unroll
    for (int x = 8; x < 64; x <<= 1) o[e] += __shfl_xor(o[e], x);
  if (r == 0) {
    T *op = (T *)g.out + (row * g.vh + h) * g.dv + j;
#pragma unroll
    for (int e = 0; e < 4; e++) op[e] = (T)o[e];
  }
}

// ---------------------------------------------------------------------------
// prompts: what a chunk has without its state
// ---------------------------------------------------------------------------
__device__ __forceinline__ v4f mfma_f32_16(float a, float b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma_b16(v4u a, v4u b, v4f c) { return Mat16<__bf16>::mul16(a, b, c); }
constexpr int kPitchB = kKey * 2 + 16;  // bytes of a 16-bit row in LDS: 16 rows' pieces lie in distinct banks
constexpr int kPitchF = kKey / 2 * 4 + 16;  // of half an fp32 row

// One workgroup a (chunk, key head).  The products of the chunk's keys with its keys
// and queries, as raw rows (their lengths divide the results), serve every value head
// of the key head: 10 lower tiles each, formed as K Q^T, so that a lane of the result
// holds four consecutive columns s of one row t.  Then a wave takes a value head:
// gates (token a lane) and their running sum, A and P tile by tile, the inverse:
// its four 16 x 16 diagonal tiles by substitution, all at once (lane = tile and
// column), the others from
//   T_ij = -(sum_{j < k <= i} T_ik A_kj) T_jj
// in transposed form on the fp32 matrix cores, where a result's registers are the next
// product's B operand as they stand.
// e^(G_t - G_s) off the diagonal tiles is e^(G_t - R) e^(R - G_s), R the sum at the end
// of s's tile: both exponents are negative, and a tile takes two factors a lane.
// Bound by the chains of a head's steps, 28 us a workgroup, two of which a compute unit
// holds (149 -> 110 us against one), and by the records it writes: 8,191 bf16 tokens of
// 64 value heads 108 us for 299 MB; five fp32 prompts, 1,764 tokens of 32 heads, 28 us.
// The inverse by 64 steps of substitution, and fp32 matrix products throughout: 290.
struct ChunkLds {
  static constexpr int kPairs = 0;                       // tiles of k k^T, then q k^T: [tile][lane] x 16 bytes
  static constexpr int kNorms = kPairs + 20 * 1024;      // |k|^-1, |q|^-1 key_dim^-1/2
  static constexpr int kWork = kNorms + 2 * kChunk * 4;  // raw rows, then per wave:
  static constexpr int kTile = 16 * 20 * 4;              // a 16 x 16 fp32 tile, rows of 80 bytes
  static constexpr int kWave = 10 * kTile + kChunk * (8 + 4 * 5);  // tiles of A, G, beta, factors
};
template <class T>
constexpr int chunk_lds() {
  constexpr int rows = 2 * kChunk * (sizeof(T) == 4 ? kPitchF : kPitchB), waves = 4 * ChunkLds::kWave;
  return ChunkLds::kWork + (rows > waves ? rows : waves);
}

template <class T>
__global__ __launch_bounds__(256) void k_delta_chunk(DeltaArgs g) {
  typedef ChunkLds L;
  typedef Rec<T> R;
  constexpr int kPitch = sizeof(T) == 4 ? kPitchF : kPitchB;
  extern __shared__ __align__(16) char lds[];
  v4f *s_pair = (v4f *)(lds + L::kPairs);
  float *s_kn = (float *)(lds + L::kNorms), *s_qn = s_kn + kChunk;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
  const int hk = blockIdx.y;
  const int s = find_span(g.chunk0, g.seqs, blockIdx.x);
  const int first = (blockIdx.x - g.chunk0[s] + g.chunk_first) * kChunk;
  const int t0 = g.begin[s] + first, n = min(kChunk, g.rows[s] - first);

  // a wave's first head's gates, on their way while the rows are
  const int rep = g.vh / g.kh;
  const size_t gate_at = (size_t)(t0 + min(lane, n - 1)) * g.vh;
  const int h_first = hk * rep + (wave < rep ? wave : 0);
  float a_ = g.a[gate_at + h_first], b_ = g.b[gate_at + h_first], al_ = g.a_log[h_first], dt_ = g.dt_bias[h_first];
  // Raw rows, zero beyond the sequence's end and beyond key_dim; fp32 ones in two halves,
  // which lets a compute unit hold two workgroups.
  constexpr int HALVES = sizeof(T) / 2, DP = kKey / HALVES;
  v4f acc[5];  // tiles wave, wave + 4, ..
#pragma unroll
  for (int i = 0; i < 5; i++) acc[i] = v4f{0.f, 0.f, 0.f, 0.f};
  auto tile_of = [](int u, int &i, int &j) {  // row and column tile, of k k^T up to 9, then of q k^T
    j = u < 10 ? u : u - 10;
    i = 0;
    while (j > i) j -= ++i;
  };
  float s2[2] = {0.0f, 0.0f};
#pragma unroll
  for (int half = 0; half < HALVES; half++) {
    const int t = threadIdx.x >> 2, p = threadIdx.x & 3;
#pragma unroll
    for (int m = 0; m < 2; m++) {
      const T *src = m ? (const T *)g.q + (size_t)(t0 + t) * g.q_stride + (size_t)hk * g.dk
                       : (const T *)g.k + (size_t)(t0 + t) * g.k_stride + (size_t)hk * g.dk;
      char *row = lds + L::kWork + (m * kChunk + t) * kPitch;
#pragma unroll
      for (int i = 0; i < DP / 32; i++) {
        const int c = p + 4 * i, d = half * DP + 8 * c;
        constexpr int V = sizeof(T) / 2;  // 16-byte pieces of eight elements
        v4u x[V];
#pragma unroll
        for (int u = 0; u < V; u++) x[u] = t < n && d < g.dk ? ((const v4u *)(src + d))[u] : v4u{0, 0, 0, 0};
        float f[8];
        load8(f, (const T *)x);
#pragma unroll
        for (int e = 0; e < 8; e++) s2[m] = __builtin_fmaf(f[e], f[e], s2[m]);
#pragma unroll
        for (int u = 0; u < V; u++) ((v4u *)(row + 8 * c * sizeof(T)))[u] = x[u];
      }
      if (half == HALVES - 1) {
        s2[m] += __shfl_xor(s2[m], 1);
        s2[m] += __shfl_xor(s2[m], 2);
        if (p == 0) (m ? s_qn : s_kn)[t] = 1.f / sqrtf(s2[m] + 1e-6f) * (m ? 1.f / sqrtf((float)g.dk) : 1.f);
      }
    }
    __syncthreads();
    const int dn = min(DP, g.dk - half * DP);
#pragma unroll
    for (int k = 0; k < 5; k++) {
      int i, j;
      tile_of(wave + 4 * k, i, j);
      const char *ks = lds + L::kWork + (16 * j + n16) * kPitch;
      const char *qt = lds + L::kWork + ((wave + 4 * k < 10 ? 0 : kChunk) + 16 * i + n16) * kPitch;
      if constexpr (sizeof(T) == 2) {
        for (int d = 0; d < dn; d += 32)
          acc[k] = Mat16<T>::mul16(*(const v4u *)(ks + 2 * d + 16 * kg), *(const v4u *)(qt + 2 * d + 16 * kg), acc[k]);
      } else {
        for (int d = 0; d < dn; d += 16) {
          const v4f x = *(const v4f *)(ks + 4 * d + 16 * kg), y = *(const v4f *)(qt + 4 * d + 16 * kg);
#pragma unroll
          for (int e = 0; e < 4; e++) acc[k] = mfma_f32_16(x[e], y[e], acc[k]);
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int k = 0; k < 5; k++) {
    const int u = wave + 4 * k;
    int i, j;
    tile_of(u, i, j);
    // row s = 16 j + 4 kg + e, column t = 16 i + n16
    const v4f kn = *(const v4f *)(s_kn + 16 * j + 4 * kg);
    s_pair[u * 64 + lane] = acc[k] * kn * (u < 10 ? s_kn : s_qn)[16 * i + n16];
  }
  __syncthreads();

  char *mine = lds + L::kWork + wave * L::kWave;
  float *s_a = (float *)mine;  // tiles [row s][t] of A^T; the diagonal ones become their inverses' transposes
  double *s_G = (double *)(s_a + 10 * 320);
  float *s_beta = (float *)(s_G + kChunk), *s_to = s_beta + kChunk, *s_from = s_to + kChunk;  // s_from [3][64]
  for (int w = wave; w < rep; w += 4) {
    const int h = hk * rep + w;
    char *rec = g.rec + ((size_t)blockIdx.x * g.vh + h) * R::kBytes;
    {
      const bool there = lane < n;
      if (w != wave) a_ = g.a[gate_at + h], b_ = g.b[gate_at + h], al_ = g.a_log[h], dt_ = g.dt_bias[h];
      const float gt = there ? log_decay(expf(al_), a_, dt_) : 0.0f;
      const double G = wave_incl_scan_dpp((double)gt), Gend = readlane_d63(G);
      const float eG = expf((float)G);
      ((float *)(rec + R::kX))[lane] = eG * s_kn[lane];
      ((float *)(rec + R::kQ))[lane] = eG * s_qn[lane];
      ((float *)(rec + R::kR))[lane] = expf((float)(Gend - G)) * s_kn[lane];
      if (lane == 0) *(float *)(rec + R::kEnd) = expf((float)Gend);
      s_G[lane] = G;
      s_beta[lane] = there ? sigmoid_ref(b_) : 0.0f;
      s_to[lane] = expf((float)(__shfl(G, lane | 15) - G));
#pragma unroll
      for (int j = 0; j < 3; j++) {
        const double R = __shfl(G, 16 * j + 15);  // by all lanes
        s_from[j * kChunk + lane] = (lane >> 4) > j ? expf((float)(G - R)) : 0.0f;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 4; i += 2)  // the tiles right of the diagonal that a 32-column operand holds
#pragma unroll
      for (int k = 0; k < 3; k++) {
        if (k < R::kParts) *(v2u *)(rec + R::kP + 2 * (k * kTri + tri_at(i, n16) + 16 * (i + 1) + 4 * kg)) = v2u{0, 0};
        *(v2u *)(rec + R::kInv + 2 * (k * kTri + tri_at(i, n16) + 16 * (i + 1) + 4 * kg)) = v2u{0, 0};
      }
    // A^T and P, tile (i, j): rows s = 16 j + 4 kg + e, column t = 16 i + n16
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int j = 0; j <= i; j++) {
        const int u = i * (i + 1) / 2 + j, t = 16 * i + n16;
        const v4f kk = s_pair[u * 64 + lane], qk = s_pair[(10 + u) * 64 + lane];
        const float beta = s_beta[t];
        float p[4];
        float *at = s_a + u * 320;
        if (j < i) {
          const float f = s_from[j * kChunk + t];
          const v4f e4 = *(const v4f *)(s_to + 16 * j + 4 * kg);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float x = f * e4[e];
            at[(4 * kg + e) * 20 + n16] = beta * x * kk[e];
            p[e] = x * qk[e];
          }
        } else {
          const double G = s_G[t];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int r = 4 * kg + e;
            const float x = r <= n16 ? expf((float)(G - s_G[16 * j + r])) : 0.0f;
            at[r * 20 + n16] = r < n16 ? beta * x * kk[e] : 0.0f;
            p[e] = r <= n16 ? x * qk[e] : 0.0f;
          }
        }
        v2u p3[3];
        split3(p, p3);
#pragma unroll
        for (int k = 0; k < R::kParts; k++)
          *(v2u *)(rec + R::kP + 2 * (k * kTri + tri_at(i, n16) + 16 * j + 4 * kg)) = p3[k];
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    // the diagonal tiles' inverses: lane (tile kg, column n16)
    {
      float *at = s_a + (kg * (kg + 1) / 2 + kg) * 320;
      float x[16];
#pragma unroll
      for (int r = 0; r < 16; r++) x[r] = r == n16 ? 1.0f : 0.0f;
#pragma unroll
      for (int u = 0; u < 15; u++) {
        float a16[16];
#pragma unroll
        for (int r = 4 * ((u + 1) / 4); r < 16; r += 4) *(v4f *)(a16 + r) = *(const v4f *)(at + u * 20 + r);
#pragma unroll
        for (int r = u + 1; r < 16; r++) x[r] = __builtin_fmaf(-a16[r], x[u], x[r]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      float *to = at + n16 * 20;
#pragma unroll
      for (int r = 0; r < 16; r += 4) *(v4f *)(to + r) = v4f{x[r], x[r + 1], x[r + 2], x[r + 3]};
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    v4f inv[4];  // T_jj^T, row s = n16, as an A operand
#pragma unroll
    for (int j = 0; j < 4; j++) inv[j] = *(const v4f *)(s_a + (j * (j + 1) / 2 + j) * 320 + n16 * 20 + 4 * kg);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      v4f T_[4];  // T_ij^T: row s = 4 kg + e, column t = n16
#pragma unroll
      for (int e = 0; e < 4; e++) T_[i][e] = s_a[(i * (i + 1) / 2 + i) * 320 + (4 * kg + e) * 20 + n16];
#pragma unroll
      for (int j = i - 1; j >= 0; j--) {
        v4f sum = v4f{0.f, 0.f, 0.f, 0.f}, y = sum;
#pragma unroll
        for (int k = j + 1; k <= i; k++) {
          const v4f ak = *(const v4f *)(s_a + (k * (k + 1) / 2 + j) * 320 + n16 * 20 + 4 * kg);
#pragma unroll
          for (int e = 0; e < 4; e++) sum = mfma_f32_16(ak[e], T_[k][e], sum);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) y = mfma_f32_16(-inv[j][e], sum[e], y);
        T_[j] = y;
      }
#pragma unroll
      for (int j = 0; j <= i; j++) {
        const v4f beta = *(const v4f *)(s_beta + 16 * j + 4 * kg);
        const float x[4] = {T_[j][0] * beta[0], T_[j][1] * beta[1], T_[j][2] * beta[2], T_[j][3] * beta[3]};
        v2u p3[3];
        split3(x, p3);
#pragma unroll
        for (int k = 0; k < 3; k++)
          *(v2u *)(rec + R::kInv + 2 * (k * kTri + tri_at(i, n16) + 16 * j + 4 * kg)) = p3[k];
      }
    }
    // the next head's values go where this one's are read
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// ---------------------------------------------------------------------------
// prompts: the state's walk over the chunks
// ---------------------------------------------------------------------------
// One workgroup of 8 waves a (value head, 32 value columns, sequence), chunk after
// chunk in four steps with a barrier between them:
//   keys, queries and the state's bf16 parts to LDS;
//   x = v - e^G |k|^-1 (k S0) and e^G |q|^-1 (q S0), a 16 x 16 tile of each a wave;
//   d = inverse x;
//   o = that + P d, and S = e^G_63 S0 + k^T (e^(G_63 - G) |k|^-1 d), two tiles a wave.
// The state slice stays in the accumulators of its update for the whole walk.  Every
// B operand ([column][8 consecutive terms] in LDS) is written from results whose lanes
// hold four consecutive rows of a column; k^T comes from k by the transposing LDS
// load.  What a chunk reads from memory is loaded into registers while the chunk
// before it is computed.
// Latency-bound: a chunk's four steps depend on each other, 3.9 us a chunk, 8,191 bf16
// tokens of 64 heads x 128 x 128 495 us on all compute units (matrix instructions busy
// for 17% of it, 463 MB fetched at 0.9 TB/s); without any load it would take 340 to
// 360, with all of them in cache 442.  In fp32, three planes of keys and queries, a
// workgroup takes all of a compute unit's LDS and a step 5.0 us (4,096 tokens of 32 heads
// 317 to 329): five prompts of 29 chunks in all, 32 heads, are 14.5 steps in turn on each
// compute unit, 93 us.  fp32 matrix instructions in place of the bf16
// parts took 1,662; slices of 16 columns 587 against 517, loads after the products 537
// against 514, padded LDS rows 520 against 502, loads free of branches 498.
template <class T>
struct ScanLds {
  static constexpr int NP = planes_of<T>();
  static constexpr int kRows = kChunk * 256;   // one plane of keys or queries: [token][128]
  static constexpr int kTok = kSlice * 128;    // one plane of x or d: [column][64 tokens]
  static constexpr int kState = kSlice * 256;  // one plane of the state: [column][128]
  static constexpr int kK = 0, kQ = NP * kRows, kS = 2 * NP * kRows;
  static constexpr int kD = kS;                                 // d lies where the state was
  static constexpr int kX = kS + 3 * kState, kR = kX + 3 * kTok, kAll = kR + 3 * kTok;
};
// byte of a 16-byte chunk: rows of 16 chunks (keys, queries, state columns), of 8 (x, d)
__device__ __forceinline__ int wide_at(int row, int chunk) { return row * 256 + ((chunk ^ chunk_xor<16>(row)) << 4); }
__device__ __forceinline__ int tok_at(int row, int chunk) { return row * 128 + ((chunk ^ ((row >> 1) & 7)) << 4); }
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"
typedef short v4s __attribute__((ext_vector_type(4)));
// 16 lanes read four rows x 16 columns, four 16-bit values a lane, and get the four
// rows of one column each
__device__ __forceinline__ v2u lds_transposed(const void *p) {
  return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                     (__attribute__((address_space(3))) v4s *)(const __attribute__((address_space(3))) void *)p));
}
#pragma clang diagnostic pop

template <class T>
__global__ __launch_bounds__(512) void k_delta_scan(DeltaArgs g) {
  typedef ScanLds<T> L;
  typedef Rec<T> R;
  constexpr int NP = L::NP, V = sizeof(T) / 2;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, n16 = lane & 15, kg = lane >> 4;
  const int rt = __builtin_amdgcn_readfirstlane(wave & 3), ct = __builtin_amdgcn_readfirstlane(wave >> 2);  // row and column tile
  const int nsl = g.dv / kSlice, units = g.vh * nsl, s = blockIdx.y;
  // the slices of a value head, and the value heads of a key head, on one die: blocks
  // go to the eight dies in turn
  const int unit = units % 8 == 0 ? (blockIdx.x % 8) * (units / 8) + blockIdx.x / 8 : blockIdx.x;
  const int h = unit / nsl, col = (unit % nsl) * kSlice + 16 * ct + n16;  // this lane's value column
  const int hk = h / (g.vh / g.kh);
  const int rows = g.rows[s];
  const int c0 = g.chunk_first, c1 = min(c0 + g.chunks, (rows + kChunk - 1) / kChunk);
  const size_t at = ((size_t)g.slot[s] * g.vh + h) * g.dk * g.dv + col;
  const float *from = c0 > 0 ? g.state_out : g.state;
  v4f S[2];  // rows 32 rt + 16 i + 4 kg + e
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int r = 32 * rt + 16 * i + 4 * kg + e;
      S[i][e] = r < g.dk ? from[at + (size_t)r * g.dv] : 0.0f;
    }

  // a chunk's part of this thread, and where the next one's lies
  const int lr = tid >> 3, lc = tid & 7;  // row, and pieces lc and lc + 8 of eight elements
  const size_t row0 = (size_t)g.begin[s] + (size_t)c0 * kChunk;
  const T *kp = (const T *)g.k + (row0 + lr) * g.k_stride + (size_t)hk * g.dk + 8 * lc;
  const T *qp = (const T *)g.q + (row0 + lr) * g.q_stride + (size_t)hk * g.dk + 8 * lc;
  const T *vp = (const T *)g.v + (row0 + 16 * rt + 4 * kg) * g.v_stride + (size_t)h * g.dv + col;
  T *op = (T *)g.out + ((row0 + 16 * rt + 4 * kg) * g.vh + h) * g.dv + col;
  const size_t orow = (size_t)g.vh * g.dv;
  const char *rec = g.rec + ((size_t)g.chunk0[s] * g.vh + h) * R::kBytes;
  const int tri = 2 * (tri_at(rt, n16) + 8 * kg), tok = 4 * (16 * rt + 4 * kg);
  v4u kraw[2][V], qraw[2][V], inv[2][3], pr[2][R::kParts];
  T vv[4];
  v4f fx, fq, fr;
  float fe;
  auto load_rows = [&](int c) {
    const int n = rows - c * kChunk;
    if (n >= kChunk && g.dk == kKey) {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int u = 0; u < V; u++) {
          kraw[i][u] = ((const v4u *)(kp + 64 * i))[u];
          qraw[i][u] = ((const v4u *)(qp + 64 * i))[u];
        }
#pragma unroll
      for (int e = 0; e < 4; e++) vv[e] = vp[(size_t)e * g.v_stride];
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const bool in = lr < n && 8 * lc + 64 * i < g.dk;
#pragma unroll
        for (int u = 0; u < V; u++) {
          kraw[i][u] = in ? ((const v4u *)(kp + 64 * i))[u] : v4u{0, 0, 0, 0};
          qraw[i][u] = in ? ((const v4u *)(qp + 64 * i))[u] : v4u{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int e = 0; e < 4; e++) vv[e] = 16 * rt + 4 * kg + e < n ? vp[(size_t)e * g.v_stride] : (T)0.0f;
    }
    kp += (size_t)kChunk * g.k_stride;
    qp += (size_t)kChunk * g.q_stride;
    vp += (size_t)kChunk * g.v_stride;
  };
  auto load_triangle = [&](auto &to, int which) {
    constexpr int parts = sizeof(to[0]) / sizeof(v4u);
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if (2 * i > rt) break;
#pragma unroll
      for (int p = 0; p < parts; p++) to[i][p] = *(const v4u *)(rec + which + 2 * p * kTri + tri + 64 * i);
    }
  };
  auto load_factors = [&] {
    fx = *(const v4f *)(rec + R::kX + tok);
    fq = *(const v4f *)(rec + R::kQ + tok);
    fr = *(const v4f *)(rec + R::kR + tok);
    fe = *(const float *)(rec + R::kEnd);
  };
  // eight raw elements as NP bf16 pieces of 16 bytes
  auto put_planes = [&](char *to, const v4u (&raw)[V]) {
    if constexpr (NP == 1) {
      *(v4u *)to = raw[0];
    } else {
      float x[8];
      load8(x, (const T *)raw);
#pragma unroll
      for (int p = 0; p < NP; p++) {
        v4u w;
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = next_part(x[2 * e], x[2 * e + 1]);
        *(v4u *)(to + p * L::kRows) = w;
      }
    }
  };
  // four consecutive rows of a column as three bf16 pieces of 8 bytes
  auto put_split = [&](char *to, int plane, const v4f &x, int parts = 3) {
    const float x4[4] = {x[0], x[1], x[2], x[3]};
    v2u p3[3];
    split3(x4, p3);
#pragma unroll
    for (int p = 0; p < 3; p++)
      if (p < parts) *(v2u *)(to + p * plane) = p3[p];
  };

  if (c0 < c1) {
    load_rows(c0);
    load_triangle(inv, R::kInv);
    load_triangle(pr, R::kP);
    load_factors();
  }
  for (int c = c0; c < c1; c++) {
    const int n = rows - c * kChunk;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      put_planes(lds + L::kK + wide_at(lr, lc + 8 * i), kraw[i]);
      put_planes(lds + L::kQ + wide_at(lr, lc + 8 * i), qraw[i]);
      put_split(lds + L::kS + wide_at(16 * ct + n16, 4 * rt + 2 * i + (kg >> 1)) + 8 * (kg & 1), L::kState, S[i]);
    }
    const v4f v_ = v4f{(float)vv[0], (float)vv[1], (float)vv[2], (float)vv[3]};
    lds_barrier();
    // the next chunk's loads go out a few a step: a wave waits to issue when many are
    if (c + 1 < c1) load_rows(c + 1);
    rec += (size_t)g.vh * R::kBytes;
    v4f ks = v4f{0.f, 0.f, 0.f, 0.f}, o = ks;
#pragma unroll
    for (int d = 0; d < kKey; d += 32) {
      if (d >= g.dk) break;
      v4u kf[NP], qf[NP], sf[3];
#pragma unroll
      for (int p = 0; p < NP; p++) {
        kf[p] = *(const v4u *)(lds + L::kK + p * L::kRows + wide_at(16 * rt + n16, d / 8 + kg));
        qf[p] = *(const v4u *)(lds + L::kQ + p * L::kRows + wide_at(16 * rt + n16, d / 8 + kg));
      }
#pragma unroll
      for (int p = 0; p < 3; p++)
        sf[p] = *(const v4u *)(lds + L::kS + p * L::kState + wide_at(16 * ct + n16, d / 8 + kg));
#pragma unroll
      for (int p = 0; p < NP; p++)
#pragma unroll
        for (int r = 0; r + p < 3; r++) {
          ks = mfma_b16(kf[p], sf[r], ks);
          if (r + p < R::kParts) o = mfma_b16(qf[p], sf[r], o);
        }
    }
    put_split(lds + L::kX + tok_at(16 * ct + n16, 2 * rt + (kg >> 1)) + 8 * (kg & 1), L::kTok, v_ - fx * ks);
    o *= fq;
    lds_barrier();
    auto triangle = [&](v4f acc, const auto &tr, const char *b) {
      constexpr int parts = sizeof(tr[0]) / sizeof(v4u);
#pragma unroll
      for (int i = 0; i < 2; i++) {
        if (2 * i > rt) break;
        v4u bf[parts];
#pragma unroll
        for (int p = 0; p < parts; p++) bf[p] = *(const v4u *)(b + p * L::kTok + tok_at(16 * ct + n16, 4 * i + kg));
#pragma unroll
        for (int p = 0; p < parts; p++)
#pragma unroll
          for (int r = 0; r + p < parts; r++) acc = mfma_b16(tr[i][p], bf[r], acc);
      }
      return acc;
    };
    const v4f d = triangle(v4f{0.f, 0.f, 0.f, 0.f}, inv, lds + L::kX);
    if (c + 1 < c1) load_triangle(inv, R::kInv);
    put_split(lds + L::kD + tok_at(16 * ct + n16, 2 * rt + (kg >> 1)) + 8 * (kg & 1), L::kTok, d, R::kParts);
    put_split(lds + L::kR + tok_at(16 * ct + n16, 2 * rt + (kg >> 1)) + 8 * (kg & 1), L::kTok, fr * d);
    lds_barrier();
    o = triangle(o, pr, lds + L::kD);
    const float fe_ = fe;
    if (c + 1 < c1) {
      load_triangle(pr, R::kP);
      load_factors();
    }
    if (n >= kChunk) {
#pragma unroll
      for (int e = 0; e < 4; e++) op[e * orow] = (T)o[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (16 * rt + 4 * kg + e < n) op[e * orow] = (T)o[e];
    }
    op += kChunk * orow;
    S[0] *= fe_;
    S[1] *= fe_;
#pragma unroll
    for (int i = 0; i < 2; i++) {  // tokens 32 i ..
      v4u bf[3];
#pragma unroll
      for (int p = 0; p < 3; p++)
        bf[p] = *(const v4u *)(lds + L::kR + p * L::kTok + tok_at(16 * ct + n16, 4 * i + kg));
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
        for (int p = 0; p < NP; p++) {
          const char *kp = lds + L::kK + p * L::kRows + 8 * (n16 & 1);
          const int row = 32 * i + 8 * kg + (n16 >> 2), chunk = 4 * rt + 2 * m + ((n16 & 3) >> 1);
          const v2u lo = lds_transposed(kp + wide_at(row, chunk)), hi = lds_transposed(kp + wide_at(row + 4, chunk));
#pragma unroll
          for (int r = 0; r + p < 3; r++) S[m] = mfma_b16(v4u{lo[0], lo[1], hi[0], hi[1]}, bf[r], S[m]);
        }
    }
    lds_barrier();
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int r = 32 * rt + 16 * i + 4 * kg + e;
      if (r < g.dk) g.state_out[at + (size_t)r * g.dv] = S[i][e];
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool delta_ok(const char *name, const ColiDelta *d, const void *out, const void *q, const void *k, const void *v,
              const float *a, const float *b, const float *a_log, const float *dt_bias, const float *state,
              const float *state_out, const int *slot, int n) {
  if (!d) return fail_arg("%s: null description", name), false;
  if (!type_bytes(d->type)) return fail_arg("%s: unknown element type %d", name, d->type), false;
  if (d->key_heads <= 0 || d->value_heads <= 0 || d->value_heads % d->key_heads || d->value_heads > 65535)
    return fail_arg("%s: value_heads %d (1..65535) must be a multiple of key_heads %d", name, d->value_heads, d->key_heads),
           false;
  if (d->key_dim <= 0 || d->key_dim > kKey || d->key_dim % 8 || d->value_dim <= 0 || d->value_dim > 256 || d->value_dim % 32)
    return fail_arg("%s: key_dim %d must be a multiple of 8 up to 128, value_dim %d a multiple of 32 up to 256", name,
                    d->key_dim, d->value_dim),
           false;
  if (d->slots <= 0) return fail_arg("%s: no state slots", name), false;
  if (!out || !q || !k || !v || !a || !b || !a_log || !dt_bias || !state || !state_out)
    return fail_arg("%s: null tensor", name), false;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out) || !aligned16(state) || !aligned16(state_out) ||
      d->q_stride % 8 || d->k_stride % 8 || d->v_stride % 8 || d->q_stride < 0 || d->k_stride < 0 || d->v_stride < 0)
    return fail_arg("%s: tensors must be 16-byte aligned, strides non-negative multiples of 8 elements", name), false;
  if (((uintptr_t)a | (uintptr_t)b | (uintptr_t)a_log | (uintptr_t)dt_bias) & 3)
    return fail_arg("%s: gates must be 4-byte aligned", name), false;
  if (n < 0 || (n && !slot)) return fail_arg("%s: null slots or negative count", name), false;
  for (int i = 0; i < n; i++)
    if (slot[i] < 0 || slot[i] >= d->slots)
      return fail_arg("%s: slot[%d] = %d is outside 0..%d", name, i, slot[i], d->slots - 1), false;
  // a slot named twice would have two new states
  int twice = -1;
  if (n <= 64) {
    for (int i = 0; i < n; i++)
      for (int j = 0; j < i; j++)
        if (slot[i] == slot[j]) twice = i;
  } else {
    unsigned char *seen = (unsigned char *)calloc((size_t)d->slots / 8 + 1, 1);
    if (!seen) return fail_arg("%s: out of host memory", name), false;
    for (int i = 0; i < n; i++) {
      if (seen[slot[i] >> 3] >> (slot[i] & 7) & 1) twice = i;
      seen[slot[i] >> 3] |= (unsigned char)(1 << (slot[i] & 7));
    }
    free(seen);
  }
  if (twice >= 0) return fail_arg("%s: slot %d is named twice", name, slot[twice]), false;
  return true;
}

template <class T>
int launch_delta(const char *name, const DeltaArgs &g, int chunks, hipStream_t st) {
  constexpr int chunk = chunk_lds<T>(), scan = ScanLds<T>::kAll;
  static_assert(chunk <= 160 * 1024 && scan <= 160 * 1024, "LDS of a compute unit");
  hipError_t e = hipFuncSetAttribute((const void *)k_delta_chunk<T>, hipFuncAttributeMaxDynamicSharedMemorySize, chunk);
  if (e == hipSuccess) e = hipFuncSetAttribute((const void *)k_delta_scan<T>, hipFuncAttributeMaxDynamicSharedMemorySize, scan);
  if (e != hipSuccess) return fail_hip(name, e);
  if (chunks) k_delta_chunk<T><<<dim3(chunks, g.kh), 256, chunk, st>>>(g);
  k_delta_scan<T><<<dim3(g.vh * (g.dv / kSlice), g.seqs), 512, scan, st>>>(g);
  return 0;
}

}  // namespace
}  // namespace sw

using namespace sw;

extern "C" int coli_cuda_delta_step(ColiCuda *ctx, const ColiDelta *d, void *out, const void *q, const void *k,
                                    const void *v, const float *a, const float *b, const float *a_log,
                                    const float *dt_bias, const float *state, float *state_out, const int *slot, int rows) {
  static const char *name = "coli_cuda_delta_step";
  if (!delta_ok(name, d, out, q, k, v, a, b, a_log, dt_bias, state, state_out, slot, rows)) return -1;
  if (!ctx) return fail_arg("%s: null context", name);
  OnDevice on(ctx);
  StepArgs g;
  memset(&g, 0, sizeof(g));
  g.q = q, g.k = k, g.v = v;
  g.out = out;
  g.a = a, g.b = b, g.a_log = a_log, g.dt_bias = dt_bias;
  g.state = state;
  g.state_out = state_out;
  g.q_stride = d->q_stride, g.k_stride = d->k_stride, g.v_stride = d->v_stride;
  g.kh = d->key_heads, g.vh = d->value_heads, g.dk = d->key_dim, g.dv = d->value_dim;
  const unsigned units = (unsigned)g.vh * (g.dv / 32);
  for (int r0 = 0; r0 < rows; r0 += kSeqs) {
    const int n = rows - r0 < kSeqs ? rows - r0 : kSeqs;
    g.row0 = r0;
    memcpy(g.slot, slot + r0, n * sizeof(int));
    const dim3 grid((units + 3) / 4, n);
    if (d->type == COLI_TYPE_F32)
      k_delta_step<float><<<grid, 256, 0, ctx->stream>>>(g);
    else if (d->type == COLI_TYPE_F16)
      k_delta_step<_Float16><<<grid, 256, 0, ctx->stream>>>(g);
    else
      k_delta_step<__bf16><<<grid, 256, 0, ctx->stream>>>(g);
  }
  return launch_status(name);
}

extern "C" int coli_cuda_delta_prompt(ColiCuda *ctx, const ColiDelta *d, void *out, const void *q, const void *k,
                                      const void *v, const float *a, const float *b, const float *a_log,
                                      const float *dt_bias, const float *state, float *state_out, const int *start,
                                      const int *slot, int sequences) {
  static const char *name = "coli_cuda_delta_prompt";
  if (!delta_ok(name, d, out, q, k, v, a, b, a_log, dt_bias, state, state_out, slot, sequences)) return -1;
  if (sequences && !start) return fail_arg("%s: null start", name);
  if (sequences && start[0] < 0) return fail_arg("%s: start[0] is negative", name);
  for (int s = 0; s < sequences; s++)
    if (start[s + 1] < start[s] || start[s + 1] > INT_MAX - kChunk)  // a chunk behind the last row is an int too
      return fail_arg("%s: sequence %d has rows %d..%d", name, s, start[s], start[s + 1]);
  if (!ctx) return fail_arg("%s: null context", name);
  OnDevice on(ctx);
  DeltaArgs g;
  memset(&g, 0, sizeof(g));
  g.q = q, g.k = k, g.v = v;
  g.out = out;
  g.a = a, g.b = b, g.a_log = a_log, g.dt_bias = dt_bias;
  g.state = state;
  g.state_out = state_out;
  g.q_stride = d->q_stride, g.k_stride = d->k_stride, g.v_stride = d->v_stride;
  g.kh = d->key_heads, g.vh = d->value_heads, g.dk = d->key_dim, g.dv = d->value_dim;
  const size_t chunk_bytes = (size_t)g.vh * (d->type == COLI_TYPE_F32 ? Rec<float>::kBytes : Rec<__bf16>::kBytes);
  const int most = delta_sequences(kSeqs, chunk_bytes);
  for (int s0 = 0; s0 < sequences; s0 += most) {
    const int n = sequences - s0 < most ? sequences - s0 : most;
    // long sequences first: their walk takes longest
    for (int s = 0; s < n; s++) {
      const int rows = start[s0 + s + 1] - start[s0 + s];
      int i = s;
      for (; i > 0 && g.rows[i - 1] < rows; i--) {
        g.begin[i] = g.begin[i - 1];
        g.rows[i] = g.rows[i - 1];
        g.slot[i] = g.slot[i - 1];
      }
      g.begin[i] = start[s0 + s];
      g.rows[i] = rows;
      g.slot[i] = slot[s0 + s];
    }
    const int longest = (int)chunks_of(g.rows[0]);
    g.chunk_first = 0;
    do {  // the first pass takes empty sequences along, which keep their state
      g.seqs = g.chunk_first ? delta_live(g.rows, n, g.chunk_first) : n;
      g.chunks = (int)delta_pass(g.rows, n, g.chunk_first, chunk_bytes);
      for (int s = 0; s < g.seqs; s++) {
        const int left = (int)chunks_of(g.rows[s]) - g.chunk_first;
        g.chunk0[s + 1] = g.chunk0[s] + (left < g.chunks ? left : g.chunks);
      }
      const int chunks = g.chunk0[g.seqs];
      const size_t bytes = (size_t)(chunks ? chunks : 1) * chunk_bytes;
      if (ensure_room(ctx, kScrDelta, bytes, bytes / 2 * 3 < kDeltaRecords ? bytes / 2 * 3 : kDeltaRecords, name)) return -1;
      g.rec = (char *)ctx->scratch[kScrDelta];
      const int rc = d->type == COLI_TYPE_F32   ? launch_delta<float>(name, g, chunks, ctx->stream)
                     : d->type == COLI_TYPE_F16 ? launch_delta<_Float16>(name, g, chunks, ctx->stream)
                                                : launch_delta<__bf16>(name, g, chunks, ctx->stream);
      if (rc) return -1;
      g.chunk_first += g.chunks;
    } while (g.chunk_first < longest);
  }
  return launch_status(name);
}
