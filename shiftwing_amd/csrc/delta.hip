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
// All products are fp32.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdlib.h>
#include <string.h>

#include "sw_serve.h"

namespace sw {
namespace {

constexpr int kChunk = 64;
constexpr int kKey = 128;   // largest key_dim
constexpr int kSlice = 32;  // value columns of a k_delta_scan workgroup
// one (chunk, value head) record of k_delta_chunk, in floats: the inverse and P, row
// by row, then per token e^G |k|^-1, e^G |q|^-1 key_dim^-1/2 and e^(G_63 - G) |k|^-1,
// then e^G_63
constexpr int kRecInv = 0, kRecP = kChunk * kChunk, kRecX = 2 * kChunk * kChunk, kRecQ = kRecX + kChunk,
              kRecR = kRecQ + kChunk, kRecEnd = kRecR + kChunk, kRec = kRecEnd + kChunk;

struct DeltaArgs {
  const void *q, *k, *v;
  void *out;
  const float *a, *b, *a_log, *dt_bias;
  const float *state;
  float *state_out;
  float *rec;
  long long q_stride, k_stride, v_stride;
  int kh, vh, dk, dv, seqs;
  int chunk_first;           // k_delta_chunk / k_delta_scan: first chunk of each sequence in this pass
  int chunks;                // chunks of a sequence in one pass, at most
  int start[kSeqs + 1], slot[kSeqs];
  int chunk0[kSeqs + 1];     // records of sequence s: chunk0[s] .. chunk0[s + 1] - 1
};

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
// line.  The state is read and written once: HBM-bound.  S may be updated in place.
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
    if (i < g.dk) *(float4 *)(g.state_out + at + (size_t)i * g.dv) = S[m];
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

// A chunk's raw rows of one key head as fp32, [token][kPitch], zero beyond the
// sequence's end and beyond key_dim, and (sq, sk not null) the inverse lengths.
constexpr int kPitch = kKey + 4;
template <class T>
__device__ __forceinline__ void stage_rows(float *rows, const T *src, long long stride, int n, int dk, float *inv) {
  const int t = threadIdx.x >> 2, p = threadIdx.x & 3;
  float s2 = 0.0f;
  for (int c = p; c < kKey / 8; c += 4) {
    float x[8];
    if (t < n && 8 * c < dk) {
      load8(x, src + (size_t)t * stride + 8 * c);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = 0.0f;
    }
#pragma unroll
    for (int e = 0; e < 8; e++) s2 = __builtin_fmaf(x[e], x[e], s2);
    *(float4 *)(rows + t * kPitch + 8 * c) = make_float4(x[0], x[1], x[2], x[3]);
    *(float4 *)(rows + t * kPitch + 8 * c + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
  if (!inv) return;
  s2 += __shfl_xor(s2, 1);
  s2 += __shfl_xor(s2, 2);
  if (p == 0) inv[t] = 1.f / sqrtf(s2 + 1e-6f);
}

// One workgroup a (chunk, key head).  The products k k^T and q k^T of the chunk (their
// lower triangles, in 16 x 16 tiles) serve every value head of the key head; then a
// wave takes a value head: lane t holds token t's gates, their running sum is a scan
// of the wave, and lane j solves column j of the inverse by forward substitution,
// x_t = (t == j) - sum_{s < t} A[t][s] x_s, the column in registers and A's row read
// from LDS by all lanes at once.
constexpr int kTri = kChunk + 4;  // pitch of the triangles
template <class T>
__global__ __launch_bounds__(256) void k_delta_chunk(DeltaArgs g) {
  extern __shared__ __align__(16) float lds[];
  float *s_k = lds, *s_q = lds + kChunk * kPitch;                       // raw rows
  float *s_kk = s_q + kChunk * kPitch, *s_qk = s_kk + kChunk * kTri;    // triangles
  float *s_kn = s_qk + kChunk * kTri, *s_qn = s_kn + kChunk;
  float *s_a = lds;                                                     // per wave, over the rows
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
  const int hk = blockIdx.y;
  const int s = find_span(g.chunk0, g.seqs, blockIdx.x);
  const int c = blockIdx.x - g.chunk0[s] + g.chunk_first;
  const int t0 = g.start[s] + c * kChunk, n = min(kChunk, g.start[s + 1] - t0);
  stage_rows(s_k, (const T *)g.k + (size_t)t0 * g.k_stride + (size_t)hk * g.dk, g.k_stride, n, g.dk, s_kn);
  stage_rows(s_q, (const T *)g.q + (size_t)t0 * g.q_stride + (size_t)hk * g.dk, g.q_stride, n, g.dk, s_qn);
  __syncthreads();
  const float dks = 1.f / sqrtf((float)g.dk);
  for (int u = wave; u < 20; u += 4) {  // 10 lower tiles of k k^T, 10 of q k^T
    int v = u < 10 ? u : u - 10, ti = 0;
    while (v > ti) v -= ++ti;
    const float *rows = u < 10 ? s_k : s_q;
    v4f acc = v4f{0.f, 0.f, 0.f, 0.f};
    for (int i = 0; i < g.dk; i += 16) {
      const float4 x = *(const float4 *)(rows + (16 * ti + n16) * kPitch + i + 4 * kg);
      const float4 y = *(const float4 *)(s_k + (16 * v + n16) * kPitch + i + 4 * kg);
      acc = mfma_f32_16(x.x, y.x, acc);
      acc = mfma_f32_16(x.y, y.y, acc);
      acc = mfma_f32_16(x.z, y.z, acc);
      acc = mfma_f32_16(x.w, y.w, acc);
    }
    const float ncol = s_kn[16 * v + n16];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = 16 * ti + 4 * kg + i;
      const float f = u < 10 ? s_kn[r] : s_qn[r] * dks;
      (u < 10 ? s_kk : s_qk)[r * kTri + 16 * v + n16] = acc[i] * f * ncol;
    }
  }
  __syncthreads();
  const int rep = g.vh / g.kh;
  float *A = s_a + wave * kChunk * kChunk;
  for (int w = wave; w < rep; w += 4) {
    const int h = hk * rep + w;
    float *rec = g.rec + ((size_t)blockIdx.x * g.vh + h) * kRec;
    const bool there = lane < n;
    const size_t tok = (size_t)(t0 + (there ? lane : 0)) * g.vh + h;
    const float gt = there ? log_decay(expf(g.a_log[h]), g.a[tok], g.dt_bias[h]) : 0.0f;
    const float beta = there ? sigmoid_ref(g.b[tok]) : 0.0f;
    const double G = wave_incl_scan_dpp((double)gt);
    const double Gend = readlane_d63(G);
    rec[kRecX + lane] = expf((float)G) * s_kn[lane];
    rec[kRecQ + lane] = expf((float)G) * s_qn[lane] * dks;
    rec[kRecR + lane] = expf((float)(Gend - G)) * s_kn[lane];
    if (lane == 0) rec[kRecEnd] = expf((float)Gend);
    for (int t = 0; t < kChunk; t++) {
      const int lo = __builtin_amdgcn_readlane(__double2loint(G), t), hi = __builtin_amdgcn_readlane(__double2hiint(G), t);
      const float bt = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, beta), t));
      const float e = lane <= t ? expf((float)(__hiloint2double(hi, lo) - G)) : 0.0f;
      A[t * kChunk + lane] = lane < t ? bt * e * s_kk[t * kTri + lane] : 0.0f;
      rec[kRecP + t * kChunk + lane] = lane <= t ? e * s_qk[t * kTri + lane] : 0.0f;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float x[kChunk];
#pragma unroll
    for (int t = 0; t < kChunk; t++) {
      float acc[4] = {t == lane ? 1.0f : 0.0f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s4 = 0; s4 < t; s4 += 4) {
        const float4 r = *(const float4 *)(A + t * kChunk + s4);
        acc[0] = __builtin_fmaf(-r.x, x[s4], acc[0]);
        if (s4 + 1 < t) acc[1] = __builtin_fmaf(-r.y, x[s4 + 1], acc[1]);
        if (s4 + 2 < t) acc[2] = __builtin_fmaf(-r.z, x[s4 + 2], acc[2]);
        if (s4 + 3 < t) acc[3] = __builtin_fmaf(-r.w, x[s4 + 3], acc[3]);
      }
      x[t] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
      rec[kRecInv + t * kChunk + lane] = x[t] * beta;
    }
    // the next head's A goes where this one's is read
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}
constexpr int kChunkLds = (2 * kChunk * kPitch + 2 * kChunk * kTri + 2 * kChunk) * 4;
static_assert(4 * kChunk * kChunk <= 2 * kChunk * kPitch, "A of four waves lies over the rows");

// ---------------------------------------------------------------------------
// prompts: the state's walk over the chunks
// ---------------------------------------------------------------------------
// One workgroup of 4 waves a (value head, 32 value columns, sequence), chunk after
// chunk.  The state slice lives in the accumulators of its update (32 key rows a
// wave) and, for the products with q and k, in LDS.
constexpr int kCol = kSlice + 4;  // pitch of [row][column] tiles
template <class T>
__global__ __launch_bounds__(256) void k_delta_scan(DeltaArgs g) {
  extern __shared__ __align__(16) float lds[];
  float *s_k = lds, *s_q = s_k + kChunk * kPitch, *s_s = s_q + kChunk * kPitch, *s_x = s_s + kKey * kCol,
        *s_d = s_x + kChunk * kCol;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n16 = lane & 15, kg = lane >> 4;
  const int nsl = g.dv / kSlice, h = blockIdx.x / nsl, col0 = (blockIdx.x % nsl) * kSlice, s = blockIdx.y;
  const int hk = h / (g.vh / g.kh);
  const int rows = g.start[s + 1] - g.start[s];
  const int c0 = g.chunk_first, c1 = min(c0 + g.chunks, (rows + kChunk - 1) / kChunk);
  if (c0 > 0 && c0 >= c1) return;  // an earlier pass ended this sequence
  const size_t at = ((size_t)g.slot[s] * g.vh + h) * g.dk * g.dv + col0;
  const float *from = c0 > 0 ? g.state_out : g.state;
  v4f S[2][2];
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int r = 32 * wave + 16 * i + 4 * kg + e;
        S[i][j][e] = r < g.dk ? from[at + (size_t)r * g.dv + 16 * j + n16] : 0.0f;
      }
  for (int c = c0; c < c1; c++) {
    const int t0 = g.start[s] + c * kChunk, n = min(kChunk, g.start[s + 1] - t0);
    const float *rec = g.rec + ((size_t)(g.chunk0[s] + c - c0) * g.vh + h) * kRec;
    stage_rows(s_k, (const T *)g.k + (size_t)t0 * g.k_stride + (size_t)hk * g.dk, g.k_stride, n, g.dk, nullptr);
    stage_rows(s_q, (const T *)g.q + (size_t)t0 * g.q_stride + (size_t)hk * g.dk, g.q_stride, n, g.dk, nullptr);
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) s_s[(32 * wave + 16 * i + 4 * kg + e) * kCol + 16 * j + n16] = S[i][j][e];
    __syncthreads();
    // rows 16 wave .. of k S0 and q S0
    v4f ks[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}}, o[2] = {ks[0], ks[0]};
    for (int i = 0; i < g.dk; i += 16) {
      const float4 kf = *(const float4 *)(s_k + (16 * wave + n16) * kPitch + i + 4 * kg);
      const float4 qf = *(const float4 *)(s_q + (16 * wave + n16) * kPitch + i + 4 * kg);
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const float sf = s_s[(i + 4 * kg + e) * kCol + 16 * j + n16];
          ks[j] = mfma_f32_16(((const float *)&kf)[e], sf, ks[j]);
          o[j] = mfma_f32_16(((const float *)&qf)[e], sf, o[j]);
        }
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int t = 16 * wave + 4 * kg + e;
      const float fx = rec[kRecX + t], fq = rec[kRecQ + t];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const float v = t < n ? (float)((const T *)g.v)[(size_t)(t0 + t) * g.v_stride + (size_t)h * g.dv + col0 + 16 * j + n16] : 0.0f;
        s_x[t * kCol + 16 * j + n16] = __builtin_fmaf(-fx, ks[j][e], v);
        o[j][e] *= fq;
      }
    }
    __syncthreads();
    // d = inverse x, lower triangular
    v4f d[2] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
    for (int i = 0; i <= wave; i++) {
      const float4 f = *(const float4 *)(rec + kRecInv + (16 * wave + n16) * kChunk + 16 * i + 4 * kg);
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          d[j] = mfma_f32_16(((const float *)&f)[e], s_x[(16 * i + 4 * kg + e) * kCol + 16 * j + n16], d[j]);
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
#pragma unroll
      for (int j = 0; j < 2; j++) s_d[(16 * wave + 4 * kg + e) * kCol + 16 * j + n16] = d[j][e];
    __syncthreads();
    for (int i = 0; i <= wave; i++) {
      const float4 f = *(const float4 *)(rec + kRecP + (16 * wave + n16) * kChunk + 16 * i + 4 * kg);
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int j = 0; j < 2; j++)
          o[j] = mfma_f32_16(((const float *)&f)[e], s_d[(16 * i + 4 * kg + e) * kCol + 16 * j + n16], o[j]);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int t = 16 * wave + 4 * kg + e;
      if (t < n)
#pragma unroll
        for (int j = 0; j < 2; j++) ((T *)g.out)[((size_t)(t0 + t) * g.vh + h) * g.dv + col0 + 16 * j + n16] = (T)o[j][e];
    }
    const float eg = rec[kRecEnd];
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
      for (int j = 0; j < 2; j++) S[i][j] *= eg;
    for (int i = 0; i < kChunk; i += 4) {
      const int t = i + kg;
      const float fr = rec[kRecR + t];
      float df[2];
#pragma unroll
      for (int j = 0; j < 2; j++) df[j] = fr * s_d[t * kCol + 16 * j + n16];
#pragma unroll
      for (int m = 0; m < 2; m++) {
        const float kf = s_k[t * kPitch + 32 * wave + 16 * m + n16];
#pragma unroll
        for (int j = 0; j < 2; j++) S[m][j] = mfma_f32_16(kf, df[j], S[m][j]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int r = 32 * wave + 16 * i + 4 * kg + e;
        if (r < g.dk) g.state_out[at + (size_t)r * g.dv + 16 * j + n16] = S[i][j][e];
      }
}
constexpr int kScanLds = (2 * kChunk * kPitch + kKey * kCol + 2 * kChunk * kCol) * 4;

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
  hipError_t e = hipFuncSetAttribute((const void *)k_delta_chunk<T>, hipFuncAttributeMaxDynamicSharedMemorySize, kChunkLds);
  if (e == hipSuccess) e = hipFuncSetAttribute((const void *)k_delta_scan<T>, hipFuncAttributeMaxDynamicSharedMemorySize, kScanLds);
  if (e != hipSuccess) return fail_hip(name, e);
  if (chunks) k_delta_chunk<T><<<dim3(chunks, g.kh), 256, kChunkLds, st>>>(g);
  k_delta_scan<T><<<dim3(g.vh * (g.dv / kSlice), g.seqs), 256, kScanLds, st>>>(g);
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
    if (start[s + 1] < start[s]) return fail_arg("%s: sequence %d has rows %d..%d", name, s, start[s], start[s + 1]);
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
  // records of a pass: 512 MiB, a chunk of every sequence at least
  const size_t chunk_bytes = (size_t)g.vh * kRec * sizeof(float);
  for (int s0 = 0; s0 < sequences; s0 += kSeqs) {
    const int n = sequences - s0 < kSeqs ? sequences - s0 : kSeqs;
    long long per = (long long)((512u << 20) / chunk_bytes) / n;
    if (per < 1) per = 1;
    int longest = 0;
    for (int s = 0; s < n; s++) {
      const int c = (int)(((long long)start[s0 + s + 1] - start[s0 + s] + kChunk - 1) / kChunk);
      if (c > longest) longest = c;
    }
    g.chunks = per < longest ? (int)per : longest;
    memcpy(g.start, start + s0, (n + 1) * sizeof(int));
    memcpy(g.slot, slot + s0, n * sizeof(int));
    g.seqs = n;
    for (g.chunk_first = 0; g.chunk_first == 0 || g.chunk_first < longest; g.chunk_first += g.chunks) {
      for (int s = 0; s < n; s++) {
        int c = (int)(((long long)g.start[s + 1] - g.start[s] + kChunk - 1) / kChunk) - g.chunk_first;
        if (c > g.chunks) c = g.chunks;
        g.chunk0[s + 1] = g.chunk0[s] + (c > 0 ? c : 0);
      }
      const int chunks = g.chunk0[n];
      if (ensure_scratch(ctx, kScrDelta, (size_t)(chunks ? chunks : 1) * chunk_bytes, name)) return -1;
      g.rec = (float *)ctx->scratch[kScrDelta];
      const int rc = d->type == COLI_TYPE_F32   ? launch_delta<float>(name, g, chunks, ctx->stream)
                     : d->type == COLI_TYPE_F16 ? launch_delta<_Float16>(name, g, chunks, ctx->stream)
                                                : launch_delta<__bf16>(name, g, chunks, ctx->stream);
      if (rc) return -1;
      if (longest == 0) break;
    }
  }
  return launch_status(name);
}
