// The paged key-value cache: appending keys and values with the position
// rotation applied on the way (coli_cuda_paged_append), attention of single new
// tokens (coli_cuda_paged_decode) and of packed prompts (coli_cuda_paged_prompt).
//
// Attention, both forms: o = sum_j p_j v_j / sum_j p_j, p_j = 2^(s_j - m) over the
// visible positions j, s_j = scale log2(e) q . k_j, with the running maximum m, the
// sum and o held in fp32 and rescaled when m grows, so the cache is read once.
// p is rounded to the cache's 16-bit type for the second product (bf16 2^-8, fp16
// 2^-11 relative a term, what the values themselves carry, as far as below() holds it
// among fp16's normal numbers); an fp32 cache keeps fp32 products throughout.
#include <hip/hip_runtime.h>
#include <limits.h>
#include <math.h>
#include <string.h>

#include "sw_lds_dma.h"
#include "sw_serve.h"

namespace sw {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// The m of a row's p_j = 2^(s_j - m), from the largest score.  Any m serves, since
// numerator and sum share it.  fp16 takes it `lift` below that score: its probabilities
// then reach 2^lift and are normal numbers down to 2^(-14 - lift) of the largest, where
// many small ones may be all of the output; below 2^-25, as it were with m the largest
// score, 100,000 of them behind a position whose values are zero came out as nothing.
// From 2^20 on, where m itself would be rounded by as much, it is the largest score.
template <class T>
__device__ __forceinline__ float below(float most, float lift) {
  if constexpr (__is_same(T, _Float16))
    return fabsf(most) < 1048576.0f ? most - lift : most;
  else
    return most;
}

// Where a sequence's positions lie.  Offsets are 64-bit: a pool may hold more
// than 2^31 elements.
struct PageMap {
  const int *table;  // [sequence][table_pages]
  int pages, table_pages, page_size;
  FastDiv div;  // by page_size
  long long stride;
  int row;  // elements of one position: kv_heads * head_dim
};
// A wave's page id by a scalar load (the table does not change during a kernel): a
// vector load would be waited for at once, to make its value scalar.
__device__ __forceinline__ int scalar_id(const int *tab, int pg) {
  return ((const __attribute__((address_space(4))) int *)tab)[pg];
}
// Element offset of position p of the sequence whose table row is `tab`; -1 where
// the table names no page.
__device__ __forceinline__ long long cell(const PageMap &m, const int *tab, int p) {
  const int pg = div_by(m.div, p);
  const int id = tab[pg];
  return (unsigned)id < (unsigned)m.pages ? (long long)id * m.stride + (long long)(p - pg * m.page_size) * m.row : -1;
}

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------
struct AppendArgs {
  const void *q, *k, *v;
  void *q_out, *k_pool, *v_pool;
  long long q_stride, k_stride, v_stride;
  const float *q_norm, *k_norm;
  int q_head, nh, nkv, rd, heads_per_block, seqs, first_seq;
  float eps;
  PageMap map;
  double freq[128];  // turns a position
  int start[kSeqs + 1], len[kSeqs];
};

template <class T, int E>
struct alignas(sizeof(T) * E) Pack {
  T v[E];
};

// Stores of 16 bytes a lane past the caches (6,379 fp32 tokens 64 -> 51 us, and what
// reads them next is faster too: 3,000 tokens with their prompt attention 135 -> 130, with
// a decode 43 -> 35); smaller ones gain nothing (bf16 heads of 256 24.3 and 23.8).
template <class P>
__device__ __forceinline__ void store_once(P *to, const P &x) {
  if constexpr (sizeof(P) == 16)
    __builtin_nontemporal_store(__builtin_bit_cast(v4u, x), (v4u *)to);
  else
    *to = x;
}

// One workgroup a (token, run of heads), one wave a head: E = HD / 64 elements a
// lane.  HBM-bound (each value read and written once): 6,379 fp32 tokens of 16 + 2
// heads of 256 (261 MB) 51 us, 5.1 TB/s, a large copy's rate (41 in calls on the same
// tokens, which the memory-side cache then holds); one bf16
// token 4.2 us, the launch and its chain of loads.  The angle is formed once a
// workgroup: turns = position * freq in 64 bits, the whole turns dropped, the rest
// to fp32 (2^-25 turns), so far positions keep theirs.  The rotation's partners meet
// in LDS, where any even rotary_dim finds them.  The result is rounded to the cache's
// type once; sums of squares are fp32.
template <class T, int HD>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
  constexpr int E = HD / 64;
  typedef Pack<T, E> P;
  __shared__ float s_co[128], s_si[128], s_row[4][HD];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int t = a.start[0] + blockIdx.x;
  const int s = find_span(a.start, a.seqs, t);
  const int pos = a.len[s] - a.start[s + 1] + t;
  const int half = a.rd >> 1, nq = a.q ? a.nh : 0;
  for (int i = threadIdx.x; i < half; i += 256) {
    double turns = (double)pos * a.freq[i];
    turns -= __builtin_rint(turns);
    float si, co;
    sincospif(2.0f * (float)turns, &si, &co);
    s_co[i] = co;
    s_si[i] = si;
  }
  __syncthreads();
  const long long at = cell(a.map, a.map.table + (size_t)(a.first_seq + s) * a.map.table_pages, pos);
  const int h1 = min(nq + a.nkv, (int)(blockIdx.y + 1) * a.heads_per_block);
  for (int h = blockIdx.y * a.heads_per_block + wave; h < h1; h += 4) {
    const bool isq = h < nq;
    const int kvh = h - nq;
    const T *src = isq ? (const T *)a.q + (size_t)t * a.q_stride + (size_t)h * a.q_head
                       : (const T *)a.k + (size_t)t * a.k_stride + (size_t)kvh * HD;
    if (!isq && at < 0) continue;
    const P in = *(const P *)(src + E * lane);
    P vin;
    if (!isq) vin = *(const P *)((const T *)a.v + (size_t)t * a.v_stride + (size_t)kvh * HD + E * lane);
    float x[E];
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = (float)in.v[e];
    const float *norm = isq ? a.q_norm : a.k_norm;
    if (norm) {
      float s2 = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e++) s2 = __builtin_fmaf(x[e], x[e], s2);
      const float r = 1.0f / sqrtf(wave_sum_dpp(s2) / (float)HD + a.eps);
#pragma unroll
      for (int e = 0; e < E; e++) x[e] = x[e] * r * (1.0f + norm[E * lane + e]);
    }
    float *row = s_row[wave];
#pragma unroll
    for (int e = 0; e < E; e++) row[E * lane + e] = x[e];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int e = 0; e < E; e++) {
      const int j = E * lane + e;
      if (j < a.rd) {
        const int i = j < half ? j : j - half;
        const float lo = row[i], hi = row[i + half], co = s_co[i], si = s_si[i];
        x[e] = j < half ? __builtin_fmaf(lo, co, -(hi * si)) : __builtin_fmaf(hi, co, lo * si);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    P out;
#pragma unroll
    for (int e = 0; e < E; e++) out.v[e] = (T)x[e];
    if (isq) {
      store_once((P *)((T *)a.q_out + ((size_t)t * a.nh + h) * HD + E * lane), out);
    } else {
      store_once((P *)((T *)a.k_pool + at + (size_t)kvh * HD + E * lane), out);
      store_once((P *)((T *)a.v_pool + at + (size_t)kvh * HD + E * lane), vin);
    }
  }
}

// ---------------------------------------------------------------------------
// attention of one new token a sequence
// ---------------------------------------------------------------------------
struct DecodeArgs {
  const void *q, *gate, *k, *v;
  void *out;
  float *po, *pm, *pl;  // partial records (null: every row has one split)
  long long gate_stride;
  int gate_head, nh, nkv, G, hgroups, rows, first_seq, per;
  float scale;  // scale * log2(e)
  PageMap map;
  int first[kSeqs + 1], len[kSeqs];  // row r's splits are first[r] .. first[r + 1] - 1
};

__device__ __forceinline__ v4f mfma_f32_16(float a, float b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// One workgroup of 4 waves a (sequence, split of its positions, kv head, group of
// 16 query heads); a wave takes every fourth block of KB positions.  The scores
// come transposed, S^T (positions x heads) = K Q^T, so that a lane holds one head's
// probabilities of the positions 4 kg + j whose values it also loads: the second
// product O^T (dims x heads) += V^T P^T takes them as they are.  Its A operand wants
// consecutive positions of one dim where memory has consecutive dims of one
// position: in 16 bits a lane loads 8 dims of 8 positions and regroups them by byte
// permutes (16 to 16 loaded registers), an fp32 lane's value is the operand itself;
// row n of dim tile d stands for dim W n + d (tiles of one load).
// Nothing goes through LDS until the waves' merge.  HBM-bound: a block's keys are
// loaded as soon as the last ones' registers are free, its values likewise, so that a
// wave always has one of them in flight.  Every key and value is fetched once (471 MB
// counted for 466 MB) by each group of 16 query heads of its kv head.  Kernel times:
// 227,641 bf16 positions of 2 kv heads x 256 79 us, 5.9 TB/s; 48
// fp16 sequences up to 9,001 at 8 x 128 137 us, 5.3 TB/s; 13 fp32 ones up to 6,000 31
// us, 4.5 TB/s; one of 4,097 positions 10 us, of which 1.6 would be the bytes' own.
// The loads leave nothing in the caches: 147 -> 141 and 87 -> 84 us with the join for the
// first two, 12.0 -> 12.4 for the last, whose keys a repeated call finds there.
// A probability is rounded to the cache's 16 bits for the second product, half a step
// of what the values themselves are rounded to; fp16's reach 2^15 and are normal numbers
// down to 2^-29 of the largest; fp32 caches take fp32 products.
// RUN16: pages hold whole runs of 16 positions, whose page the wave then looks up
// once, by a scalar load, a block ahead; otherwise every lane looks up its own.
template <class T, int HD, bool RUN16>
struct DecodeShape {
  static constexpr bool B16 = sizeof(T) == 2;
  // workgroups of a compute unit, by their registers (one lane's own look-ups take more)
  static constexpr int kPerCu = HD == 64 ? (RUN16 ? 4 : 3) : HD == 128 ? (RUN16 ? 3 : 2) : 1;
  static constexpr int kLeast = 4 * (B16 ? 32 : 16);               // positions of a split: one block a wave
};
template <class T, int HD, bool RUN16>
__global__ __launch_bounds__(256, (DecodeShape<T, HD, RUN16>::kPerCu)) void k_paged_decode(DecodeArgs a) {
  constexpr bool B16 = sizeof(T) == 2;
  constexpr int NB = B16 ? 2 : 1, KB = 16 * NB;            // runs and positions of a block
  constexpr int NT = HD / 16;                              // dim tiles
  constexpr int KR = HD * (int)sizeof(T) / 64;             // registers x 4 of a run's keys
  constexpr int W = B16 ? (HD >= 128 ? 8 : 4) : 4;         // values of one load
  constexpr int NW = NT / W;                               // loads of one position
  constexpr int LV = W * (int)sizeof(T) / 4;               // registers of one load
  typedef unsigned VL __attribute__((ext_vector_type(LV)));
  constexpr int OP = HD + 4;                               // pitch of a head's outputs in LDS
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __align__(16) float s_o[4][16 * OP];          // fp32: the queries first, [chunk][lane] x 16 bytes
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4;
  const int per_split = a.nkv * a.hgroups;
  const int slot = blockIdx.x / per_split, sub = blockIdx.x % per_split;
  const int kvh = sub / a.hgroups, hg = sub % a.hgroups;
  const int r = a.rows == 1 ? 0 : find_span(a.first, a.rows, slot);
  const int len = a.len[r];
  const int heads = min(16, a.G - 16 * hg), h0 = kvh * a.G + 16 * hg;
  const int key_first = (slot - a.first[r]) * a.per, key_end = min(len, key_first + a.per);
  const int *tab = a.map.table + (size_t)(a.first_seq + r) * a.map.table_pages;
  const T *kc = (const T *)a.k + (size_t)kvh * HD, *vc = (const T *)a.v + (size_t)kvh * HD;

  // where the positions of a block lie: a run's first cell, or this lane's cells (of
  // key n, of the values 4 kg + j); -1 where there is none
  struct Loc {
    int id[NB];                        // RUN16: the runs' page ids
    long long k[NB], v[NB][RUN16 ? 1 : 4];
  };
  auto look_up = [&](Loc &l, int key0) {
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const int p0 = key0 + 16 * b;
      if constexpr (RUN16) {
        l.id[b] = p0 < key_end ? scalar_id(tab, div_by(a.map.div, p0)) : -1;
      } else {
        l.k[b] = p0 + n < key_end ? cell(a.map, tab, p0 + n) : -1;
#pragma unroll
        for (int j = 0; j < 4; j++) l.v[b][j] = p0 + 4 * kg + j < key_end ? cell(a.map, tab, p0 + 4 * kg + j) : -1;
      }
    }
  };
  auto find_runs = [&](Loc &l, int key0) {  // RUN16: the ids have come
    if constexpr (RUN16)
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const int p0 = key0 + 16 * b, pg = div_by(a.map.div, p0);
        l.k[b] = (unsigned)l.id[b] < (unsigned)a.map.pages
                     ? (long long)l.id[b] * a.map.stride + (long long)(p0 - pg * a.map.page_size) * a.map.row
                     : -1;
      }
  };
  // a position that is not there reads another cell of the pool and is masked below
  v4u kr[NB][KR];
  VL vr[NB][4][NW];
  auto load_keys = [&](const Loc &l, int key0) {
#pragma unroll
    for (int b = 0; b < NB; b++) {
      const T *kp;
      if constexpr (RUN16)
        kp = kc + (l.k[b] >= 0 ? l.k[b] : 0) + (unsigned)max(0, min(n, key_end - 1 - key0 - 16 * b)) * (unsigned)a.map.row;
      else
        kp = kc + (l.k[b] >= 0 ? l.k[b] : 0);
#pragma unroll
      for (int i = 0; i < KR; i++) kr[b][i] = __builtin_nontemporal_load((const v4u *)(kp + (64 / sizeof(T)) * i + (16 / sizeof(T)) * kg));
    }
  };
  auto load_values = [&](const Loc &l, int key0) {
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const T *vp;
        if constexpr (RUN16)
          vp = vc + (l.k[b] >= 0 ? l.k[b] : 0) +
               (unsigned)max(0, min(4 * kg + j, key_end - 1 - key0 - 16 * b)) * (unsigned)a.map.row;
        else
          vp = vc + (l.v[b][j] >= 0 ? l.v[b][j] : 0);
        vp += W * n;
#pragma unroll
        for (int w = 0; w < NW; w++) vr[b][j][w] = __builtin_nontemporal_load((const VL *)(vp + 16 * W * w));
      }
  };

  // the queries, B operand of the first product (fp32 ones by way of LDS; heads beyond
  // the group are zero), go out before the first block: loads come back in order
  constexpr int QR = B16 ? KR : KR / 4;
  v4u qv[QR];
  {
    const T *qrow = (const T *)a.q + ((size_t)r * a.nh + h0 + n) * HD;
#pragma unroll
    for (int i = 0; i < QR; i++)
      qv[i] = n < heads ? *(const v4u *)(qrow + (64 / sizeof(T)) * (B16 ? i : 4 * i + wave) + (16 / sizeof(T)) * kg) : v4u{0, 0, 0, 0};
  }
  int key0 = key_first + wave * KB;
  Loc cur, nxt;
  if (key0 < key_end) {
    look_up(cur, key0);
    find_runs(cur, key0);
    load_keys(cur, key0);
    load_values(cur, key0);
  }
  if constexpr (!B16) {
#pragma unroll
    for (int i = 0; i < QR; i++) ((v4u *)s_o)[(4 * i + wave) * 64 + lane] = qv[i];
    lds_barrier();
  }
  v4f o[NT];
#pragma unroll
  for (int d = 0; d < NT; d++) o[d] = v4f{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.0f;

  if (key0 < key_end) for (;;) {
    const int next0 = key0 + 4 * KB;
    const bool more = next0 < key_end;
    if (more) look_up(nxt, next0);
    float sv[NB][4];
#pragma unroll
    for (int b = 0; b < NB; b++) {
      v4f sc;
      if constexpr (B16) {
        v4f c0 = v4f{0.f, 0.f, 0.f, 0.f}, c1 = c0;
#pragma unroll
        for (int i = 0; i < KR; i += 2) {
          c0 = Mat16<T>::mul16(kr[b][i], qv[i], c0);
          c1 = Mat16<T>::mul16(kr[b][i + 1], qv[i + 1], c1);
        }
        sc = c0 + c1;
      } else {
        v4f c[4] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < KR; i++) {
          const v4u qq = ((const v4u *)s_o)[i * 64 + lane];
#pragma unroll
          for (int e = 0; e < 4; e++) c[e] = mfma_f32_16(__uint_as_float(kr[b][i][e]), __uint_as_float(qq[e]), c[e]);
        }
        sc = (c[0] + c[1]) + (c[2] + c[3]);
      }
#pragma unroll
      for (int j = 0; j < 4; j++) sv[b][j] = sc[j] * a.scale;
    }
    if (more) {
      find_runs(nxt, next0);
      load_keys(nxt, next0);
    }
    // positions behind the end or without a page: no score, and a zero value (what lies
    // there may be anything, and 0 * NaN is NaN)
    bool there[NB][4], whole = true;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        there[b][j] = RUN16 ? cur.k[b] >= 0 && key0 + 16 * b + 4 * kg + j < key_end : cur.v[b][RUN16 ? 0 : j] >= 0;
        whole &= there[b][j];
      }
    if (!__all(whole)) {
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          sv[b][j] = there[b][j] ? sv[b][j] : -INFINITY;
#pragma unroll
          for (int w = 0; w < NW; w++) vr[b][j][w] = there[b][j] ? vr[b][j][w] : VL(0u);
        }
    }
    float bm = -INFINITY;
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int j = 0; j < 4; j++) bm = fmaxf(bm, sv[b][j]);
    bm = fmaxf(bm, __shfl_xor(bm, 16));
    bm = fmaxf(bm, __shfl_xor(bm, 32));
    const float m_new = fmaxf(m_run, below<T>(bm, 15.0f)), m_use = m_new == -INFINITY ? 0.0f : m_new;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    float ps = 0.0f;  // this lane's positions; the lanes of a head meet at the end
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        sv[b][j] = __builtin_amdgcn_exp2f(sv[b][j] - m_use);
        ps += sv[b][j];
      }
    l_run = __builtin_fmaf(l_run, alpha, ps);
    m_run = m_new;
#pragma unroll
    for (int d = 0; d < NT; d++) o[d] *= alpha;
    if constexpr (B16) {
      const v4u pf = v4u{pack2<T>(sv[0][0], sv[0][1]), pack2<T>(sv[0][2], sv[0][3]), pack2<T>(sv[1][0], sv[1][1]),
                         pack2<T>(sv[1][2], sv[1][3])};
#pragma unroll
      for (int d = 0; d < NT; d++) {
        const int w = d / W, e = (d % W) / 2;
        const unsigned sel = d % 2 ? 0x07060302u : 0x05040100u;
        v4u vf;
#pragma unroll
        for (int b = 0; b < 2; b++) {
          vf[2 * b] = __builtin_amdgcn_perm(vr[b][1][w][e], vr[b][0][w][e], sel);
          vf[2 * b + 1] = __builtin_amdgcn_perm(vr[b][3][w][e], vr[b][2][w][e], sel);
        }
        o[d] = Mat16<T>::mul16(vf, pf, o[d]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int d = 0; d < NT; d++) o[d] = mfma_f32_16(__uint_as_float(vr[0][j][d / W][d % W]), sv[0][j], o[d]);
    }
    if (!more) break;
    load_values(nxt, next0);
    cur = nxt;
    key0 = next0;
  }

  // the waves meet in LDS, summed in wave order
  l_run += __shfl_xor(l_run, 16);
  l_run += __shfl_xor(l_run, 32);
  if (kg == 0) {
    s_m[wave][n] = m_run;
    s_l[wave][n] = l_run;
  }
  if (!B16) __syncthreads();  // the queries have been read
#pragma unroll
  for (int d = 0; d < NT; d += 4)
#pragma unroll
    for (int i = 0; i < 4; i++)
      *(v4f *)(s_o[wave] + n * OP + 16 * W * (d / W) + W * (4 * kg + i) + d % W) = v4f{o[d][i], o[d + 1][i], o[d + 2][i], o[d + 3][i]};
  __syncthreads();
  auto total = [&](int h, float &M, float (&f)[4]) {  // largest score, sum, and the waves' weights
    M = fmaxf(fmaxf(s_m[0][h], s_m[1][h]), fmaxf(s_m[2][h], s_m[3][h]));
    float L = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      f[w] = s_m[w][h] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[w][h] - M);
      // a wave without a visible position has sums of zero; a NaN sum is kept
      L = __builtin_fmaf(s_l[w][h], s_m[w][h] == -INFINITY ? 1.0f : f[w], L);
    }
    return L;
  };
  if (a.po && threadIdx.x < heads) {
    float M, f[4];
    const float L = total(threadIdx.x, M, f);
    a.pm[(size_t)slot * a.nh + h0 + threadIdx.x] = L == 0.0f ? -INFINITY : M == -INFINITY ? 0.0f : M;
    a.pl[(size_t)slot * a.nh + h0 + threadIdx.x] = L;
  }
  for (int u = threadIdx.x; u < heads * HD / 4; u += 256) {
    const int h = u / (HD / 4), d = u % (HD / 4) * 4;
    float M, f[4];
    const float L = total(h, M, f);
    v4f x = *(const v4f *)(s_o[0] + h * OP + d) * f[0];
#pragma unroll
    for (int w = 1; w < 4; w++) x += *(const v4f *)(s_o[w] + h * OP + d) * f[w];
    if (a.po) {
      *(v4f *)(a.po + ((size_t)slot * a.nh + h0 + h) * HD + d) = x;
      continue;
    }
    const float inv = L > 0.0f ? 1.0f / L : L;  // 0 stays, and a NaN
    Pack<T, 4> y, g;
    if (a.gate) g = *(const Pack<T, 4> *)((const T *)a.gate + (size_t)r * a.gate_stride + (size_t)(h0 + h) * a.gate_head + d);
#pragma unroll
    for (int e = 0; e < 4; e++) y.v[e] = (T)(x[e] * inv * (a.gate ? gate_sigmoid((float)g.v[e]) : 1.0f));
    *(Pack<T, 4> *)((T *)a.out + ((size_t)r * a.nh + h0 + h) * HD + d) = y;
  }
}

// Joins the splits of one (row, query head): the weights 2^(m - M) in LDS, while the
// first outputs are on their way; a thread has four dims of every NG-th split, eight
// loads in flight, and the groups meet in LDS in their order.
// grid (query heads, rows); THREADS 512, or 128 where two rounds of theirs take all
// splits and there are many (1,536 (row, head) pairs of 50 splits and less 11.2 -> 5.2
// us); S <= kMaxSplits.  Latency-bound: 4.1 us at 66 splits of 32 heads, 5.4 at 121.
constexpr int kMaxSplits = 256;
struct JoinArgs {
  const float *po, *pm, *pl;
  const void *gate;
  void *out;
  long long gate_stride;
  int gate_head, nh, flat;
  int S, step;       // not flat: record of split s of row t is s * step + t
  long long row0;    // first row of out and gate
  int first[kSeqs + 1];  // flat: row r's records
};
constexpr int kJoinLoads = 8;  // of a thread in flight
template <class T, int HD, int THREADS>
__global__ __launch_bounds__(THREADS) void k_paged_join(JoinArgs a) {
  constexpr int TH = HD / 4, NG = THREADS / TH, B = kJoinLoads, NW = THREADS / 64;
  __shared__ float s_w[THREADS < kMaxSplits ? THREADS : kMaxSplits], s_red[2 * NW];
  __shared__ v4f s_o[NG][TH];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, h = blockIdx.x, t = blockIdx.y;
  const int S = a.flat ? a.first[t + 1] - a.first[t] : a.S;
  const size_t base = a.flat ? (size_t)a.first[t] : (size_t)t, step = a.flat ? 1 : (size_t)a.step;
  const int d = tid % TH, g = tid / TH;
  const float *po = a.po + (base * a.nh + h) * HD + 4 * d;
  const size_t pitch = step * a.nh * HD;
  v4f x[B];
  auto load = [&](int s0) {
#pragma unroll
    for (int k = 0; k < B; k++) {
      const int s = s0 + k * NG;
      x[k] = *(const v4f *)(po + (s < S ? s : 0) * pitch);
    }
  };
  load(g);
  const size_t row = (size_t)a.row0 + t;
  Pack<T, 4> y, gt;
  if (a.gate && g == 0) gt = *(const Pack<T, 4> *)((const T *)a.gate + row * a.gate_stride + (size_t)h * a.gate_head + 4 * d);
  const size_t rec = ((base + (size_t)(tid < S ? tid : 0) * step) * a.nh) + h;
  const float m = tid < S ? a.pm[rec] : -INFINITY, lv = tid < S ? a.pl[rec] : 0.0f;
  const float wm = wave_max_dpp(m);
  if (lane == 0) s_red[wave] = wm;
  __syncthreads();
  float M = s_red[0];
#pragma unroll
  for (int w = 1; w < NW; w++) M = fmaxf(M, s_red[w]);
  // a record without a visible position holds nothing and gets the weight -1: one of
  // weight zero counts, for zero times a NaN is a NaN
  const float w = m == -INFINITY ? -1.0f : __builtin_amdgcn_exp2f(m - M);
  if (tid < S) s_w[tid] = w;
  const float ls = wave_sum_dpp(w < 0.0f ? 0.0f : lv * w);
  if (lane == 0) s_red[NW + wave] = ls;
  __syncthreads();
  float L = s_red[NW];
#pragma unroll
  for (int k = 1; k < NW; k++) L += s_red[NW + k];
  v4f o = v4f{0.f, 0.f, 0.f, 0.f};
  for (int s0 = g; s0 < S; s0 += B * NG) {
    if (s0 != g) load(s0);
#pragma unroll
    for (int k = 0; k < B; k++) {
      const int s = s0 + k * NG;
      if (s < S && !(s_w[s] < 0.0f)) o += x[k] * s_w[s];
    }
  }
  s_o[g][d] = o;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int k = 1; k < NG; k++) o += s_o[k][d];
  const float inv = L > 0.0f ? 1.0f / L : L;  // 0 stays, and a NaN
#pragma unroll
  for (int e = 0; e < 4; e++) y.v[e] = (T)(o[e] * inv * (a.gate ? gate_sigmoid((float)gt.v[e]) : 1.0f));
  *(Pack<T, 4> *)((T *)a.out + (row * a.nh + h) * HD + 4 * d) = y;
}

// ---------------------------------------------------------------------------
// attention of packed prompts
// ---------------------------------------------------------------------------
struct PromptArgs {
  const void *q, *gate, *k, *v;
  void *out;
  float *po, *pm, *pl;  // partial records [split][row - row0][head] (null: one split)
  long long gate_stride;
  int gate_head, nh, nkv, G, seqs, first_seq, splits, rows;
  float scale;      // |scale| * log2(e)
  unsigned q_sign;  // sign bits of a register of queries where scale is negative
  FastDiv by_group, by_heads;  // by G, by nkv
  PageMap map;
  int start[kSeqs + 1], len[kSeqs], tile0[kSeqs + 1];  // sequence s's tiles are tile0[s] .. tile0[s + 1] - 1
};

__device__ float g_zero_row[256];  // never written: what copies of absent positions read (a row of 1 KB at most)

__device__ __forceinline__ v16f mfma_f32_32(float a, float b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// LDS by its 32-bit address
typedef short v4s __attribute__((ext_vector_type(4)));
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Wint-to-pointer-cast"
__device__ __forceinline__ v4u lds_v4u(unsigned at) { return *(__attribute__((address_space(3))) const v4u *)at; }
__device__ __forceinline__ float lds_f32(unsigned at) { return *(__attribute__((address_space(3))) const float *)at; }
// 16 lanes read four rows x 16 columns, four 16-bit values a lane, and get the four
// rows of one column each
__device__ __forceinline__ v2u lds_transposed(unsigned at) {
  return __builtin_bit_cast(v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s *)at));
}
#pragma clang diagnostic pop

template <class T, int HD, int C>
struct PromptShape {
  static constexpr bool B16 = sizeof(T) == 2;
  // rows of a wave, the columns of its matrix instructions: 32 (32x32x16), or 16
  // (16x16x32, 16-bit types), which two waves a SIMD share: where the outputs of 32
  // would leave it one (head dim 256), and where there are no more workgroups than
  // compute units, which would leave it one too, with twice the softmax a tile.  bf16
  // prompts of one length, 32 against 16 rows, us a call: head dim 64, 120 workgroups 12.5
  // and 10.6, 240 17.0 and 15.4, then 336 17.8 and 20.4, 432 18.9 and 22.3, 720 44.5 and
  // 58.1; head dim 128, 192 18.3 and 15.1, then 320 20.9 and 22.6, 640 43.7 and 42.3, 896
  // 49.2 and 56.4, 1,880 150 and 189; fp16 the same within 2 us
  static_assert(C == 32 || (C == 16 && B16), "shapes of the matrix instructions");
  static constexpr int kWaves = 128 / C;
  static constexpr int kKeys = B16 ? 64 : 32;               // positions of a tile
  static constexpr int kRowBytes = HD * (int)sizeof(T);
  static constexpr int kTileBytes = kKeys * kRowBytes;      // of one matrix
  static constexpr int kLds = 4 * kTileBytes + 16;          // K and V, two buffers, flags
  static constexpr int kRows = 128;                         // (token, head) rows of a workgroup
  static constexpr int kPerSimd = B16 || HD < 256 ? 2 : 1;  // waves of a SIMD
  // how far the maximum may outgrow the softmax's reference, in powers of two
  static constexpr float kLag = __is_same(T, _Float16) ? 2.0f : 8.0f;
};

// Tile x of a launch, heavy ones first: tiles by their number within their sequence
// (later ones see more), the sequences' last ones first.  Tile number l is preceded by
// count(l + 1) tiles, count(l) = sum over sequences of max(0, tiles - l).
__device__ __forceinline__ void pick_tile(const int *tile0, int seqs, int x, int &seq, int &tile) {
  if (seqs == 1) {
    seq = 0;
    tile = tile0[1] - 1 - x;
    return;
  }
  static_assert(kSeqs == 128, "two sequences a lane");
  const int lane = threadIdx.x & 63;
  const int n0 = lane < seqs ? tile0[lane + 1] - tile0[lane] : 0;
  const int n1 = lane + 64 < seqs ? tile0[lane + 65] - tile0[lane + 64] : 0;
  auto count = [&](int l) { return wave_sum_dpp(max(0, n0 - l) + max(0, n1 - l)); };
  int lo = 0, hi = (int)wave_max_u32((unsigned)max(n0, n1));  // count(lo) > x >= count(hi)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (count(mid) <= x)
      hi = mid;
    else
      lo = mid;
  }
  tile = hi - 1;
  int rank = x - count(hi);
  unsigned long long have = __ballot(n0 >= hi);
  seq = 0;
  if (rank >= __builtin_popcountll(have)) {
    rank -= __builtin_popcountll(have);
    have = __ballot(n1 >= hi);
    seq = 64;
  }
  const unsigned long long below = have & ((1ull << lane) - 1);
  seq += __builtin_ctzll(__ballot((have >> lane & 1) && __builtin_popcountll(below) == rank));
}

// One workgroup a (tile of rows, kv head, split of the tile's positions).  A row is
// one (token, query head of the kv head's group), tokens in order, so that a tile's
// heads share every key and value it reads; a wave has C of them, the columns of its
// C x C matrix instructions, C = 32 or 16 (PromptShape; at head dim 256 8,682 tokens
// took 950 us at 32 rows and one wave a SIMD, 841 at 16 and two).  Tiles
// of kKeys positions go through two LDS buffers, copied straight from the pages (16
// bytes a lane from any address), the next tile while one is multiplied: one barrier a
// tile.  S^T = K Q^T leaves a lane 1 / NG of the tile's scores of one row, so the
// row's maximum and sum take one exchange between the NG = 64 / C lanes of a column,
// and the probabilities are the second product's B operand as they stand (positions in
// the order that the first product left them).  Its A operand, V^T, comes from the
// untransposed tile by the transposing LDS load (16 bits) or as single values (fp32).
// LDS rows are stored with their 16-byte chunks exchanged by an XOR with the row
// number, which spreads every access over all banks (no conflicts counted; 841 -> 772
// us with the order of tiles).
// 8,682 bf16 tokens of 32 query heads on 2 kv heads x 256 in three prompts (546 GFLOP)
// 690 us a call, 790 TFLOP/s (755 under the profiler), where the library's 8192^3 bf16
// product reaches 1,186.  No unit is full: counted, the matrix units are busy for 35% of
// the cycles and LDS for as many, since with 16 rows a matrix instruction of 16 cycles
// takes a fragment of 1 KB of its own; two waves a SIMD do not overlap the rest, a tile's
// products, softmax and barrier in turn.  32 rows at head dim 128 (43% and 22%) 376 us
// for two prompts of 6,000 and 2,121, 880 TFLOP/s.  9 short prompts 12.6 us: the longest
// one's chain of tiles.  14 drafted tokens behind 20,000 positions, split 32 ways, 36 to
// 41 us, 4 TB/s: ten tiles a workgroup in turn, in which 18 of 32 waves multiply rows
// that do not exist; 5.8 of join.  fp32, two prompts of 1,999 and 706 tokens, 16 heads of
// 256: 59 of the 154 TFLOP/s the fp32 library product reaches; matrix units busy for 69%
// of the cycles of a busy compute unit, which holds one wave a SIMD and one of 340
// workgroups of unequal length.
// Registers: the 32-row 16-bit kernels at head dim 128 spill 2 or 3 of theirs; of the
// fp32 ones, head dim 256 spills 4 (34 where pages do not hold whole runs), head dim 128
// 189 on such pages.
// Probabilities are rounded to 16 bits for the second product as in the decode kernel;
// fp16's reach 2^13 where the reference is new, 2^15 at most, and are normal numbers down
// to 2^-27 of the largest.
// RUN: pages hold whole runs of the WR positions that a wave copies, whose page is
// then looked up once, by a scalar load.
template <class T, int HD, bool RUN, int C>
__global__ __launch_bounds__((64 * PromptShape<T, HD, C>::kWaves), (PromptShape<T, HD, C>::kPerSimd)) void k_paged_prompt(PromptArgs a) {
  typedef PromptShape<T, HD, C> Sh;
  constexpr bool B16 = Sh::B16;
  constexpr int KT = Sh::kKeys, RB = Sh::kRowBytes, CPR = RB / 16, NI = Sh::kTileBytes / 1024 / Sh::kWaves;
  constexpr int NG = 64 / C, NA = C * C / 64;  // lane groups, registers of a C x C result
  constexpr int NS = KT / C, ND = HD / C;                     // tiles of positions, of dims
  constexpr int KC = CPR / NG;                                // 16-byte chunks of a lane's part of a row
  typedef float Acc __attribute__((ext_vector_type(NA)));     // register i: row 4 NG (i / 4) + 4 g + i % 4
  extern __shared__ __align__(1024) unsigned char smem[];
  // tag of the latest tile of its residue with an absent page: written a tile ahead,
  // while others may still read the one before
  int *s_bad = (int *)(smem + 4 * Sh::kTileBytes);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, c = lane & (C - 1),
            g = lane / C;
  // kv heads in turn, so that each die, which gets every eighth workgroup, has few
  const int x = div_by(a.by_heads, blockIdx.x), kvh = blockIdx.x - x * a.nkv, split = blockIdx.z;
  int s, tile;
  pick_tile(a.tile0, a.seqs, x, s, tile);
  const int rows = (a.start[s + 1] - a.start[s]) * a.G;        // of the sequence and kv head
  const int row0 = tile * Sh::kRows;
  const int base = a.len[s] - (a.start[s + 1] - a.start[s]);  // positions before the first row
  const int *tab = a.map.table + (size_t)(a.first_seq + s) * a.map.table_pages;
  const T *kc = (const T *)a.k + (size_t)kvh * HD, *vc = (const T *)a.v + (size_t)kvh * HD;

  // the positions of this split
  const int last_row = min(rows, row0 + Sh::kRows) - 1;
  const int extent = base + div_by(a.by_group, last_row) + 1;
  const int per = ((extent + a.splits - 1) / a.splits + KT - 1) / KT * KT;
  const int key_first = split * per, key_end = min(extent, key_first + per);

  // this lane's row
  const int row = row0 + C * wave + c;
  const bool live = row < rows;
  const int tok = div_by(a.by_group, live ? row : last_row), head = kvh * a.G + (live ? row : last_row) - tok * a.G;
  const size_t qrow = (size_t)(a.start[s] + tok) * a.nh + head;
  const int lim = base + tok;  // the last visible position
  // of the wave's rows: no mask is needed up to wave_all, nothing is seen after wave_any
  const int wrow = min(rows - 1, row0 + C * wave), wlast = min(rows - 1, row0 + C * wave + C - 1);
  const int wave_all = base + div_by(a.by_group, wrow), wave_any = base + div_by(a.by_group, wlast);

  v4u qv[KC];
  {
    const T *qp = (const T *)a.q + qrow * HD;
#pragma unroll
    for (int i = 0; i < KC; i++)
      qv[i] = (live ? *(const v4u *)(qp + (16 / sizeof(T)) * (NG * i + g)) : v4u{0, 0, 0, 0}) ^ a.q_sign;
  }
  Acc o[ND];
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int i = 0; i < NA; i++) o[d][i] = 0.0f;
  float m_ref = -INFINITY, l_run = 0.0f;  // the lane's own part of the sum

  // This wave's part of a tile's copies: WR rows, this lane's 16-byte chunk of row
  // u / CPR in each of NI pieces.  A tile's page ids are loaded two tiles ahead and
  // looked at one tile ahead: a wait for them between would also wait for the copies.
  // Absent positions and those behind key_end copy zeros (0 * NaN is NaN).
  constexpr int WR = KT / Sh::kWaves;
  const unsigned lds0 = lds_addr(smem);
  auto swz_chunk = [&](int i) {  // source chunk of piece i
    const int u = (wave * NI + i) * 64 + lane;
    return (u % CPR) ^ chunk_xor<CPR>(u / CPR);
  };
  int id[RUN ? 1 : NI];
  auto load_ids = [&](int key0) {
    if constexpr (RUN) {
      const int p = key0 + wave * WR;
      id[0] = p < key_end ? scalar_id(tab, div_by(a.map.div, p)) : -1;
    } else {
#pragma unroll
      for (int i = 0; i < NI; i++) id[i] = tab[div_by(a.map.div, min(key0 + ((wave * NI + i) * 64 + lane) / CPR, key_end - 1))];
    }
  };
  unsigned voff[RUN ? NI : 1];  // bytes from the run's first row
  if constexpr (RUN) {
#pragma unroll
    for (int i = 0; i < NI; i++)
      voff[i] = (unsigned)((i * 64 + lane) / CPR) * (unsigned)a.map.row * (unsigned)sizeof(T) + 16 * swz_chunk(i);
  }
  auto copy = [&](int key0, int tag) {
    const unsigned dst = lds0 + (tag & 1) * 2 * Sh::kTileBytes + wave * NI * 1024;
    bool bad = false;
    if constexpr (RUN) {
      const int p = key0 + wave * WR, pg = div_by(a.map.div, p);
      const bool there = (unsigned)id[0] < (unsigned)a.map.pages;
      bad = p < key_end && !there;
      const long long base = there ? (long long)id[0] * a.map.stride + (long long)(p - pg * a.map.page_size) * a.map.row : 0;
      if (there && p + WR <= key_end) {
#pragma unroll
        for (int i = 0; i < NI; i++) {
          dma_b128_s(kc + base, voff[i], dst + i * 1024);
          dma_b128_s(vc + base, voff[i], dst + i * 1024 + Sh::kTileBytes);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NI; i++) {
          const bool in = there && p + (i * 64 + lane) / CPR < key_end;
          const char *z = (const char *)g_zero_row + 16 * swz_chunk(i);
          dma_b128(in ? (const char *)(kc + base) + voff[i] : z, dst + i * 1024);
          dma_b128(in ? (const char *)(vc + base) + voff[i] : z, dst + i * 1024 + Sh::kTileBytes);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; i++) {
        const int p = key0 + ((wave * NI + i) * 64 + lane) / CPR, pg = div_by(a.map.div, p);
        const bool there = (unsigned)id[i] < (unsigned)a.map.pages, in = there && p < key_end;
        bad |= p < key_end && !there;
        const long long at = (long long)id[i] * a.map.stride + (long long)(p - pg * a.map.page_size) * a.map.row;
        const int ch = swz_chunk(i);
        const char *z = (const char *)g_zero_row + 16 * ch;
        dma_b128(in ? (const char *)(kc + at) + 16 * ch : z, dst + i * 1024);
        dma_b128(in ? (const char *)(vc + at) + 16 * ch : z, dst + i * 1024 + Sh::kTileBytes);
      }
    }
    if (__ballot(bad) && lane == 0) s_bad[tag & 3] = tag;
  };

  // Addresses within a tile, base ^ (chunk << 4) + row * RB: rows that differ by
  // 16 share their XOR, so a tile's reads have few distinct addresses and the rest
  // are immediate offsets.
  const unsigned k_at = c * RB + ((g ^ chunk_xor<CPR>(c)) << 4);
  const int vr0 = B16 ? 4 * g + ((lane & 15) >> 2) : 4 * g;
  const unsigned v_at = B16 ? vr0 * RB + (((C == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((lane & 3) >> 1)) ^ chunk_xor<CPR>(vr0)) * 16 + 8 * (lane & 1)
                            : vr0 * RB + (((c >> 2) ^ chunk_xor<CPR>(vr0)) << 4) + 4 * (c & 3);
  // the larger, or the sum, of a column's lane groups
  auto over_groups = [&](float x, auto op) {
    if constexpr (NG == 4) {
      const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      x = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
    }
    const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return op(__uint_as_float(p[0]), __uint_as_float(p[1]));
  };

  const int tiles = key_end > key_first ? (key_end - key_first + KT - 1) / KT : 0;
  if (tid < 4) s_bad[tid] = -1;
  __syncthreads();
  if (tiles > 0) {
    load_ids(key_first);
    copy(key_first, 0);
    if (tiles > 1) load_ids(key_first + KT);
  }
  for (int it = 0; it < tiles; it++) {
    const int key0 = key_first + it * KT;
    wait_dma();
    __syncthreads();
    if (it + 1 < tiles) {
      copy(key0 + KT, it + 1);
      if (it + 2 < tiles) load_ids(key0 + 2 * KT);
    }
    if (key0 > wave_any) continue;
    const unsigned tile_at = lds0 + (it & 1) * 2 * Sh::kTileBytes;
    // formed anew for each tile: kept over the loop, they would fill the registers
    unsigned ka = k_at + tile_at, va = v_at + tile_at + Sh::kTileBytes;
    asm volatile("" : "+v"(ka), "+v"(va));
    Acc sc[NS];
#pragma unroll
    for (int b = 0; b < NS; b++)
#pragma unroll
      for (int i = 0; i < NA; i++) sc[b][i] = 0.0f;
    const bool bad = s_bad[it & 3] == it;
    // S^T, the fragments of the next GK chunks on their way while GK are multiplied;
    // the fences keep the compiler from loading each where it is used
    {
      constexpr int GK = B16 ? (C == 16 ? 1 : 2) : 1, N = KC / GK;
      v4u kf[2][GK][NS];
      auto read = [&](int n) {
#pragma unroll
        for (int i = 0; i < GK; i++)
#pragma unroll
          for (int b = 0; b < NS; b++) kf[n & 1][i][b] = lds_v4u((ka ^ ((n * GK + i) * NG << 4)) + C * b * RB);
      };
      read(0);
#pragma unroll
      for (int n = 0; n < N; n++) {
        if (n + 1 < N) read(n + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < GK; i++)
#pragma unroll
          for (int b = 0; b < NS; b++) {
            if constexpr (!B16) {
#pragma unroll
              for (int e = 0; e < 4; e++)
                sc[b] = mfma_f32_32(__uint_as_float(kf[n & 1][i][b][e]), __uint_as_float(qv[n * GK + i][e]), sc[b]);
            } else if constexpr (C == 32) {
              sc[b] = Mat16<T>::mul32(kf[n & 1][i][b], qv[n * GK + i], sc[b]);
            } else {
              sc[b] = Mat16<T>::mul16(kf[n & 1][i][b], qv[n * GK + i], sc[b]);
            }
          }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (key0 + KT - 1 > wave_all || key0 + KT > key_end || bad) {
      unsigned long long present = ~0ull;
      if (bad) present = __ballot(key0 + lane < key_end && lane < KT && cell(a.map, tab, min(key0 + lane, key_end - 1)) >= 0);
      const int see = min(lim, key_end - 1) - key0;
#pragma unroll
      for (int b = 0; b < NS; b++)
#pragma unroll
        for (int i = 0; i < NA; i++) {
          const int p = C * b + 4 * NG * (i / 4) + 4 * g + i % 4;
          if (p > see || !(present >> p & 1)) sc[b][i] = -INFINITY;
        }
    }
    float bm = sc[0][0];
#pragma unroll
    for (int b = 0; b < NS; b++)
#pragma unroll
      for (int i = 0; i < NA; i++) bm = fmaxf(bm, sc[b][i]);
    bm = over_groups(bm, [](float x, float y) { return fmaxf(x, y); }) * a.scale;
    bm = below<T>(bm, 13.0f);
    // any reference serves the softmax: it follows the maximum only when that has
    // outgrown it by 2^kLag, so o is hardly ever rescaled.  The difference is exact where
    // m_ref + kLag is not: at 2^27, where numbers lie 16 apart, such a sum may be 16 more,
    // and 2^16 is no fp16 probability.
    if (__any(bm - m_ref > Sh::kLag)) {
      const float m_new = fmaxf(m_ref, bm), alpha = __builtin_amdgcn_exp2f(m_ref - (m_new == -INFINITY ? 0.0f : m_new));
      m_ref = m_new;
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < NA; i++) o[d][i] *= alpha;
    }
    const float m_use = m_ref == -INFINITY ? 0.0f : m_ref;
    float pr[KT / NG];  // in the order of the scores' registers
#pragma unroll
    for (int j = 0; j < KT / NG; j++) {
      pr[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[j / NA][j % NA], a.scale, -m_use));
      l_run += pr[j];
    }
    if constexpr (B16) {
      // eight probabilities of a lane: positions 8 NG st + 4 NG q + 4 g + 0 .. 3
      constexpr int swzq = chunk_xor<CPR>(4 * NG);
      constexpr int GV = C == 32 ? 2 : 4, N = KT / (8 * NG) * ND / GV;  // dim tiles of a group, groups
      v2u vf[2][GV][2];
      auto read = [&](int n) {
        const int st = n / (ND / GV), d0 = n % (ND / GV) * GV;
#pragma unroll
        for (int d = 0; d < GV; d++)
#pragma unroll
          for (int q = 0; q < 2; q++)
            vf[n & 1][d][q] = lds_transposed((va ^ ((d0 + d) * (C / 8) << 4) ^ (q * swzq << 4)) + (8 * NG * st + 4 * NG * q) * RB);
      };
      read(0);
#pragma unroll
      for (int n = 0; n < N; n++) {
        const int st = n / (ND / GV), d0 = n % (ND / GV) * GV;
        if (n + 1 < N) read(n + 1);
        const float *p8 = pr + 8 * st;
        const v4u pf = v4u{pack2<T>(p8[0], p8[1]), pack2<T>(p8[2], p8[3]), pack2<T>(p8[4], p8[5]), pack2<T>(p8[6], p8[7])};
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < GV; d++) {
          const v2u lo = vf[n & 1][d][0], hi = vf[n & 1][d][1];
          const v4u vt = v4u{lo[0], lo[1], hi[0], hi[1]};
          if constexpr (C == 32)
            o[d0 + d] = Mat16<T>::mul32(vt, pf, o[d0 + d]);
          else
            o[d0 + d] = Mat16<T>::mul16(vt, pf, o[d0 + d]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      float vf[2][ND];
      auto read = [&](int i) {
        const int r = 8 * (i / 4) + i % 4;
#pragma unroll
        for (int d = 0; d < ND; d++) vf[i & 1][d] = lds_f32((va ^ (((8 * d) ^ chunk_xor<CPR>(r)) << 4)) + r * RB);
      };
      read(0);
#pragma unroll
      for (int i = 0; i < 16; i++) {
        if (i + 1 < 16) read(i + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = mfma_f32_32(vf[i & 1][d], pr[i], o[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  l_run = over_groups(l_run, [](float x, float y) { return x + y; });

  // A position of a tile that a row does not see has the probability zero, and zero times
  // an infinite or NaN value is NaN.  Rows of the wave that are not finite are formed anew
  // from what they see, one by one, if one of the positions unseen by the first row
  // holds such a value: nothing any ordinary prompt pays for.  Where it runs, one wave
  // takes 1 to 2 ms a row and 5,000 positions: a NaN value in the last position of
  // prompts of 5,000 to 6,000 tokens 0.69 -> 35 ms (16 rows) and 0.43 -> 42 (32); in the
  // first, which every row sees, no more than without.
  float zero = 0.0f;
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int i = 0; i < NA; i++) zero += o[d][i] * 0.0f;
  unsigned long long odd = __ballot(live && zero != 0.0f);
  if (odd) {
    constexpr int E = HD / 64;  // dims of a lane
    typedef Pack<T, E> P;
    const int behind = min(key_end, key_first + ((wave_any - key_first) / KT + 1) * KT);
    bool hidden = false;
    for (int p = max(key_first, wave_all + 1); p < behind; p++) {
      const long long at = cell(a.map, tab, p);
      if (at < 0) continue;
      const P x = *(const P *)(vc + at + E * lane);
#pragma unroll
      for (int e = 0; e < E; e++) hidden |= (float)x.v[e] * 0.0f != 0.0f;
    }
    if (!__any(hidden)) odd = 0;
    for (int r = 0; r < C; r++) {
      if (!(odd >> r & (NG == 4 ? 0x1000100010001ull : 0x100000001ull))) continue;
      const int end = min(key_end, base + __shfl(tok, r) + 1);
      const float m = __shfl(m_ref == -INFINITY ? 0.0f : m_ref, r), sign = a.q_sign ? -a.scale : a.scale;
      const T *qp = (const T *)a.q + ((size_t)(a.start[s] + __shfl(tok, r)) * a.nh + __shfl(head, r)) * HD;
      float x[E] = {};
      for (int p0 = key_first; p0 < end; p0 += 64) {  // a lane a position, then all lanes a value
        const long long at = p0 + lane < end ? cell(a.map, tab, p0 + lane) : -1;
        const T *kp = kc + (at < 0 ? 0 : at);
        float w = 0.0f;
        for (int d = 0; d < HD; d += 4) {
          const Pack<T, 4> kv = *(const Pack<T, 4> *)(kp + d), qv = *(const Pack<T, 4> *)(qp + d);
#pragma unroll
          for (int e = 0; e < 4; e++) w = __builtin_fmaf((float)kv.v[e], (float)qv.v[e], w);
        }
        w = __builtin_amdgcn_exp2f(__builtin_fmaf(w, sign, -m));
        for (int j = 0; j < min(64, end - p0); j++) {
          const long long from = __shfl(at, j);
          if (from < 0) continue;
          const float wj = __shfl(w, j);
          const P v = *(const P *)(vc + from + E * lane);
#pragma unroll
          for (int e = 0; e < E; e++) x[e] = __builtin_fmaf(wj, (float)v.v[e], x[e]);
        }
      }
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < NA; i++) {
          const int dim = C * d + 4 * NG * (i / 4) + 4 * g + i % 4;
          const float y = __shfl(x[i % E], dim / E);
          if (c == r) o[d][i] = y;
        }
    }
  }
  if (!live) return;
  if (a.po) {
    const size_t rec = ((size_t)split * a.rows + (a.start[s] - a.start[0] + tok)) * a.nh + head;
    if (g == 0) {
      a.pm[rec] = l_run == 0.0f ? -INFINITY : m_ref == -INFINITY ? 0.0f : m_ref;  // a NaN sum is kept
      a.pl[rec] = l_run;
    }
    if (l_run == 0.0f) return;
    float *po = a.po + rec * HD;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int i = 0; i < NA / 4; i++)
        *(v4f *)(po + C * d + 4 * NG * i + 4 * g) = v4f{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
    return;
  }
  const float inv = l_run > 0.0f ? 1.0f / l_run : l_run == 0.0f ? 0.0f : l_run;
  const T *gp = a.gate ? (const T *)a.gate + (size_t)(a.start[s] + tok) * a.gate_stride + (size_t)head * a.gate_head : nullptr;
  T *op = (T *)a.out + qrow * HD;
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int i = 0; i < NA / 4; i++) {
      const int dim = C * d + 4 * NG * i + 4 * g;
      float y[4];
#pragma unroll
      for (int e = 0; e < 4; e++) y[e] = o[d][4 * i + e] * inv;
      if (gp) {
        const Pack<T, 4> gate = *(const Pack<T, 4> *)(gp + dim);
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] *= gate_sigmoid((float)gate.v[e]);
      }
      Pack<T, 4> r;
#pragma unroll
      for (int e = 0; e < 4; e++) r.v[e] = (T)y[e];
      *(Pack<T, 4> *)(op + dim) = r;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
bool pools_ok(const char *name, const ColiPaged *c, const void *k_pool, const void *v_pool, const int *table) {
  if (!c) return fail_arg("%s: null cache description", name), false;
  if (!type_bytes(c->type)) return fail_arg("%s: unknown element type %d", name, c->type), false;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail_arg("%s: head_dim %d is not 64, 128 or 256", name, c->head_dim), false;
  if (c->kv_heads <= 0 || c->query_heads <= 0 || c->query_heads % c->kv_heads || c->query_heads > 65535)
    return fail_arg("%s: query_heads %d (1..65535) must be a multiple of kv_heads %d", name, c->query_heads, c->kv_heads),
           false;
  if (c->page_size <= 0 || c->pages <= 0 || c->table_pages <= 0 || (long long)c->pages * c->page_size > INT_MAX ||
      (long long)c->table_pages * c->page_size > 1 << 30)  // a tile behind the last position is an int too
    return fail_arg("%s: page_size, pages and table_pages must be positive, pages * page_size below 2^31, "
                    "table_pages * page_size at most 2^30", name),
           false;
  const long long page = (long long)c->page_size * c->kv_heads * c->head_dim;
  if (c->page_stride < page || c->page_stride % 8 || c->page_stride > LLONG_MAX / 8 / c->pages)
    return fail_arg("%s: page_stride %lld must be a multiple of 8 and at least one page's %lld elements", name,
                    c->page_stride, page),
           false;
  if (!k_pool || !v_pool || !table) return fail_arg("%s: null pool or page table", name), false;
  if (!aligned16(k_pool) || !aligned16(v_pool)) return fail_arg("%s: pools must be 16-byte aligned", name), false;
  if ((uintptr_t)table & 3) return fail_arg("%s: the page table must be 4-byte aligned", name), false;
  return true;
}

constexpr int kMostRows = (1 << 24) - 1;
bool rows_ok(const char *name, const ColiPaged *c, const int *start, const int *length, int sequences) {
  if (sequences < 0 || (sequences && !length)) return fail_arg("%s: null lengths or negative sequence count", name), false;
  if (start && sequences && start[0] < 0) return fail_arg("%s: start[0] is negative", name), false;
  // a launch takes fewer than 2^32 threads
  if (start && sequences && (long long)start[sequences] - start[0] > kMostRows)
    return fail_arg("%s: %d rows in a call, more than 2^24 - 1", name, start[sequences] - start[0]), false;
  for (int s = 0; s < sequences; s++) {
    if (length[s] < 0 || length[s] > (long long)c->table_pages * c->page_size)
      return fail_arg("%s: length[%d] = %d is outside 0..%lld", name, s, length[s], (long long)c->table_pages * c->page_size),
             false;
    if (start && (start[s + 1] < start[s] || start[s + 1] - start[s] > length[s]))
      return fail_arg("%s: sequence %d has rows %d..%d and length %d", name, s, start[s], start[s + 1], length[s]), false;
  }
  return true;
}

bool gate_ok(const char *name, const ColiPaged *c, const void *gate, long long stride, int head) {
  if (!gate) return true;
  if (((uintptr_t)gate & (4 * type_bytes(c->type) - 1)) || stride % 4 || head % 4 || stride < 0 || head < 0)
    return fail_arg("%s: gates must be aligned to four elements, their strides non-negative multiples of 4", name), false;
  return true;
}

PageMap page_map(const ColiPaged *c, const int *table) {
  return {table, c->pages, c->table_pages, c->page_size, fast_div(c->page_size), c->page_stride, c->kv_heads * c->head_dim};
}

int cus_of(const ColiCuda *ctx) { return ctx->sm_count > 0 ? ctx->sm_count : 256; }

template <class T>
void launch_append(const AppendArgs &a, int hd, dim3 grid, hipStream_t st) {
  if (hd == 64)
    k_paged_append<T, 64><<<grid, 256, 0, st>>>(a);
  else if (hd == 128)
    k_paged_append<T, 128><<<grid, 256, 0, st>>>(a);
  else
    k_paged_append<T, 256><<<grid, 256, 0, st>>>(a);
}

template <class T, int HD>
void launch_decode(const DecodeArgs &a, unsigned grid, hipStream_t st) {
  if (a.map.page_size % 16 == 0)
    k_paged_decode<T, HD, true><<<grid, 256, 0, st>>>(a);
  else
    k_paged_decode<T, HD, false><<<grid, 256, 0, st>>>(a);
}
template <class T>
void launch_decode(const DecodeArgs &a, int hd, unsigned grid, hipStream_t st) {
  if (hd == 64)
    launch_decode<T, 64>(a, grid, st);
  else if (hd == 128)
    launch_decode<T, 128>(a, grid, st);
  else
    launch_decode<T, 256>(a, grid, st);
}

template <class T, int HD>
void launch_join(const JoinArgs &a, int splits, dim3 grid, hipStream_t st) {
  if (splits <= 2 * kJoinLoads * (128 / (HD / 4)) && (long long)grid.x * grid.y >= 1024)
    k_paged_join<T, HD, 128><<<grid, 128, 0, st>>>(a);
  else
    k_paged_join<T, HD, 512><<<grid, 512, 0, st>>>(a);
}
// splits: of a row, at most
template <class T>
void launch_join(const JoinArgs &a, int hd, int splits, int rows, hipStream_t st) {
  const dim3 grid(a.nh, rows);  // a prompt in splits has fewer tiles of 128 rows than there are compute units
  if (hd == 64)
    launch_join<T, 64>(a, splits, grid, st);
  else if (hd == 128)
    launch_join<T, 128>(a, splits, grid, st);
  else
    launch_join<T, 256>(a, splits, grid, st);
}

template <class T, int HD, bool RUN, int C>
int launch_prompt(const char *name, const PromptArgs &a, dim3 grid, hipStream_t st) {
  typedef PromptShape<T, HD, C> Sh;
  const hipError_t e =
      hipFuncSetAttribute((const void *)k_paged_prompt<T, HD, RUN, C>, hipFuncAttributeMaxDynamicSharedMemorySize, Sh::kLds);
  if (e != hipSuccess) return fail_hip(name, e);
  k_paged_prompt<T, HD, RUN, C><<<grid, 64 * Sh::kWaves, Sh::kLds, st>>>(a);
  return 0;
}
template <class T, int HD, int C>
int launch_prompt(const char *name, const PromptArgs &a, dim3 grid, hipStream_t st) {
  typedef PromptShape<T, HD, C> Sh;
  return a.map.page_size % (Sh::kKeys / Sh::kWaves) == 0 ? launch_prompt<T, HD, true, C>(name, a, grid, st)
                                                         : launch_prompt<T, HD, false, C>(name, a, grid, st);
}
// few: no more workgroups than compute units
template <class T, int HD>
int launch_prompt(const char *name, const PromptArgs &a, bool few, dim3 grid, hipStream_t st) {
  if constexpr (sizeof(T) == 4)
    return launch_prompt<T, HD, 32>(name, a, grid, st);
  else if constexpr (HD == 256)
    return launch_prompt<T, HD, 16>(name, a, grid, st);
  else
    return few ? launch_prompt<T, HD, 16>(name, a, grid, st) : launch_prompt<T, HD, 32>(name, a, grid, st);
}
constexpr int kPromptRows = PromptShape<float, 64, 32>::kRows;
static_assert(PromptShape<__bf16, 256, 16>::kRows == kPromptRows, "rows of a tile, the same for all");
template <class T>
int launch_prompt(const char *name, const PromptArgs &a, int hd, bool few, dim3 grid, hipStream_t st) {
  return hd == 64    ? launch_prompt<T, 64>(name, a, few, grid, st)
         : hd == 128 ? launch_prompt<T, 128>(name, a, few, grid, st)
                     : launch_prompt<T, 256>(name, a, few, grid, st);
}
int prompt_keys(int type) { return type != COLI_TYPE_F32 ? 64 : 32; }

// Partial records of n (split, row) pairs: outputs, maxima, sums.  A decoding loop needs a
// split more every some hundred tokens, so the first call takes what its heads can come
// to: (split, row, head) records of 128 rows a compute unit for prompts, of 16 heads a
// workgroup and three rounds of four workgroups a compute unit for single tokens, and one
// for each sequence of a launch; 64 MiB at most (14, 28, 55 MB at 32 heads of 64, 128, 256).
int partials(ColiCuda *ctx, const char *name, size_t n, int nh, int hd, float **po, float **pm, float **pl) {
  const size_t heads = n * nh, record = (hd + 2) * sizeof(float), cus = cus_of(ctx);
  size_t room = 12 * 16 * cus + (size_t)kSeqs * nh;
  if (room < 128 * cus) room = 128 * cus;
  room = room * record < (64u << 20) ? room * record : 64u << 20;
  if (room < heads * record) room = heads * record / 2 * 3;
  if (ensure_room(ctx, kScrPaged, heads * record, room, name)) return -1;
  *po = (float *)ctx->scratch[kScrPaged];
  *pm = *po + heads * hd;
  *pl = *pm + heads;
  return 0;
}

}  // namespace
}  // namespace sw

using namespace sw;

extern "C" int coli_cuda_paged_append(ColiCuda *ctx, const ColiPaged *c, void *k_pool, void *v_pool, const int *table,
                                      const int *start, const int *length, int sequences, void *q_out, const void *q,
                                      long long q_stride, int q_head_stride, const void *k, long long k_stride,
                                      const void *v, long long v_stride, const float *q_norm, const float *k_norm,
                                      float eps, int rotary_dim, float theta) {
  static const char *name = "coli_cuda_paged_append";
  if (!pools_ok(name, c, k_pool, v_pool, table)) return -1;
  if (sequences && !start) return fail_arg("%s: null start", name);
  if (!rows_ok(name, c, start, length, sequences)) return -1;
  if (!k || !v || !q != !q_out) return fail_arg("%s: null keys or values, or one of q and q_out", name);
  if (!aligned16(k) || !aligned16(v) || !aligned16(q) || !aligned16(q_out) || k_stride % 8 || v_stride % 8 ||
      (q && (q_stride % 8 || q_head_stride % 8)) || k_stride < 0 || v_stride < 0 || q_stride < 0 || q_head_stride < 0)
    return fail_arg("%s: tensors must be 16-byte aligned, strides non-negative multiples of 8 elements", name);
  if (((uintptr_t)q_norm | (uintptr_t)k_norm) & 3) return fail_arg("%s: norms must be 4-byte aligned", name);
  if (rotary_dim < 0 || rotary_dim > c->head_dim || rotary_dim % 2)
    return fail_arg("%s: rotary_dim %d must be even and within head_dim", name, rotary_dim);
  if (rotary_dim && !(theta > 0.0f && theta < INFINITY)) return fail_arg("%s: theta must be positive and finite", name);
  if ((q_norm || k_norm) && !(eps >= 0.0f && eps < INFINITY)) return fail_arg("%s: eps must be finite, not negative", name);
  if (!ctx) return fail_arg("%s: null context", name);
  OnDevice on(ctx);
  AppendArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q, a.k = k, a.v = v;
  a.q_out = q_out, a.k_pool = k_pool, a.v_pool = v_pool;
  a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride;
  a.q_norm = q_norm, a.k_norm = k_norm;
  a.q_head = q_head_stride, a.nh = c->query_heads, a.nkv = c->kv_heads, a.rd = rotary_dim;
  a.eps = eps;
  a.map = page_map(c, table);
  if (rotary_dim) {
    // theta^(-2 i / rotary_dim) / 2 pi by repeated products in 64 bits (127 of them: 2^-46)
    const double ratio = pow((double)theta, -2.0 / rotary_dim);
    a.freq[0] = 0.15915494309189535;
    for (int i = 1; i < rotary_dim / 2; i++) a.freq[i] = a.freq[i - 1] * ratio;
  }
  const int heads = (q ? c->query_heads : 0) + c->kv_heads;
  for (int s0 = 0; s0 < sequences; s0 += kSeqs) {
    const int n = sequences - s0 < kSeqs ? sequences - s0 : kSeqs, rows = start[s0 + n] - start[s0];
    if (!rows) continue;
    memcpy(a.start, start + s0, (n + 1) * sizeof(int));
    memcpy(a.len, length + s0, n * sizeof(int));
    a.seqs = n;
    a.first_seq = s0;
    // few tokens: their heads over several workgroups, four heads (one a wave) at least
    int gy = 4 * cus_of(ctx) / rows;
    if (gy > (heads + 3) / 4) gy = (heads + 3) / 4;
    if (gy < 1) gy = 1;
    a.heads_per_block = ((heads + gy - 1) / gy + 3) / 4 * 4;
    const dim3 grid(rows, (heads + a.heads_per_block - 1) / a.heads_per_block);
    if (c->type == COLI_TYPE_F32)
      launch_append<float>(a, c->head_dim, grid, ctx->stream);
    else if (c->type == COLI_TYPE_F16)
      launch_append<_Float16>(a, c->head_dim, grid, ctx->stream);
    else
      launch_append<__bf16>(a, c->head_dim, grid, ctx->stream);
  }
  return launch_status(name);
}

extern "C" int coli_cuda_paged_decode(ColiCuda *ctx, const ColiPaged *c, void *out, const void *q, const void *gate,
                                      long long gate_stride, int gate_head_stride, const void *k_pool, const void *v_pool,
                                      const int *table, const int *length, int sequences, float scale) {
  static const char *name = "coli_cuda_paged_decode";
  if (!pools_ok(name, c, k_pool, v_pool, table) || !rows_ok(name, c, nullptr, length, sequences) ||
      !gate_ok(name, c, gate, gate_stride, gate_head_stride))
    return -1;
  if (!out || !q || !aligned16(out) || !aligned16(q)) return fail_arg("%s: q and out must be 16-byte aligned", name);
  if (!isfinite(scale * kLog2e)) return fail_arg("%s: scale, or scale * log2(e), is not finite", name);
  if (!ctx) return fail_arg("%s: null context", name);
  OnDevice on(ctx);
  const int nh = c->query_heads, hd = c->head_dim, size = type_bytes(c->type);
  DecodeArgs a;
  memset(&a, 0, sizeof(a));
  a.k = k_pool, a.v = v_pool;
  a.gate_stride = gate_stride;
  a.gate_head = gate_head_stride;
  a.nh = nh, a.nkv = c->kv_heads, a.G = nh / c->kv_heads;
  a.hgroups = (a.G + 15) / 16;
  a.scale = scale * kLog2e;
  a.map = page_map(c, table);
  const long long items = (long long)c->kv_heads * a.hgroups;
  const bool runs = c->page_size % 16 == 0;
  const int least = c->type == COLI_TYPE_F32 ? DecodeShape<float, 64, true>::kLeast : DecodeShape<__bf16, 64, true>::kLeast;
  const int per_cu = hd == 64    ? (runs ? DecodeShape<__bf16, 64, true>::kPerCu : DecodeShape<__bf16, 64, false>::kPerCu)
                     : hd == 128 ? (runs ? DecodeShape<__bf16, 128, true>::kPerCu : DecodeShape<__bf16, 128, false>::kPerCu)
                                 : DecodeShape<__bf16, 256, true>::kPerCu;
  for (int s0 = 0; s0 < sequences; s0 += kSeqs) {
    const int n = sequences - s0 < kSeqs ? sequences - s0 : kSeqs;
    int longest = 0;
    long long total = 0;
    for (int r = 0; r < n; r++) {
      total += length[s0 + r];
      if (length[s0 + r] > longest) longest = length[s0 + r];
    }
    // All splits of one length, in blocks of the four waves.  Where a compute unit holds
    // one workgroup, the least length whose workgroups all run at once: 13 fp32
    // sequences up to 6,000 positions 31 us and 4.6 of join, in two and three rounds 41 and
    // 48; three bf16 ones up to 131,071 79 and 4.8, against 83 and 6.4, 91 and 7.6.  Where it holds several (or one
    // round leaves the longest split half as much again as an even share, beside many
    // short sequences), a third of an even share, in rounds that level out: 48 fp16
    // sequences up to 9,001 at head dim 128 160 us in one round, 145 / 143 / 143 at a
    // half / third / quarter, at head dim 64 124 and 109 / 105 / 104.
    const long long slots = (long long)per_cu * cus_of(ctx), share = (total * items + slots - 1) / slots;
    const long long most = ((longest + kMaxSplits - 1) / kMaxSplits + least - 1) / least;  // kMaxSplits a sequence
    long long lo = most, hi = ((long long)longest + least - 1) / least;
    if (lo < 1) lo = 1;
    if (hi < lo) hi = lo;
    if (per_cu == 1) {
      auto workgroups = [&](long long per) {
        long long sum = 0;
        for (int r = 0; r < n; r++) sum += length[s0 + r] <= per ? 1 : (length[s0 + r] + per - 1) / per;
        return sum * items;
      };
      while (lo < hi) {  // the least in [lo, hi] that fits, or hi: one split a sequence
        const long long mid = (lo + hi) / 2;
        if (workgroups(mid * least) <= slots)
          hi = mid;
        else
          lo = mid + 1;
      }
    }
    if (per_cu > 1 || 2 * lo * least > 3 * share) {
      const long long third = (share / 3 + least - 1) / least;
      lo = third > most ? third : most;
      if (lo < 1) lo = 1;
    }
    a.per = (int)(lo * least < INT_MAX / 2 ? lo * least : INT_MAX / 2 / least * least);
    int splits = 1;
    a.first[0] = 0;
    for (int r = 0; r < n; r++) {
      const int S = length[s0 + r] <= a.per ? 1 : (int)(((long long)length[s0 + r] + a.per - 1) / a.per);
      a.first[r + 1] = a.first[r] + S;
      if (S > splits) splits = S;
    }
    memcpy(a.len, length + s0, n * sizeof(int));
    a.rows = n;
    a.first_seq = s0;
    a.q = (const char *)q + (size_t)s0 * nh * hd * size;
    a.out = (char *)out + (size_t)s0 * nh * hd * size;
    a.gate = gate ? (const char *)gate + (size_t)s0 * gate_stride * size : nullptr;
    a.po = a.pm = a.pl = nullptr;
    if (splits > 1 && partials(ctx, name, a.first[n], nh, hd, &a.po, &a.pm, &a.pl)) return -1;
    const unsigned grid = (unsigned)(a.first[n] * items);
    if (c->type == COLI_TYPE_F32)
      launch_decode<float>(a, hd, grid, ctx->stream);
    else if (c->type == COLI_TYPE_F16)
      launch_decode<_Float16>(a, hd, grid, ctx->stream);
    else
      launch_decode<__bf16>(a, hd, grid, ctx->stream);
    if (splits == 1) continue;
    JoinArgs j;
    memset(&j, 0, sizeof(j));
    j.po = a.po, j.pm = a.pm, j.pl = a.pl;
    j.gate = a.gate;
    j.out = a.out;
    j.gate_stride = gate_stride;
    j.gate_head = gate_head_stride;
    j.nh = nh;
    j.flat = 1;
    memcpy(j.first, a.first, sizeof(a.first));
    if (c->type == COLI_TYPE_F32)
      launch_join<float>(j, hd, splits, n, ctx->stream);
    else if (c->type == COLI_TYPE_F16)
      launch_join<_Float16>(j, hd, splits, n, ctx->stream);
    else
      launch_join<__bf16>(j, hd, splits, n, ctx->stream);
  }
  return launch_status(name);
}

extern "C" int coli_cuda_paged_prompt(ColiCuda *ctx, const ColiPaged *c, void *out, const void *q, const void *gate,
                                      long long gate_stride, int gate_head_stride, const void *k_pool, const void *v_pool,
                                      const int *table, const int *start, const int *length, int sequences, float scale) {
  static const char *name = "coli_cuda_paged_prompt";
  if (!pools_ok(name, c, k_pool, v_pool, table)) return -1;
  if (sequences && !start) return fail_arg("%s: null start", name);
  if (!rows_ok(name, c, start, length, sequences) || !gate_ok(name, c, gate, gate_stride, gate_head_stride)) return -1;
  if (!out || !q || !aligned16(out) || !aligned16(q)) return fail_arg("%s: q and out must be 16-byte aligned", name);
  if (!isfinite(scale * kLog2e)) return fail_arg("%s: scale, or scale * log2(e), is not finite", name);
  const int nh = c->query_heads, hd = c->head_dim, G = nh / c->kv_heads, R = kPromptRows;
  // (token, head) rows of a call, which also bounds a launch's threads: 256 a tile of 128
  // rows, or 512 at head_dim 256
  long long all = 0;
  for (int s = 0; s < sequences; s++) all += ((long long)(start[s + 1] - start[s]) * G + R - 1) / R * R * c->kv_heads;
  if (all > 1 << 29) return fail_arg("%s: %lld (row, query head) pairs in tiles of %d, more than 2^29", name, all, R);
  if (!ctx) return fail_arg("%s: null context", name);
  OnDevice on(ctx);
  PromptArgs a;
  memset(&a, 0, sizeof(a));
  a.q = q, a.k = k_pool, a.v = v_pool;
  a.out = out;
  a.gate = gate;
  a.gate_stride = gate_stride;
  a.gate_head = gate_head_stride;
  a.nh = nh, a.nkv = c->kv_heads, a.G = G;
  a.scale = fabsf(scale) * kLog2e;
  if (!(a.scale >= 1e-38f)) a.scale = 1e-38f;  // no scores at all: equal ones
  if (scale < 0.0f) a.q_sign = c->type == COLI_TYPE_F32 ? 0x80000000u : 0x80008000u;
  a.by_group = fast_div(G);
  a.by_heads = fast_div(c->kv_heads);
  a.map = page_map(c, table);
  for (int s0 = 0; s0 < sequences; s0 += kSeqs) {
    const int n = sequences - s0 < kSeqs ? sequences - s0 : kSeqs, rows = start[s0 + n] - start[s0];
    if (!rows) continue;
    long long tiles = 0;
    int longest = 0;
    a.tile0[0] = 0;
    for (int s = 0; s < n; s++) {
      const int m = start[s0 + s + 1] - start[s0 + s];
      tiles += ((long long)m * G + R - 1) / R;
      a.tile0[s + 1] = (int)tiles;
      if (m && length[s0 + s] > longest) longest = length[s0 + s];
    }
    memcpy(a.start, start + s0, (n + 1) * sizeof(int));
    memcpy(a.len, length + s0, n * sizeof(int));
    a.seqs = n;
    a.first_seq = s0;
    a.rows = rows;
    // few tiles: their positions over several workgroups, four tiles of positions each at least
    long long splits = cus_of(ctx) / (tiles * c->kv_heads), most = longest / (4 * prompt_keys(c->type));
    if (splits > most) splits = most;
    if (splits > kMaxSplits) splits = kMaxSplits;
    a.splits = splits < 1 ? 1 : (int)splits;
    a.po = a.pm = a.pl = nullptr;
    if (a.splits > 1 && partials(ctx, name, (size_t)a.splits * rows, nh, hd, &a.po, &a.pm, &a.pl)) return -1;
    const dim3 grid((unsigned)(tiles * c->kv_heads), 1, a.splits);
    const bool few = tiles * c->kv_heads <= cus_of(ctx);  // the splits fill no more than the compute units
    const int rc = c->type == COLI_TYPE_F32   ? launch_prompt<float>(name, a, hd, few, grid, ctx->stream)
                   : c->type == COLI_TYPE_F16 ? launch_prompt<_Float16>(name, a, hd, few, grid, ctx->stream)
                                              : launch_prompt<__bf16>(name, a, hd, few, grid, ctx->stream);
    if (rc) return -1;
    if (a.splits == 1) continue;
    JoinArgs j;
    memset(&j, 0, sizeof(j));
    j.po = a.po, j.pm = a.pm, j.pl = a.pl;
    j.gate = gate;
    j.out = out;
    j.gate_stride = gate_stride;
    j.gate_head = gate_head_stride;
    j.nh = nh;
    j.S = a.splits;
    j.step = rows;
    j.row0 = start[s0];
    if (c->type == COLI_TYPE_F32)
      launch_join<float>(j, hd, a.splits, rows, ctx->stream);
    else if (c->type == COLI_TYPE_F16)
      launch_join<_Float16>(j, hd, a.splits, rows, ctx->stream);
    else
      launch_join<__bf16>(j, hd, a.splits, rows, ctx->stream);
  }
  return launch_status(name);
}
