// Differential attention: the difference of two softmax maps over shared values, with a learned weight per head,
//   P_c = softmax(Q_c K_c^T scale + mask)  (c = 1, 2),   O = (P_1 - lam P_2) V,
// its backward pass
//   dP = dO V^T,  delta_c = sum_n dO_n O_c,n,  dS_1 = P_1 (dP - delta_1),  dS_2 = -lam P_2 (dP - delta_2)
//   dQ_c = scale dS_c K_c,  dK_c = scale dS_c^T Q_c,  dV = (P_1 - lam P_2)^T dO,  dlam = -sum P_2 dP
// and its single-token form over a long cache (the keys split over workgroups and joined).
//
// Layout.  The G = H / Hkv query heads that share a key head are packed into the rows of one problem: row r of
// (batch, key head) is position r / G of head r % G, so a key tile is read once for all of them, their gradients add up
// inside one workgroup (no atomics), and a single token still has G rows for the matrix unit.
// A wave holds 32 rows (keys in the dK / dV kernel) as the COLUMNS of every product on
// v_mfma_f32_32x32x16: the scores come out transposed, S^T = K Q^T, so a row's softmax statistics live in one lane (and its
// neighbour 32 away), the probabilities are already the B operand of O^T = V^T P^T, and a rescale is a lane's own
// factor.  K, V (Q, dO) tiles of 32 rows go through LDS, read once along a row (ds_read_b128) and once down the columns
// (the LDS transpose read); 16-byte chunks are XORed with the row so that both are free of bank conflicts.
// Softmax in base 2 with one running maximum per map, taken up only when a score passes it by 2^8; statistics,
// accumulators and dlam's sum are fp32.  Roundings to 16 bits: P and dS as matrix operands (the instruction's
// type) and the results; fp16's dS is first scaled by a power of two that follows its size.
#include <algorithm>
#include <atomic>

#include "ctr_hip.h"
#include "vec16.h"

namespace ctr {
namespace {

struct DaArgs {
  const void *q, *k, *v, *dout;
  const float* lam;
  void *o, *o2;                  // (B, T, H, 2 D); o2 = P_2 V, kept for the backward (may be null)
  float* stat;                   // 4 planes of rows: log2 sums of the maps, then delta_1, delta_2
  void *dq, *dk, *dv;
  float* dlrow;                  // per row sum_j P_2 dP
  float* part;                   // split keys: partial results
  const int *q_lens, *kv_lens;
  long q_sb, q_st, q_sh, q_sc, k_sb, k_ss, k_sh, k_sc, v_sb, v_ss, v_sh, g_sb, g_st, g_sh;
  long rows;                     // B Hkv R
  float c, scale;                // scale log2(e), scale
  int B, T, S, H, Hkv, G, R, causal, splits, tiles;
};

template <typename T> struct Mfma;
template <> struct Mfma<__bf16> {
  static __device__ __forceinline__ f32x16 run(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma<_Float16> {
  static __device__ __forceinline__ f32x16 run(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));

// C layout of a 32x32 tile: register r of lane l holds row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32
__device__ __forceinline__ int c_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// A tile of rows of CH 16-byte chunks in LDS.  Chunk c of a row stands at slot(row, c): sixteen consecutive rows' equal
// chunks, and four consecutive rows' four-chunk groups, cover the 64 banks once.
template <int CH>
__device__ __forceinline__ int slot(int row, int c) {
  if constexpr (CH >= 16) return row * CH + (c ^ (((row & 3) << 2) | ((row >> 2) & 3)));
  else return row * CH + (c ^ ((((row >> 1) & 1) << 2) | ((row >> 2) & 3)));
}
// 32 rows x 16 k, k contiguous along a row: lane l has row l % 32, k = 16 kk + 8 (l / 32) + 0..7
template <typename T, int CH>
__device__ __forceinline__ typename Vec<T>::v8 frag_row(const T* s, int kk, int lane) {
  return *(const typename Vec<T>::v8*)(s + slot<CH>(lane & 31, 2 * kk + (lane >> 5)) * 8);
}
// 16 rows (from r0) as k x 32 columns (from c0): lane l has column l % 32 and the rows 4 (l / 32) + 0..3, 8 + 4 (l / 32)
// + 0..3 -- the order in which a C tile's registers 8 i .. 8 i + 7 hold the rows of its i-th half
template <typename T, int CH>
__device__ __forceinline__ typename Vec<T>::v8 frag_col(const T* s, int r0, int c0, int lane) {
  const int row = r0 + 4 * (lane >> 5) + ((lane & 15) >> 2), c = c0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  auto p = (__attribute__((address_space(3))) s16x4*)(s + slot<CH>(row, c >> 3) * 8 + (c & 4));
  auto p8 = (__attribute__((address_space(3))) s16x4*)(s + slot<CH>(row + 8, c >> 3) * 8 + (c & 4));
  const auto u = __builtin_bit_cast(typename Vec<T>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
  const auto w = __builtin_bit_cast(typename Vec<T>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p8));
  return __builtin_shufflevector(u, w, 0, 1, 2, 3, 4, 5, 6, 7);
}
// registers 8 i .. 8 i + 7 of a C tile as an operand
template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 pack(const f32x16& v, int i) {
  f32x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = v[8 * i + j];
  return __builtin_convertvector(o, typename Vec<T>::v8);
}

// 32 rows to LDS: NT threads, row r from src + row_off(r), its second half at `half` elements more; rows from `valid` on
// are zeros (what stands behind the end of a cache is not read)
template <typename T, int CH, int NT, typename F>
__device__ __forceinline__ void load_tile(T* dst, int valid, long half, F row_ptr) {
  typedef typename Vec<T>::v8 v8;
#pragma unroll
  for (int j = 0; j < (32 * CH + NT - 1) / NT; ++j) {
    const int i = threadIdx.x + j * NT, r = i / CH, c = i % CH;
    if ((32 * CH) % NT && i >= 32 * CH) break;
    v8 x = {};
    if (r < valid) x = *(const v8*)(row_ptr(r) + (c < CH / 2 ? c * 8 : half + (c - CH / 2) * 8));
    *(v8*)(dst + slot<CH>(r, c) * 8) = x;
  }
}

struct Seq {
  int b, hk, ql, kl;      // batch, key head, rows' and keys' valid lengths
  __device__ __forceinline__ Seq(const DaArgs& a, int bh) {
    b = bh / a.Hkv;
    hk = bh - b * a.Hkv;
    ql = a.q_lens ? min(max(a.q_lens[b], 0), a.T) : a.T;
    kl = a.kv_lens ? min(max(a.kv_lens[b], 0), a.S) : a.S;
  }
  // keys that position t sees: [0, limit)
  __device__ __forceinline__ int limit(const DaArgs& a, int t) const {
    if (t >= ql) return 0;
    return a.causal ? min(kl, max(0, t + 1 + kl - ql)) : kl;
  }
};

// ------------------------------------------------------------------------------------------------ forward
template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 128 ? 1 : 2) void da_fwd(const DaArgs a) {
  constexpr int CH = D / 4, DV = 2 * D, NT = 64 * NW, KQ = D / 16, NO = DV / 32;
  typedef typename Vec<T>::v8 v8;
  __shared__ __align__(16) T ks[32 * DV], vs[32 * DV];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
  int id = blockIdx.x;
  const int tile = id % a.tiles;
  id /= a.tiles;
  const int bh = id % (a.B * a.Hkv), sp = id / (a.B * a.Hkv);
  const Seq s(a, bh);
  const int row = tile * 32 * NW + wave * 32 + (lane & 31), rr = min(row, a.R - 1), t = rr / a.G, head = s.hk * a.G + rr - t * a.G;
  const int lim = s.limit(a, t);
  // the keys of the block: those its last row sees, and of them this split's share
  const int t_last = min((min(tile * 32 * NW + 32 * NW, a.R) - 1) / a.G, s.ql - 1);
  int k0 = 0, k1 = t_last < 0 ? 0 : s.limit(a, t_last);
  if (a.splits > 1) {
    const int per = (((k1 + a.splits - 1) / a.splits) + 31) / 32 * 32;
    k0 = min(k1, sp * per);
    k1 = min(k1, k0 + per);
  }
  const T* qp = (const T*)a.q + s.b * a.q_sb + t * a.q_st + head * a.q_sh;
  v8 qf[2][KQ];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int k = 0; k < KQ; ++k) qf[c][k] = *(const v8*)(qp + c * a.q_sc + 16 * k + 8 * h);
  const T* kp = (const T*)a.k + s.b * a.k_sb + s.hk * a.k_sh;
  const T* vp = (const T*)a.v + s.b * a.v_sb + s.hk * a.v_sh;
  f32x16 o[2][NO];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < NO; ++j) o[c][j] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  for (int kb = k0; kb < k1; kb += 32) {
    __syncthreads();
    load_tile<T, CH, NT>(ks, min(32, k1 - kb), a.k_sc, [&](int r) { return kp + (long)(kb + r) * a.k_ss; });
    load_tile<T, CH, NT>(vs, min(32, k1 - kb), D, [&](int r) { return vp + (long)(kb + r) * a.v_ss; });
    __syncthreads();
    f32x16 sc[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      sc[c] = 0.f;
#pragma unroll
      for (int k = 0; k < KQ; ++k) sc[c] = Mfma<T>::run(frag_row<T, CH>(ks, c * KQ + k, lane), qf[c][k], sc[c]);
    }
    const int end = min(lim, k1) - kb;
    if (__any(end < 32)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool seen = c_row(r, h) < end;
        sc[0][r] = seen ? sc[0][r] : -INFINITY;
        sc[1][r] = seen ? sc[1][r] : -INFINITY;
      }
    }
    v8 pf[2][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float top = sc[c][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) top = fmaxf(top, sc[c][r]);
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      if (__any((top - m[c]) * a.c > 8.f)) {        // also the first keys: from -inf (equal -inf gives NaN: no)
        const float mn = fmaxf(m[c], top), f = m[c] == mn ? 1.f : exp2f((m[c] - mn) * a.c);
        l[c] *= f;
#pragma unroll
        for (int j = 0; j < NO; ++j) o[c][j] *= f;
        m[c] = mn;
      }
      const float base = m[c] == -INFINITY ? 0.f : m[c] * a.c;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        sc[c][r] = __builtin_amdgcn_exp2f(fmaf(sc[c][r], a.c, -base));
        l[c] += sc[c][r];
      }
      pf[c][0] = pack<T>(sc[c], 0);
      pf[c][1] = pack<T>(sc[c], 1);
    }
#pragma unroll
    for (int j = 0; j < NO; ++j)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const v8 vf = frag_col<T, CH>(vs, 16 * i, 32 * j, lane);
        o[0][j] = Mfma<T>::run(vf, pf[0][i], o[0][j]);
        o[1][j] = Mfma<T>::run(vf, pf[1][i], o[1][j]);
      }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) l[c] += __shfl_xor(l[c], 32, 64);
  if (row >= a.R) return;
  const long n = (long)bh * a.R + row;
  if (a.splits > 1) {
    float* p = a.part + ((long)sp * a.rows + n) * (2 * DV + 4);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int j = 0; j < NO; ++j)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          f32x4 x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = o[c][j][4 * r4 + r];
          *(f32x4*)(p + c * DV + 32 * j + 8 * r4 + 4 * h) = x;
        }
      if (h == 0) {
        p[2 * DV + 2 * c] = m[c];
        p[2 * DV + 2 * c + 1] = l[c];
      }
    }
    return;
  }
  const float lam = a.lam[head];
  const float i1 = l[0] > 0.f ? 1.f / l[0] : (l[0] == 0.f ? 0.f : l[0]), i2 = l[1] > 0.f ? 1.f / l[1] : (l[1] == 0.f ? 0.f : l[1]);
  const long out = ((long)(s.b * a.T + t) * a.H + head) * DV;
#pragma unroll
  for (int j = 0; j < NO; ++j)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      typename Vec<T>::v4 x, y;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float u = o[0][j][4 * r4 + r] * i1, w = o[1][j][4 * r4 + r] * i2;
        x[r] = (T)(u - lam * w);
        y[r] = (T)w;
      }
      const long p = out + 32 * j + 8 * r4 + 4 * h;
      *(typename Vec<T>::v4*)((T*)a.o + p) = x;
      if (a.o2) *(typename Vec<T>::v4*)((T*)a.o2 + p) = y;
    }
  if (a.stat && h == 0) {          // a row that sees nothing: +inf, so that its P comes out 0
#pragma unroll
    for (int c = 0; c < 2; ++c) a.stat[c * a.rows + n] = l[c] == 0.f ? INFINITY : fmaf(m[c], a.c, log2f(l[c]));
  }
}

// joins the splits of a row: a wave per row, lane = value columns
template <typename T, int D>
__global__ __launch_bounds__(64) void da_join(const DaArgs a) {
  constexpr int DV = 2 * D, PER = DV / 64;
  const long n = blockIdx.x;
  const int bh = (int)(n / a.R), r = (int)(n - (long)bh * a.R), b = bh / a.Hkv, hk = bh - b * a.Hkv, t = r / a.G,
            head = hk * a.G + r - t * a.G, lane = threadIdx.x;
  const float* p = a.part + n * (2 * DV + 4);
  const long step = a.rows * (2 * DV + 4);
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[2][PER];
  for (int s = 0; s < a.splits; ++s)
#pragma unroll
    for (int c = 0; c < 2; ++c) m[c] = fmaxf(m[c], p[s * step + 2 * DV + 2 * c]);
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < PER; ++j) o[c][j] = 0.f;
  for (int s = 0; s < a.splits; ++s)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const float ms = p[s * step + 2 * DV + 2 * c];
      const float f = ms == -INFINITY ? 0.f : ms == m[c] ? 1.f : exp2f((ms - m[c]) * a.c);
      l[c] = fmaf(p[s * step + 2 * DV + 2 * c + 1], f, l[c]);
#pragma unroll
      for (int j = 0; j < PER; ++j) o[c][j] = fmaf(p[s * step + c * DV + lane * PER + j], f, o[c][j]);
    }
  const float lam = a.lam[head], i1 = l[0] == 0.f ? 0.f : 1.f / l[0], i2 = l[1] == 0.f ? 0.f : 1.f / l[1];
  const long out = ((long)(b * a.T + t) * a.H + head) * DV + lane * PER;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const float w = o[1][j] * i2;
    ((T*)a.o)[out + j] = (T)(o[0][j] * i1 - lam * w);
    if (a.o2) ((T*)a.o2)[out + j] = (T)w;
  }
  if (a.stat && lane < 2) {
    const float ll = lane ? l[1] : l[0], mm = lane ? m[1] : m[0];
    a.stat[lane * a.rows + n] = ll == 0.f ? INFINITY : fmaf(mm, a.c, log2f(ll));
  }
}

// ------------------------------------------------------------------------------------------------ backward
// Power-of-two scale under which a tile of dS fits fp16 with all its bits: it starts beyond every value and comes down,
// with the accumulators, when a tile would pass 2^15 (bf16 has fp32's range: always 1)
template <typename T>
struct DsScale {
  float f;
  __device__ __forceinline__ DsScale() : f(sizeof(T) == 2 && __is_same(T, _Float16) ? 0x1p100f : 1.f) {}
  // returns the accumulators' factor (1: nothing to do)
  __device__ __forceinline__ float fit(const f32x16& x, const f32x16& y) {
    if constexpr (!__is_same(T, _Float16)) return 1.f;
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fmaxf(fabsf(x[r]), fabsf(y[r])));
    if (!__any(top * f > 32768.f)) return 1.f;
    top = wave_max(top);
    if (!(top < 0x1p120f)) return 1.f;         // infinities and NaN stay what they are
    int e;
    frexpf(top, &e);
    const float nf = ldexpf(1.f, 12 - e), down = nf / f;
    f = nf;
    return down;
  }
};

// dQ: a wave owns 32 rows, walks the keys; also delta_c for the dK / dV kernel and each row's sum of P_2 dP
template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 128 ? 1 : 2) void da_bwd_q(const DaArgs a) {
  constexpr int CH = D / 4, DV = 2 * D, NT = 64 * NW, KQ = D / 16, KV = DV / 16, NQ = D / 32;
  typedef typename Vec<T>::v8 v8;
  __shared__ __align__(16) T ks[32 * DV], vs[32 * DV];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
  const int tile = blockIdx.x % a.tiles, bh = blockIdx.x / a.tiles;
  const Seq s(a, bh);
  const int row = tile * 32 * NW + wave * 32 + (lane & 31), rr = min(row, a.R - 1), t = rr / a.G, head = s.hk * a.G + rr - t * a.G;
  const int lim = s.limit(a, t);
  const int t_last = min((min(tile * 32 * NW + 32 * NW, a.R) - 1) / a.G, s.ql - 1);
  const int k1 = t_last < 0 ? 0 : s.limit(a, t_last);
  const T* qp = (const T*)a.q + s.b * a.q_sb + t * a.q_st + head * a.q_sh;
  const T* gp = (const T*)a.dout + s.b * a.g_sb + t * a.g_st + head * a.g_sh;
  const long orow = ((long)(s.b * a.T + t) * a.H + head) * DV, n = (long)bh * a.R + rr;
  const float lam = a.lam[head];
  v8 qf[2][KQ], gf[KV];
  float d1 = 0.f, d2 = 0.f;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int k = 0; k < KQ; ++k) qf[c][k] = *(const v8*)(qp + c * a.q_sc + 16 * k + 8 * h);
#pragma unroll
  for (int k = 0; k < KV; ++k) {
    gf[k] = *(const v8*)(gp + 16 * k + 8 * h);
    const v8 o = *(const v8*)((const T*)a.o + orow + 16 * k + 8 * h), o2 = *(const v8*)((const T*)a.o2 + orow + 16 * k + 8 * h);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      d1 = fmaf((float)gf[k][i], (float)o[i], d1);
      d2 = fmaf((float)gf[k][i], (float)o2[i], d2);
    }
  }
  d1 += __shfl_xor(d1, 32, 64);
  d2 += __shfl_xor(d2, 32, 64);
  d1 = fmaf(lam, d2, d1);           // O_1 = O + lam O_2
  if (lim == 0) d1 = d2 = 0.f;      // a row that sees nothing gives nothing, whatever its dO holds
  const float l1 = a.stat[n], l2 = a.stat[a.rows + n];
  if (row < a.R && h == 0) {
    a.stat[2 * a.rows + n] = d1;
    a.stat[3 * a.rows + n] = d2;
  }
  const T* kp = (const T*)a.k + s.b * a.k_sb + s.hk * a.k_sh;
  const T* vp = (const T*)a.v + s.b * a.v_sb + s.hk * a.v_sh;
  f32x16 dq[2][NQ];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < NQ; ++j) dq[c][j] = 0.f;
  float dl = 0.f;
  DsScale<T> fit;
  for (int kb = 0; kb < k1; kb += 32) {
    __syncthreads();
    load_tile<T, CH, NT>(ks, min(32, k1 - kb), a.k_sc, [&](int r) { return kp + (long)(kb + r) * a.k_ss; });
    load_tile<T, CH, NT>(vs, min(32, k1 - kb), D, [&](int r) { return vp + (long)(kb + r) * a.v_ss; });
    __syncthreads();
    f32x16 sc[2], dp = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      sc[c] = 0.f;
#pragma unroll
      for (int k = 0; k < KQ; ++k) sc[c] = Mfma<T>::run(frag_row<T, CH>(ks, c * KQ + k, lane), qf[c][k], sc[c]);
    }
#pragma unroll
    for (int k = 0; k < KV; ++k) dp = Mfma<T>::run(frag_row<T, CH>(vs, k, lane), gf[k], dp);
    const int end = lim - kb;
    const bool edge = __any(end < 32);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const bool seen = !edge || c_row(r, h) < end;
      const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[0][r], a.c, -l1)), p2 = __builtin_amdgcn_exp2f(fmaf(sc[1][r], a.c, -l2));
      sc[0][r] = seen ? p1 * (dp[r] - d1) : 0.f;
      sc[1][r] = seen ? p2 * (dp[r] - d2) : 0.f;
      dl += seen ? p2 * dp[r] : 0.f;
    }
    const float down = fit.fit(sc[0], sc[1]);
    if (down != 1.f) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < NQ; ++j) dq[c][j] *= down;
    }
    if constexpr (__is_same(T, _Float16)) {
      sc[0] *= fit.f;
      sc[1] *= fit.f;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const v8 df = pack<T>(sc[c], i);
#pragma unroll
        for (int j = 0; j < NQ; ++j) dq[c][j] = Mfma<T>::run(frag_col<T, CH>(ks, 16 * i, c * D + 32 * j, lane), df, dq[c][j]);
      }
  }
  dl += __shfl_xor(dl, 32, 64);
  if (row >= a.R) return;
  if (h == 0) a.dlrow[n] = dl;
  T* out = (T*)a.dq + ((long)(s.b * a.T + t) * a.H + head) * DV;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float f = a.scale / fit.f * (c ? -lam : 1.f);
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        typename Vec<T>::v4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = (T)(dq[c][j][4 * r4 + r] * f);
        *(typename Vec<T>::v4*)(out + c * D + 32 * j + 8 * r4 + 4 * h) = x;
      }
  }
}

// dK and dV: a wave owns 32 keys, walks the rows that see them
template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, 1) void da_bwd_kv(const DaArgs a) {
  constexpr int CH = D / 4, DV = 2 * D, NT = 64 * NW, KQ = D / 16, KV = DV / 16, NQ = D / 32, NO = DV / 32;
  constexpr bool HALF = __is_same(T, _Float16);
  constexpr float PS = HALF ? 1024.f : 1.f;       // |P_1 - lam P_2| <= max(1, |lam|): keeps fp16's P out of the subnormals
  typedef typename Vec<T>::v8 v8;
  __shared__ __align__(16) T qs[32 * DV], gs[32 * DV];
  __shared__ __align__(16) float st[5][32];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = threadIdx.x >> 6;
  const int tile = blockIdx.x % a.tiles, bh = blockIdx.x / a.tiles;
  const Seq s(a, bh);
  const int kb = tile * 32 * NW, key = kb + wave * 32 + (lane & 31), kr = min(key, a.S - 1);
  const T* kp = (const T*)a.k + s.b * a.k_sb + s.hk * a.k_sh + (long)kr * a.k_ss;
  const T* vp = (const T*)a.v + s.b * a.v_sb + s.hk * a.v_sh + (long)kr * a.v_ss;
  v8 kf[2][KQ], vf[KV];
#pragma unroll
  for (int k = 0; k < KQ; ++k) {
    kf[0][k] = *(const v8*)(kp + 16 * k + 8 * h);
    kf[1][k] = *(const v8*)(kp + a.k_sc + 16 * k + 8 * h);
  }
#pragma unroll
  for (int k = 0; k < KV; ++k) vf[k] = *(const v8*)(vp + 16 * k + 8 * h);
  f32x16 dk[2][NQ], dv[NO];
#pragma unroll
  for (int j = 0; j < NQ; ++j) dk[0][j] = dk[1][j] = 0.f;
#pragma unroll
  for (int j = 0; j < NO; ++j) dv[j] = 0.f;
  DsScale<T> fit;
  // rows that see a key of the block: positions from t0 to the sequence's end
  const int t0 = kb >= s.kl ? s.ql : a.causal ? max(0, kb - (s.kl - s.ql)) : 0;
  const int r1 = s.ql * a.G;
  for (int rb = t0 * a.G / 32 * 32; rb < r1; rb += 32) {
    __syncthreads();
    const int valid = min(32, r1 - rb);
    const auto q_row = [&](int r) {
      const int t = (rb + r) / a.G, head = s.hk * a.G + rb + r - t * a.G;
      return (const T*)a.q + s.b * a.q_sb + t * a.q_st + head * a.q_sh;
    };
    const auto g_row = [&](int r) {
      const int t = (rb + r) / a.G, head = s.hk * a.G + rb + r - t * a.G;
      return (const T*)a.dout + s.b * a.g_sb + t * a.g_st + head * a.g_sh;
    };
    load_tile<T, CH, NT>(qs, valid, a.q_sc, q_row);
    load_tile<T, CH, NT>(gs, valid, D, g_row);
    if (threadIdx.x < 32) {
      const int r = threadIdx.x;
      const long n = (long)bh * a.R + rb + r;
      const bool on = r < valid;
      st[0][r] = on ? a.stat[n] : INFINITY;
      st[1][r] = on ? a.stat[a.rows + n] : INFINITY;
      st[2][r] = on ? a.stat[2 * a.rows + n] : 0.f;
      st[3][r] = on ? a.stat[3 * a.rows + n] : 0.f;
      st[4][r] = on ? a.lam[s.hk * a.G + (rb + r) % a.G] : 0.f;
    }
    __syncthreads();
    f32x16 sc[2], dp = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      sc[c] = 0.f;
#pragma unroll
      for (int k = 0; k < KQ; ++k) sc[c] = Mfma<T>::run(frag_row<T, CH>(qs, c * KQ + k, lane), kf[c][k], sc[c]);
    }
#pragma unroll
    for (int k = 0; k < KV; ++k) dp = Mfma<T>::run(frag_row<T, CH>(gs, k, lane), vf[k], dp);
    // a row below the diagonal of the wave's last key, or a key behind the end, needs the mask
    const bool edge = kb + wave * 32 + 32 > s.kl || (a.causal && rb / a.G + s.kl - s.ql < kb + wave * 32 + 31);
    f32x16 pc;
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x4 l1 = *(const f32x4*)&st[0][8 * r4 + 4 * h], l2 = *(const f32x4*)&st[1][8 * r4 + 4 * h],
                  d1 = *(const f32x4*)&st[2][8 * r4 + 4 * h], d2 = *(const f32x4*)&st[3][8 * r4 + 4 * h],
                  lm = *(const f32x4*)&st[4][8 * r4 + 4 * h];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * r4 + j;
        const bool seen = !edge || key < s.limit(a, (rb + c_row(r, h)) / a.G);
        const float p1 = seen ? __builtin_amdgcn_exp2f(fmaf(sc[0][r], a.c, -l1[j])) : 0.f;
        const float p2 = seen ? lm[j] * __builtin_amdgcn_exp2f(fmaf(sc[1][r], a.c, -l2[j])) : 0.f;
        pc[r] = (p1 - p2) * PS;
        sc[0][r] = seen ? p1 * (dp[r] - d1[j]) : 0.f;
        sc[1][r] = seen ? p2 * (d2[j] - dp[r]) : 0.f;
      }
    }
    const float down = fit.fit(sc[0], sc[1]);
    if (down != 1.f) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < NQ; ++j) dk[c][j] *= down;
    }
    if constexpr (HALF) {
      sc[0] *= fit.f;
      sc[1] *= fit.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const v8 pf = pack<T>(pc, i);
#pragma unroll
      for (int j = 0; j < NO; ++j) dv[j] = Mfma<T>::run(frag_col<T, CH>(gs, 16 * i, 32 * j, lane), pf, dv[j]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const v8 df = pack<T>(sc[c], i);
#pragma unroll
        for (int j = 0; j < NQ; ++j) dk[c][j] = Mfma<T>::run(frag_col<T, CH>(qs, 16 * i, c * D + 32 * j, lane), df, dk[c][j]);
      }
    }
  }
  if (key >= a.S) return;
  const long out = ((long)(s.b * a.S + key) * a.Hkv + s.hk) * DV;
  const float f = a.scale / fit.f;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < NQ; ++j)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        typename Vec<T>::v4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = (T)(dk[c][j][4 * r4 + r] * f);
        *(typename Vec<T>::v4*)((T*)a.dk + out + c * D + 32 * j + 8 * r4 + 4 * h) = x;
      }
#pragma unroll
  for (int j = 0; j < NO; ++j)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      typename Vec<T>::v4 x;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = (T)(dv[j][4 * r4 + r] * (1.f / PS));
      *(typename Vec<T>::v4*)((T*)a.dv + out + 32 * j + 8 * r4 + 4 * h) = x;
    }
}

// dlam of a head: minus the sum over its rows, in fp64, in a fixed order
__global__ __launch_bounds__(1024) void da_dlam(const DaArgs a, float* __restrict__ dlam) {
  __shared__ double red[16];
  const int head = blockIdx.x, hk = head / a.G, g = head - hk * a.G;
  double v = 0.;
  const long total = (long)a.B * a.T;
  for (long i = threadIdx.x; i < total; i += 1024) {
    const long b = i / a.T, t = i - b * a.T;
    v += a.dlrow[(b * a.Hkv + hk) * a.R + t * a.G + g];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.;
    for (int i = 0; i < 16; ++i) sum += red[i];
    dlam[head] = (float)-sum;
  }
}

// ------------------------------------------------------------------------------------------------ host side
// four waves share a key tile where that still gives every compute unit a workgroup; else a wave is one by itself
bool da_wide(long rows_per_bh, long bh) { return cdiv(rows_per_bh, 128) * bh >= 256; }

int da_splits(const ctr_diffattn_t* p) {
  const int R = p->T * (p->H / p->Hkv);
  const long bh = (long)p->B * p->Hkv, blocks = da_wide(R, bh) ? cdiv(R, 128) * bh : cdiv(R, 32) * bh;
  return (int)std::max<long>(1, std::min<long>(1024 / std::max<long>(1, blocks), cdiv(p->S, 128)));
}

int da_check(const ctr_diffattn_t* p, bool bwd) {
  CTR_REQUIRE(p, "null argument");
  CTR_REQUIRE(p->type == TY_BF16 || p->type == TY_F16, "type (1 bf16, 2 fp16)");
  CTR_REQUIRE(p->D == 32 || p->D == 64 || p->D == 128, "map width D in {32, 64, 128}");
  CTR_REQUIRE(p->B >= 0 && p->T >= 0 && p->S >= 0 && p->H >= 1 && p->Hkv >= 1 && p->H % p->Hkv == 0, "sizes");
  CTR_REQUIRE((long)p->T * (p->H / p->Hkv) < (1L << 30) && p->S < (1 << 30), "sizes");
  CTR_REQUIRE((long)p->B * p->Hkv * cdiv((long)p->T * (p->H / p->Hkv), 32) < (1L << 31) &&
                  (long)p->B * p->Hkv * cdiv(p->S, 32) < (1L << 31) && (long)p->B * p->H * p->T < (1L << 31), "sizes");
  CTR_REQUIRE(p->scale > 0.f && std::isfinite(p->scale), "scale > 0");
  if ((long)p->B * p->T == 0 && !(bwd && (long)p->B * p->S > 0)) return 0;
  CTR_REQUIRE(p->lam, "null lam");
  const auto ok = [](const void* q, std::initializer_list<long> st) {
    if (!q || (uintptr_t)q % 16) return false;
    for (long s : st)
      if (s % 8) return false;
    return true;
  };
  CTR_REQUIRE((long)p->B * p->T == 0 || ok(p->q, {p->q_sb, p->q_st, p->q_sh, p->q_sc}), "q: 16-byte aligned rows");
  CTR_REQUIRE((long)p->B * p->S == 0 || ok(p->k, {p->k_sb, p->k_ss, p->k_sh, p->k_sc}), "k: 16-byte aligned rows");
  CTR_REQUIRE((long)p->B * p->S == 0 || ok(p->v, {p->v_sb, p->v_ss, p->v_sh}), "v: 16-byte aligned rows");
  CTR_REQUIRE((long)p->B * p->T == 0 || (p->o && (uintptr_t)p->o % 16 == 0 && (uintptr_t)p->o2 % 16 == 0), "output");
  return 0;
}

DaArgs da_args(const ctr_diffattn_t* p) {
  DaArgs a = {};
  a.q = p->q; a.k = p->k; a.v = p->v; a.lam = p->lam;
  a.o = p->o; a.o2 = p->o2; a.stat = p->stat;
  a.q_lens = p->q_lens; a.kv_lens = p->kv_lens;
  a.q_sb = p->q_sb; a.q_st = p->q_st; a.q_sh = p->q_sh; a.q_sc = p->q_sc;
  a.k_sb = p->k_sb; a.k_ss = p->k_ss; a.k_sh = p->k_sh; a.k_sc = p->k_sc;
  a.v_sb = p->v_sb; a.v_ss = p->v_ss; a.v_sh = p->v_sh;
  a.scale = p->scale;
  a.c = p->scale * 1.44269504088896341f;
  a.B = p->B; a.T = p->T; a.S = p->S; a.H = p->H; a.Hkv = p->Hkv; a.G = p->H / p->Hkv; a.R = p->T * a.G;
  a.rows = (long)p->B * p->Hkv * a.R;
  a.causal = p->causal;
  a.splits = 1;
  return a;
}

template <typename T, int D>
int da_run_fwd(DaArgs a, hipStream_t s) {
  const long bh = (long)a.B * a.Hkv;
  const bool wide = da_wide(a.R, bh);
  a.tiles = cdiv(a.R, wide ? 128 : 32);
  const long blocks = a.tiles * bh * a.splits;
  if (wide) da_fwd<T, D, 4><<<(unsigned)blocks, 256, 0, s>>>(a);
  else da_fwd<T, D, 1><<<(unsigned)blocks, 64, 0, s>>>(a);
  if (a.splits > 1) da_join<T, D><<<(unsigned)a.rows, 64, 0, s>>>(a);
  return check_launch("diffattn_fwd");
}

template <typename T, int D>
int da_run_bwd(DaArgs a, float* dlam, hipStream_t s) {
  const long bh = (long)a.B * a.Hkv;
  const bool wq = da_wide(a.R, bh), wk = da_wide(a.S, bh);
  if (a.rows > 0) {
    a.tiles = cdiv(a.R, wq ? 128 : 32);
    if (wq) da_bwd_q<T, D, 4><<<(unsigned)(a.tiles * bh), 256, 0, s>>>(a);
    else da_bwd_q<T, D, 1><<<(unsigned)(a.tiles * bh), 64, 0, s>>>(a);
  }
  if (bh * a.S > 0) {
    a.tiles = cdiv(a.S, wk ? 128 : 32);
    if (wk) da_bwd_kv<T, D, 4><<<(unsigned)(a.tiles * bh), 256, 0, s>>>(a);
    else da_bwd_kv<T, D, 1><<<(unsigned)(a.tiles * bh), 64, 0, s>>>(a);
  }
  da_dlam<<<a.H, 1024, 0, s>>>(a, dlam);
  return check_launch("diffattn_bwd");
}

}  // namespace
}  // namespace ctr

using namespace ctr;

#define DA_TYPES(CALL)                                            \
  if (p->type == TY_BF16) {                                       \
    if (p->D == 32) return CALL(__bf16, 32);                      \
    if (p->D == 64) return CALL(__bf16, 64);                      \
    return CALL(__bf16, 128);                                     \
  }                                                               \
  if (p->D == 32) return CALL(_Float16, 32);                      \
  if (p->D == 64) return CALL(_Float16, 64);                      \
  return CALL(_Float16, 128)

extern "C" size_t ctr_diffattn_fwd_ws_size(const ctr_diffattn_t* p) {
  if (!p || p->B <= 0 || p->T <= 0 || p->S <= 0 || p->Hkv <= 0 || p->H < p->Hkv) return 0;
  const int splits = da_splits(p);
  return splits > 1 ? (size_t)splits * p->B * p->H * p->T * (4 * p->D + 4) * sizeof(float) : 0;
}

extern "C" int ctr_diffattn_fwd(const ctr_diffattn_t* p, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = da_check(p, false)) return rc;
  if ((long)p->B * p->T == 0) return 0;
  CTR_REQUIRE(ws_bytes >= ctr_diffattn_fwd_ws_size(p), "workspace too small");
  DaArgs a = da_args(p);
  a.splits = p->S > 0 ? da_splits(p) : 1;
  a.part = (float*)ws;
#define DA_CALL(T, D) da_run_fwd<T, D>(a, (hipStream_t)stream)
  DA_TYPES(DA_CALL);
#undef DA_CALL
}

extern "C" size_t ctr_diffattn_bwd_ws_size(const ctr_diffattn_t* p) {
  return p && p->B > 0 && p->T > 0 ? (size_t)p->B * p->T * p->H * sizeof(float) : 0;
}

extern "C" int ctr_diffattn_bwd(const ctr_diffattn_t* p, const void* dout, long g_sb, long g_st, long g_sh, void* dq, void* dk,
                                void* dv, float* dlam, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = da_check(p, true)) return rc;
  CTR_REQUIRE(dlam, "null dlam");
  const bool q_on = (long)p->B * p->T > 0, k_on = (long)p->B * p->S > 0;
  CTR_REQUIRE(!q_on || (p->o2 && p->stat && dq && dout), "null operand");
  CTR_REQUIRE(!q_on || ((uintptr_t)dout % 16 == 0 && g_sb % 8 == 0 && g_st % 8 == 0 && g_sh % 8 == 0), "dout: 16-byte aligned rows");
  CTR_REQUIRE(!k_on || (dk && dv), "null operand");
  CTR_REQUIRE(((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) % 16 == 0, "gradients: 16-byte aligned");
  CTR_REQUIRE(ws_bytes >= ctr_diffattn_bwd_ws_size(p), "workspace too small");
  DaArgs a = da_args(p);
  a.dout = dout;
  a.g_sb = g_sb;
  a.g_st = g_st;
  a.g_sh = g_sh;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.dlrow = (float*)ws;
#define DA_CALL(T, D) da_run_bwd<T, D>(a, dlam, (hipStream_t)stream)
  DA_TYPES(DA_CALL);
#undef DA_CALL
}
