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
// factor.  K, V (Q, dO) tiles of 32 rows go to LDS by buffer loads that write it directly, the next tile's under this
// tile's products, one barrier a tile; rows behind the end are out of the load's range and come as zeros.  A tile is
// read once along a row (ds_read_b128) and once down the columns (the LDS transpose read); the 16-byte chunks of a row
// are XORed with the row, in the global address, so that both reads are free of bank conflicts.
// Softmax in base 2 with one running maximum per map, taken up only when a score passes it by 2^8 (fp16: 2); statistics,
// accumulators and dlam's sum are fp32.
// Roundings to 16 bits.  The forward's P enter the product with V as two 16-bit terms each (the value and what that leaves
// out): O is a difference, and where the maps agree one rounding of either would be larger than the result's own.  fp16's are
// scaled up by 2^14, so that a probability keeps both terms down to 2^-17 of its row's largest, one down to 2^-28, and is held to
// 2^-39 of it below (unscaled, many keys 15 nats below one of no value lost 3 % of the output, at 17.5 nats all of it).  In
// the backward P_1 - lam P_2 and dS are rounded once, in fp16 under a power of two that follows their size, a row's own in dQ and
// a key's own in dK and dV.  What
// the roundings of O and of P_2 V left out is kept too: deltas from the rounded ones would add as much again to dQ of short rows.
// delta_1 is of O + lam P_2 V, so its error grows with lam: |lam| 2^-17 (fp16 2^-23) of |dO| |P_2 V|, below dS's own rounding up to
// |lam| of a few hundred.
#include <algorithm>
#include <type_traits>

#include "ctr_hip.h"
#include "vec16.h"

namespace ctr {
namespace {

struct DaArgs {
  const void *q, *k, *v, *dout;
  const float* lam;
  void *o, *o2, *ol;             // (B, T, H, 2 D); kept for the backward (may be null): o2 = P_2 V and, `plane` elements
                                 // on, what its rounding left out; ol = what o's rounding left out (rest())
  float* stat;                   // 2 planes of rows: log2 sums of the maps
  void *dq, *dk, *dv;
  float* dlam;
  float* part;                   // forward, split keys: partial results; backward: row statistics (RS_*)
  float* kvpart;                 // backward, split rows: partial dK, dV
  const int *q_lens, *kv_lens;
  long q_sb, q_st, q_sh, q_sc, k_sb, k_ss, k_sh, k_sc, v_sb, v_ss, v_sh, g_sb, g_st, g_sh;
  long rows, plane;              // B Hkv R; B T H 2 D
  float c, scale;                // scale log2(e), scale
  int B, T, S, H, Hkv, G, R, causal, splits, tiles, tiles32;
};

// Row statistics of the backward, written by the dQ kernel for the dK / dV kernel: a tile of 32 packed rows is 8 lines
// of 32 words, one 1 KB load
enum { RS_L1, RS_L2, RS_D1, RS_LD2, RS_LAM, RS_LIM, RS_DL, RS_LINES = 8 };      // RS_LD2: lam delta_2

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

// The forward's exponentials are 2^(UP + s - m) with m at most LAG bits below the largest score: fp16 takes them as near to the top
// of its range as they go (2^15), bf16 has fp32's range.  The factor cancels in the quotient and in the joins.  The smaller LAG takes
// the maximum up more often: 1531 rows on 5627 keys, fp16, D = 128, 314 us unscaled (LAG 8), 317 at 11 + 4, 321 at 13 + 2, 326 so.
template <typename T> struct Prob { static constexpr float UP = 0.f, LAG = 8.f; };
template <> struct Prob<_Float16> { static constexpr float UP = 14.f, LAG = 1.f; };

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// C layout of a 32x32 tile: register r of lane l holds row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32
__device__ __forceinline__ int c_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// A tile of 32 rows of W elements in LDS, CH = W / 8 chunks of 16 bytes a row: chunk c of a row stands at chunk
// c ^ turn(row).  Sixteen consecutive rows' equal chunks, and four consecutive rows' four-chunk groups, then cover the
// 64 banks once.
template <int CH>
__device__ __forceinline__ int turn(int row) {
  if constexpr (CH >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
  else if constexpr (CH == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else return (row >> 2) & 3;
}
// 32 rows x 16 k, k contiguous along a row: lane l has row l % 32, k = 16 kk + 8 (l / 32) + 0..7
template <typename T, int W>
__device__ __forceinline__ typename Vec<T>::v8 frag_row(const T* s, int kk, int lane) {
  const int row = lane & 31;
  return *(const typename Vec<T>::v8*)(s + row * W + ((2 * kk + (lane >> 5)) ^ turn<W / 8>(row)) * 8);
}
// Transposed reads.  The 32 rows of a tile as k x 32 columns: for the first and second 16 rows, lane l gets of column l % 32
// the rows 4 (l / 32) + 0..3 and 8 + 4 (l / 32) + 0..3 -- the order in which a C tile's registers 8 i .. 8 i + 7 hold the
// rows of its i-th half.  A group of 16 lanes takes 4 rows of 16 columns: lane i of it the address of row i / 4,
// columns 4 (i % 4), and it gets column i.  `col_base` is the lane's address for the columns from 0; columns 32 j on are
// at col_base ^ (j << 6), since a panel's chunks are XORed and its rows start at multiples of their power-of-two size; 8 rows
// on the turn differs by 2, 16 rows on it is the same.
template <typename T, int W>
__device__ __forceinline__ uint32_t col_base(const T* s, int lane) {
  const int row = 4 * (lane >> 5) + ((lane & 15) >> 2), c = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)(s + row * W + ((c >> 3) ^ turn<W / 8>(row)) * 8 + (c & 4));
}
// columns 32 j .. of the panel's first (i = 0) or second 16 rows
template <typename T, int W>
__device__ __forceinline__ typename Vec<T>::v8 frag_col(uint32_t base, int i, int j) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const uint32_t p = (base ^ (j << 6)) + i * 32 * W, q = ((base ^ (j << 6)) + 16 * W ^ 32) + i * 32 * W;
  const auto u = __builtin_bit_cast(typename Vec<T>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p));
  const auto v = __builtin_bit_cast(typename Vec<T>::v4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)q));
  return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
}
// What the rounding of a kept output left out, x - T(x), in T again: fp16's is kept 2^11 times as large, since that of a value below
// 2^-13 would fall under the type's smallest step.
template <typename T> constexpr float REST = __is_same(T, _Float16) ? 2048.f : 1.f;
template <typename T>
__device__ __forceinline__ float rest(float x) { return (x - (float)(T)x) * REST<T>; }
// registers 8 i .. 8 i + 7 of a C tile as an operand, and what the rounding left out
template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 pack(const f32x16& v, int i) {
  f32x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = v[8 * i + j];
  return __builtin_convertvector(o, typename Vec<T>::v8);
}
template <typename T>
__device__ __forceinline__ typename Vec<T>::v8 pack_rest(const f32x16& v, typename Vec<T>::v8 hi, int i) {
  f32x8 o;
  if constexpr (__is_same(T, __bf16)) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 w = __builtin_bit_cast(u32x4, hi);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[2 * j] = v[8 * i + 2 * j] - __builtin_bit_cast(float, w[j] << 16);
      o[2 * j + 1] = v[8 * i + 2 * j + 1] - __builtin_bit_cast(float, w[j] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = v[8 * i + j] - (float)hi[j];
  }
  return __builtin_convertvector(o, typename Vec<T>::v8);
}

// Direct loads of a tile of 32 rows to LDS: two panels of width D (the maps) and one of 2 D (values, or dO), as four
// roles dealt over the waves: panel 0, panel 1, the upper and the lower 16 rows of panel 2.  Each role is PER loads of
// 64 lanes x 16 bytes, whose LDS places are consecutive.
template <typename T, int D, int NW>
struct Stage {
  static constexpr int ROLES = NW >= 4 ? 1 : 4 / NW, SHARE = NW > 4 ? NW / 4 : 1;      // roles of a wave, waves of a role
  static constexpr int PER = D / 16 / SHARE, TILE = 32 * 4 * D;      // a wave's loads for a role; elements of the three panels
  int row[ROLES], byte[ROLES][PER];      // the lane's row for load 0 of its roles, and its byte in the row for each load
  static __device__ __forceinline__ int role(int i, int wave) { return SHARE > 1 ? wave & 3 : i * NW + wave; }
  // where a wave's loads for a role begin in LDS (elements)
  static __device__ __forceinline__ int place(int role, int wave) {
    return (role < 2 ? role * 32 * D : 64 * D + (role - 2) * 32 * D) + (SHARE > 1 ? (wave >> 2) * PER * 512 : 0);
  }
  static __device__ __forceinline__ int step(int role) { return role < 2 ? 512 / D : 256 / D; }      // rows from load to load
  __device__ __forceinline__ Stage(int wave, int lane) {
#pragma unroll
    for (int i = 0; i < ROLES; ++i) {
      const int ro = role(i, wave);
      const bool map = ro < 2;
      row[i] = (map ? lane / (D / 8) : lane / (D / 4) + (ro - 2) * 16) + (SHARE > 1 ? (wave >> 2) * PER * step(ro) : 0);
      const int c = map ? lane % (D / 8) : lane % (D / 4);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int r = row[i] + j * step(ro);
        byte[i][j] = (c ^ (map ? turn<D / 8>(r) : turn<D / 4>(r))) * 16;
      }
    }
  }
};

// 64 lanes x 16 bytes from r at off to consecutive LDS places.  Nothing comes back in registers, and tile_ready() waits: as a
// builtin it would have the compiler wait for it before any transpose read, whose address it does not see.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"      // m0 is a reserved register; it is named because it changes
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, const void* lds, uint32_t off) {
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(off), "s"(r) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ __amdgpu_buffer_rsrc_t open_range(const void* p) { return buf_rsrc(p, 0x7ffffff0u); }

// every wave's loads of the next tile are in LDS and every wave is done with the last one
__device__ __forceinline__ void tile_ready() {
  asm volatile("" ::: "memory");           // the builtins order nothing for the compiler
  __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// keys [kb, kb + 32) of K_1, K_2, V to one buffer; rows from `valid` on come as zeros
template <typename T, int D, int NW>
__device__ __forceinline__ void stage_keys(const DaArgs& a, const Stage<T, D, NW>& p, const T* kp, const T* vp, int kb, int valid,
                                           T* buf, int wave) {
  typedef Stage<T, D, NW> St;
#pragma unroll
  for (int i = 0; i < St::ROLES; ++i) {
    const int role = St::role(i, wave);
    const T* base = role < 2 ? kp + (long)kb * a.k_ss + (role ? a.k_sc : 0) : vp + (long)kb * a.v_ss;
    const int stride = (int)((role < 2 ? a.k_ss : a.v_ss) * sizeof(T)), step = St::step(role);
    const auto rs = open_range(base);
    T* dst = buf + St::place(role, wave);
    int row = p.row[i], off = row * stride;
    if (valid >= 32) {
#pragma unroll
      for (int j = 0; j < St::PER; ++j, off += step * stride) dma16(rs, dst + j * 512, off + p.byte[i][j]);
    } else {
#pragma unroll
      for (int j = 0; j < St::PER; ++j, off += step * stride, row += step)
        dma16(rs, dst + j * 512, row < valid ? off + p.byte[i][j] : BUF_OOB);
    }
  }
}

// every wave's LDS writes before it are seen after it; loads in flight stay in flight
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);      // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
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
// A pair of waves owns 32 rows, one of them each map: nothing but the value tile's reads is done twice, a wave's
// accumulators are half as many, and three (D = 64) or two (D = 128) waves share a SIMD, so that one's exponentials run
// under another's products.  RG pairs a workgroup.  Two 16-bit terms of P make 20 D operations a pair of the 12 D that the
// definition has; the exponentials and their packing hide under the products only in part: of a compute unit's busy cycles the
// matrix unit works in 59 % and the VALU issues in 68 % at D = 64, 52 and 37 % at D = 128.  Measured: causal 2 x 4096, 16 over 4
// heads, D = 64, bf16: 330 - 339 us, 0.61 PFLOP/s of the definition's, 1.01 issued; 1531 rows on 5627 keys, 16 over 8 heads,
// D = 128, fp16: 326 us, 0.56 and 0.94 PFLOP/s.  One token on 131072 keys, 8 over 2 heads, D = 128, bf16: 42 us, 6.4 TB/s.
// Workgroups: (batch, key head) fastest, so that the eight XCDs, which take workgroups in turn, each keep few heads'
// keys in their L2; then the splits, then the row tiles, the causally longest first.
template <typename T, int D, int RG>
__global__ __launch_bounds__(128 * RG, D == 128 ? (RG == 2 ? 2 : 1) : 3) void da_fwd(const DaArgs a) {
  constexpr int DV = 2 * D, KQ = D / 16, NO = DV / 32, NW = 2 * RG, TILE = Stage<T, D, NW>::TILE;
  constexpr int JG = NO < 4 ? NO : 4;
  static_assert(RG * DV * 32 * sizeof(float) <= 2 * TILE * sizeof(T), "the maps meet in the tiles' place");
  typedef typename Vec<T>::v8 v8;
  __shared__ __align__(1024) T tiles[2][TILE];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nbh = a.B * a.Hkv;
  const Stage<T, D, NW> plan(wave, lane);
  const int map = wave & 1, pair = wave >> 1;
  int id = blockIdx.x;
  const int bh = id % nbh;
  id /= nbh;
  const int sp = id % a.splits, tile = a.tiles - 1 - id / a.splits;
  const Seq s(a, bh);
  const int row = tile * 32 * RG + pair * 32 + (lane & 31), rr = min(row, a.R - 1), t = rr / a.G, head = s.hk * a.G + rr - t * a.G;
  const int lim = s.limit(a, t);
  // the keys of the block: those its last row sees, and of them this split's share
  const int t_last = min((min(tile * 32 * RG + 32 * RG, a.R) - 1) / a.G, s.ql - 1);
  int k0 = 0, k1 = t_last < 0 ? 0 : s.limit(a, t_last);
  if (a.splits > 1) {
    const int per = (((k1 + a.splits - 1) / a.splits) + 31) / 32 * 32;
    k0 = min(k1, sp * per);
    k1 = min(k1, k0 + per);
  }
  const T* kp = (const T*)a.k + s.b * a.k_sb + s.hk * a.k_sh;
  const T* vp = (const T*)a.v + s.b * a.v_sb + s.hk * a.v_sh;
  if (k0 < k1) stage_keys<T, D, NW>(a, plan, kp, vp, k0, k1 - k0, tiles[0], wave);
  const T* qp = (const T*)a.q + s.b * a.q_sb + t * a.q_st + head * a.q_sh + map * a.q_sc;
  v8 qf[KQ];
#pragma unroll
  for (int k = 0; k < KQ; ++k) qf[k] = *(const v8*)(qp + 16 * k + 8 * h);
  f32x16 o[NO];
#pragma unroll
  for (int j = 0; j < NO; ++j) o[j] = 0.f;
  float m = -INFINITY, l = 0.f;
  const uint32_t vcol = col_base<T, DV>(tiles[0] + 64 * D, lane);
  int cur = 0;
  for (int kb = k0; kb < k1; kb += 32, cur ^= 1) {
    tile_ready();
    if (kb + 32 < k1) stage_keys<T, D, NW>(a, plan, kp, vp, kb + 32, k1 - kb - 32, tiles[cur ^ 1], wave);
    const T* ks = tiles[cur] + map * 32 * D;
    f32x16 sc = 0.f;
#pragma unroll
    for (int k = 0; k < KQ; ++k) sc = Mfma<T>::run(frag_row<T, D>(ks, k, lane), qf[k], sc);
    const int end = min(lim, k1) - kb;
    if (__any(end < 32)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) sc[r] = c_row(r, h) < end ? sc[r] : -INFINITY;
    }
    float top = sc[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, sc[r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any((top - m) * a.c > Prob<T>::LAG)) {        // also the first keys, from -inf (-inf - -inf is NaN: no)
      const float mn = fmaxf(m, top), f = m == mn ? 1.f : exp2f((m - mn) * a.c);
      l *= f;
#pragma unroll
      for (int j = 0; j < NO; ++j) o[j] *= f;
      m = mn;
    }
    const float base = m == -INFINITY ? 0.f : fmaf(m, a.c, -Prob<T>::UP);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      sc[r] = __builtin_amdgcn_exp2f(fmaf(sc[r], a.c, -base));
      l += sc[r];
    }
    v8 pf[2], pr[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      pf[i] = pack<T>(sc, i);
      pr[i] = pack_rest<T>(sc, pf[i], i);
    }
    const uint32_t vc = vcol + cur * TILE * sizeof(T);
#pragma unroll
    for (int j0 = 0; j0 < NO; j0 += JG)
#pragma unroll
      for (int i = 0; i < 2; ++i) {        // no two products in a row into one accumulator
        v8 vf[JG];
#pragma unroll
        for (int j = 0; j < JG; ++j) vf[j] = frag_col<T, DV>(vc, i, j0 + j);
#pragma unroll
        for (int j = 0; j < JG; ++j) o[j0 + j] = Mfma<T>::run(vf[j], pr[i], o[j0 + j]);
#pragma unroll
        for (int j = 0; j < JG; ++j) o[j0 + j] = Mfma<T>::run(vf[j], pf[i], o[j0 + j]);
      }
  }
  l += __shfl_xor(l, 32, 64);
  const long n = (long)bh * a.R + row;
  if (a.splits > 1) {
    if (row >= a.R) return;
    float* p = a.part + ((long)sp * a.rows + n) * (2 * DV + 4);
#pragma unroll
    for (int j = 0; j < NO; ++j)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = o[j][4 * r4 + r];
        *(f32x4*)(p + map * DV + 32 * j + 8 * r4 + 4 * h) = x;
      }
    if (h == 0) {
      p[2 * DV + 2 * map] = m;
      p[2 * DV + 2 * map + 1] = l;
    }
    return;
  }
  const bool none = l == 0.f;                  // sees no key: zeros, whatever the keys' values are
  const float inv = none ? 0.f : 1.f / l;
  if (a.stat && h == 0 && row < a.R)           // a row that sees nothing: +inf, so that its P comes out 0
    a.stat[map * a.rows + n] = none ? INFINITY : fmaf(m, a.c, log2f(l) - Prob<T>::UP);
  // the second map's part goes through LDS to the first map's wave (each path by itself: a value that both change would be
  // copied register by register)
  float* meet = (float*)&tiles[0][0] + pair * DV * 32 + (lane & 31);
  const long at = ((long)(s.b * a.T + t) * a.H + head) * DV;
  __syncthreads();
  if (map) {
#pragma unroll
    for (int j = 0; j < NO; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) meet[(32 * j + c_row(r, h)) * 32] = none ? 0.f : o[j][r] * inv;
  }
  __syncthreads();
  if (row >= a.R) return;
  const auto put = [&](T* out, int j, int r4, const f32x4& v) {
    *(typename Vec<T>::v4*)(out + 32 * j + 8 * r4 + 4 * h) = __builtin_convertvector(v, typename Vec<T>::v4);
  };
  if (map) {
    if (!a.o2) return;
#pragma unroll
    for (int j = 0; j < NO; ++j)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = none ? 0.f : o[j][4 * r4 + r] * inv;
        put((T*)a.o2 + at, j, r4, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = rest<T>(x[r]);
        put((T*)a.o2 + a.plane + at, j, r4, x);
      }
  } else {
    const float lam = a.lam[head];
#pragma unroll
    for (int j = 0; j < NO; ++j) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = none ? 0.f : o[j][4 * r4 + r] * inv - lam * meet[(32 * j + c_row(4 * r4 + r, h)) * 32];
        put((T*)a.o + at, j, r4, x);
        if (a.ol) {
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = rest<T>(x[r]);
          put((T*)a.ol + at, j, r4, x);
        }
      }
      __builtin_amdgcn_sched_barrier(0);       // one tile's reads at a time: the accumulators fill the registers
    }
  }
}

// joins the splits of a row: a workgroup takes 32 value columns of it, GR threads a column the splits in turn; the splits'
// factors are formed once, in LDS
// (a thread each: at most 32 GR splits)
template <typename T, int D, int GR>
__global__ __launch_bounds__(32 * GR) void da_join(const DaArgs a) {
  constexpr int DV = 2 * D, NW = GR / 2;
  __shared__ float fac[2][32 * GR], sh[2][GR][33], red[4][NW];
  const long n = blockIdx.x;
  const int bh = (int)(n / a.R), r = (int)(n - (long)bh * a.R), b = bh / a.Hkv, hk = bh - b * a.Hkv, t = r / a.G,
            head = hk * a.G + r - t * a.G, col = threadIdx.x & 31, grp = threadIdx.x >> 5, c0 = blockIdx.y * 32 + col;
  const float* p = a.part + n * (2 * DV + 4);
  const long step = a.rows * (2 * DV + 4);
  const int s0 = threadIdx.x;                      
  f32x4 ml = {-INFINITY, 0.f, -INFINITY, 0.f};
  if (s0 < a.splits) ml = *(const f32x4*)(p + s0 * step + 2 * DV);
  float m[2], l[2];
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    m[c] = wave_max(ml[2 * c]);
    if ((threadIdx.x & 63) == 0) red[c][threadIdx.x >> 6] = m[c];
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 2; ++c) {
#pragma unroll
    for (int w = 0; w < NW; ++w) m[c] = fmaxf(m[c], red[c][w]);
    const float f = ml[2 * c] == -INFINITY ? 0.f : ml[2 * c] == m[c] ? 1.f : exp2f((ml[2 * c] - m[c]) * a.c);
    if (s0 < a.splits) fac[c][s0] = f;
    l[c] = wave_sum(ml[2 * c + 1] * f);
    if ((threadIdx.x & 63) == 0) red[2 + c][threadIdx.x >> 6] = l[c];
  }
  __syncthreads();
  float o[2] = {0.f, 0.f};
#pragma unroll 8
  for (int s = grp; s < a.splits; s += GR) {
    o[0] = fmaf(p[s * step + c0], fac[0][s], o[0]);
    o[1] = fmaf(p[s * step + DV + c0], fac[1][s], o[1]);
  }
  sh[0][grp][col] = o[0];
  sh[1][grp][col] = o[1];
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    l[c] = o[c] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) l[c] += red[2 + c][w];
#pragma unroll
    for (int g = 0; g < GR; ++g) o[c] += sh[c][g][col];
  }
  const float w = l[1] == 0.f ? 0.f : o[1] / l[1];
  const long out = ((long)(b * a.T + t) * a.H + head) * DV + c0;
  const float u = (l[0] == 0.f ? 0.f : o[0] / l[0]) - a.lam[head] * w;
  ((T*)a.o)[out] = (T)u;
  if (a.o2) {
    ((T*)a.o2)[out] = (T)w;
    ((T*)a.o2)[a.plane + out] = (T)rest<T>(w);
    ((T*)a.ol)[out] = (T)rest<T>(u);
  }
  if (a.stat && blockIdx.y == 0 && col < 2) {
    const float ll = col ? l[1] : l[0], mm = col ? m[1] : m[0];
    a.stat[col * a.rows + n] = ll == 0.f ? INFINITY : fmaf(mm, a.c, log2f(ll) - Prob<T>::UP);
  }
}

// ------------------------------------------------------------------------------------------------ backward
// Power-of-two scale under which a column (a row of dQ, a key of dK or dV) fits fp16 with all its bits: it starts beyond every value and
// comes down, with the column's accumulators, when one would pass 2^15; values down to 2^-25 of the column's largest keep 11
// bits, and those below are held to 2^-36 of it.  (Up to 2^15 at once it would be 2^-39, but each small rise is then a new scale:
// backward at 2 x 4096 causal, 16 over 4 heads, D = 64: 872 us against 843; 4 x 2048, 8 heads, D = 32: 192 against 182.)
// A lane's own: under one scale for the tile a column far below its neighbours lost its bits, and an infinity in one reached all.
// (bf16 has fp32's range: always 1)
template <typename T>
struct ColScale {
  static constexpr bool ON = __is_same(T, _Float16);
  float f;
  __device__ __forceinline__ ColScale() : f(ON ? 0x1p100f : 1.f) {}
  // top: the largest size among the lane's values; returns the accumulators' factor (1: nothing to do).  All lanes take part.
  __device__ __forceinline__ float fit(float top) {
    if (!ON || !__any(top * f > 32768.f)) return 1.f;
    top = fmaxf(top, __shfl_xor(top, 32, 64));           // the column's other half
    if (!(top * f > 32768.f) || !(top < INFINITY)) return 1.f;      // infinities and NaN stay what they are
    int e;
    frexpf(top, &e);
    const float nf = ldexpf(1.f, 12 - e), down = nf / f;      // top then lies in [2^11, 2^12)
    f = nf;
    return down;
  }
};
template <typename T>
__device__ __forceinline__ float top_of(const f32x16& x, float top = 0.f) {
  if constexpr (ColScale<T>::ON) {
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(x[r]));
  }
  return top;
}

// acc[j] += (columns 32 j .. of a panel of width W)^T x
template <typename T, int W, int N>
__device__ __forceinline__ void add_cols(uint32_t base, const typename Vec<T>::v8 (&x)[2], f32x16 (&acc)[N]) {
  static_assert(N == W / 32, "panel");
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] = Mfma<T>::run(frag_col<T, W>(base, i, j), x[i], acc[j]);
}

// dQ: a wave owns 32 rows, walks the keys; also the rows' statistics for the dK / dV kernel.  Bound by the products and the
// exponentials in turn, two waves a SIMD (D <= 64): 253 - 265 us at 2 x 4096 causal, 16 over 4 heads, D = 64, bf16 (matrix unit
// 41 %, VALU 59 % of the busy cycles).
template <typename T, int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 128 ? 1 : 2) void da_bwd_q(const DaArgs a) {
  constexpr int DV = 2 * D, KQ = D / 16, KV = DV / 16, NQ = D / 32, TILE = Stage<T, D, NW>::TILE;
  typedef typename Vec<T>::v8 v8;
  __shared__ __align__(1024) T tiles[2][TILE];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nbh = a.B * a.Hkv;
  const Stage<T, D, NW> plan(wave, lane);
  const int bh = blockIdx.x % nbh, tile = a.tiles - 1 - blockIdx.x / nbh;
  const Seq s(a, bh);
  const int row = tile * 32 * NW + wave * 32 + (lane & 31), rr = min(row, a.R - 1), t = rr / a.G, head = s.hk * a.G + rr - t * a.G;
  const int lim = s.limit(a, t);
  const int t_last = min((min(tile * 32 * NW + 32 * NW, a.R) - 1) / a.G, s.ql - 1);
  const int k1 = t_last < 0 ? 0 : s.limit(a, t_last);
  const T* kp = (const T*)a.k + s.b * a.k_sb + s.hk * a.k_sh;
  const T* vp = (const T*)a.v + s.b * a.v_sb + s.hk * a.v_sh;
  if (0 < k1) stage_keys<T, D, NW>(a, plan, kp, vp, 0, k1, tiles[0], wave);
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
    const long at = orow + 16 * k + 8 * h;
    const v8 o = *(const v8*)((const T*)a.o + at), o2 = *(const v8*)((const T*)a.o2 + at), ol = *(const v8*)((const T*)a.ol + at),
             o2l = *(const v8*)((const T*)a.o2 + a.plane + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      d1 = fmaf((float)gf[k][i], fmaf((float)ol[i], 1.f / REST<T>, (float)o[i]), d1);
      d2 = fmaf((float)gf[k][i], fmaf((float)o2l[i], 1.f / REST<T>, (float)o2[i]), d2);
    }
  }
  d1 += __shfl_xor(d1, 32, 64);
  d2 += __shfl_xor(d2, 32, 64);
  d1 = fmaf(lam, d2, d1);           // O_1 = O + lam O_2
  if (lim == 0) d1 = d2 = 0.f;      // a row that sees nothing gives nothing, whatever its dO holds
  const float l1 = a.stat[n], l2 = a.stat[a.rows + n];
  f32x16 dq[2][NQ];
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int j = 0; j < NQ; ++j) dq[c][j] = 0.f;
  float dl = 0.f;
  ColScale<T> fit;
  const uint32_t kcol = col_base<T, D>(tiles[0], lane);
  int cur = 0;
  for (int kb = 0; kb < k1; kb += 32, cur ^= 1) {
    tile_ready();
    if (kb + 32 < k1) stage_keys<T, D, NW>(a, plan, kp, vp, kb + 32, k1 - kb - 32, tiles[cur ^ 1], wave);
    const T* ks = tiles[cur];
    const T* vs = ks + 64 * D;
    f32x16 sc[2], dp = 0.f;
    sc[0] = sc[1] = 0.f;
#pragma unroll
    for (int k = 0; k < KQ; ++k) {         // three accumulators in turn
      sc[0] = Mfma<T>::run(frag_row<T, D>(ks, k, lane), qf[0][k], sc[0]);
      dp = Mfma<T>::run(frag_row<T, DV>(vs, 2 * k, lane), gf[2 * k], dp);
      sc[1] = Mfma<T>::run(frag_row<T, D>(ks + 32 * D, k, lane), qf[1][k], sc[1]);
      dp = Mfma<T>::run(frag_row<T, DV>(vs, 2 * k + 1, lane), gf[2 * k + 1], dp);
    }
    const int end = lim - kb;
    const bool edge = __any(end < 32);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float p1 = __builtin_amdgcn_exp2f(fmaf(sc[0][r], a.c, -l1)), p2 = __builtin_amdgcn_exp2f(fmaf(sc[1][r], a.c, -l2));
      sc[0][r] = p1 * (dp[r] - d1);
      sc[1][r] = p2 * (dp[r] - d2);
      dp[r] *= p2;
    }
    if (edge) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const bool seen = c_row(r, h) < end;
        sc[0][r] = seen ? sc[0][r] : 0.f;
        sc[1][r] = seen ? sc[1][r] : 0.f;
        dp[r] = seen ? dp[r] : 0.f;
      }
    }
    float dl_tile = 0.f;              // a tile's sum by itself: long rows then add few numbers
#pragma unroll
    for (int r = 0; r < 16; ++r) dl_tile += dp[r];
    dl += dl_tile;
    const float down = fit.fit(top_of<T>(sc[1], top_of<T>(sc[0])));
    if (__any(down != 1.f)) {
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int j = 0; j < NQ; ++j) dq[c][j] *= down;
    }
    if constexpr (ColScale<T>::ON) {
      sc[0] *= fit.f;
      sc[1] *= fit.f;
    }
    const v8 df[2][2] = {{pack<T>(sc[0], 0), pack<T>(sc[0], 1)}, {pack<T>(sc[1], 0), pack<T>(sc[1], 1)}};
#pragma unroll
    for (int c = 0; c < 2; ++c) add_cols<T, D>(kcol + (cur * TILE + c * 32 * D) * sizeof(T), df[c], dq[c]);
  }
  dl += __shfl_xor(dl, 32, 64);
  const int t32 = tile * NW + wave;
  if (h == 0 && t32 < a.tiles32) {
    float* rs = a.part + ((long)bh * a.tiles32 + t32) * (RS_LINES * 32) + lane;
    const bool on = row < a.R;
    rs[32 * RS_L1] = on && lim ? l1 : INFINITY;
    rs[32 * RS_L2] = on && lim ? l2 : INFINITY;
    rs[32 * RS_D1] = on ? d1 : 0.f;
    rs[32 * RS_LD2] = on ? lam * d2 : 0.f;
    rs[32 * RS_LAM] = on ? lam : 0.f;
    rs[32 * RS_LIM] = __builtin_bit_cast(float, on ? lim : 0);
    rs[32 * RS_DL] = on ? dl : 0.f;
  }
  if (row >= a.R) return;
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

// dlam of a head: minus the sum over its rows of sum_j P_2 dP, in fp64, in a fixed order
__device__ __forceinline__ void head_dlam(const DaArgs& a, int head) {
  __shared__ double red[16];
  const int hk = head / a.G, g = head - hk * a.G;
  double v = 0.;
  const long total = (long)a.B * a.T;
  for (long i = threadIdx.x; i < total; i += blockDim.x) {
    const long b = i / a.T, r = (i - b * a.T) * a.G + g;
    v += a.part[((b * a.Hkv + hk) * a.tiles32 + (r >> 5)) * (RS_LINES * 32) + 32 * RS_DL + (r & 31)];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0) {
    double sum = 0.;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) sum += red[i];
    a.dlam[head] = (float)-sum;
  }
}
__global__ __launch_bounds__(1024) void da_dlam(const DaArgs a) { head_dlam(a, blockIdx.x); }

// dK and dV of 32 keys a pair of waves, NP pairs a workgroup, walking the rows that see them.  The pair divides the work, with
// the same number of matrix instructions each: the first wave forms the maps and dV = (P_1 - lam P_2)^T dO, the second
// dP, dS and dK_c = dS_c^T Q_c; the probabilities pass from one to the other through LDS in fp32, once a tile.  Each so
// holds half of the accumulators and three waves (two at D = 128) fit a SIMD: one's exponentials run under the other's products.
// Bound by the two barriers a tile and the pass through LDS (matrix unit 28 %, VALU 40 % of the busy cycles): 435 - 480 us at
// 2 x 4096 causal, 16 over 4 heads, D = 64, bf16, where a wave that did a key's whole work alone took 905 (its accumulators leave
// one wave a SIMD).
template <typename T, int D, int NP>
__global__ __launch_bounds__(128 * NP, D == 128 ? 2 : 3) void da_bwd_kv(const DaArgs a) {
  constexpr int DV = 2 * D, KQ = D / 16, KV = DV / 16, NQ = D / 32, NO = DV / 32, NW = 2 * NP, TILE = Stage<T, D, NW>::TILE;
  constexpr bool HALF = ColScale<T>::ON;
  typedef Stage<T, D, NW> St;
  typedef typename Vec<T>::v8 v8;
  __shared__ __align__(1024) T tiles[2][TILE];
  __shared__ __align__(16) float stats[2][RS_LINES * 32];
  __shared__ __align__(16) f32x4 probs[NP][2][4][64];
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nbh = a.B * a.Hkv;
  const int pair = wave % NP;
  const St plan(wave, lane);
  // the causally longest come first
  const int bh = blockIdx.x % nbh, tile = blockIdx.x / nbh / a.splits, sp = blockIdx.x / nbh % a.splits;
  const Seq s(a, bh);
  const int kb = tile * 32 * NP, kw = kb + pair * 32, key = kw + (lane & 31), kr = min(key, a.S - 1);
  // rows that see a key of the block: positions from t0 to the sequence's end
  const int t0 = kb >= s.kl ? s.ql : a.causal ? max(0, kb - (s.kl - s.ql)) : 0;
  // (rows of the first tile before t0 come as zeros: a row that sees no key adds nothing, whatever its dO holds)
  const int r_lo = t0 * a.G;
  int r0 = r_lo / 32 * 32, r1 = s.ql * a.G;
  if (a.splits > 1) {              // this split's share of them
    const int per = (max(0, r1 - r0) / 32 + a.splits) / a.splits * 32;
    r0 += sp * per;
    r1 = min(r1, r0 + per);
  }
  // row rb is position tb, head `rem`; rb moves by 32.  A row's position from there is a division of a number below G + 32
  // by G: the upper half of its product with ceil(2^32 / G), exact below 2^16.
  int tb = r0 / a.G, rem = r0 - tb * a.G;
  const uint32_t magic = a.G == 1 ? 0 : (uint32_t)((0x100000000ull + a.G - 1) / a.G);
  const auto over_g = [&](int n) { return a.G == 1 ? n : (int)__umulhi((uint32_t)n, magic); };
  const auto stage = [&](int rb, int cur, auto first) {
    const auto qb = (const T*)a.q + s.b * a.q_sb + tb * a.q_st + s.hk * a.G * a.q_sh;
    const auto gb = (const T*)a.dout + s.b * a.g_sb + tb * a.g_st + s.hk * a.G * a.g_sh;
#pragma unroll
    for (int i = 0; i < St::ROLES; ++i) {
      const int role = St::role(i, wave), step = St::step(role);
      const auto rs = open_range(role < 2 ? qb + (role ? a.q_sc : 0) : gb);
      const int st = (int)((role < 2 ? a.q_st : a.g_st) * sizeof(T)), sh = (int)((role < 2 ? a.q_sh : a.g_sh) * sizeof(T));
#pragma unroll
      for (int j = 0; j < St::PER; ++j) {
        const int x = plan.row[i] + j * step, t = over_g(rem + x), g = rem + x - t * a.G;
        const uint32_t off = t * st + g * sh + plan.byte[i][j];
        bool in = rb + x < r1;
        if constexpr (decltype(first)::value) in = in && rb + x >= r_lo;
        dma16(rs, tiles[cur] + St::place(role, wave) + j * 512, in ? off : BUF_OOB);
      }
    }
    rem += 32;
    const int t = over_g(rem);
    tb += t;
    rem -= t * a.G;
    if (wave == 0) dma16(open_range(a.part + ((long)bh * a.tiles32 + rb / 32) * (RS_LINES * 32)), stats[cur], lane * 16);
  };
  if (r0 < r1) stage(r0, 0, std::true_type());
  const long out = ((long)s.b * a.S + key) * a.Hkv + s.hk;
  // four elements of the key's dK (from 0) or dV (from DV), or of their part
  const auto put = [&](T* to, int from, int c, const f32x4& x) {
    if (a.splits > 1) *(f32x4*)(a.kvpart + (((long)sp * a.B * a.S * a.Hkv + out) * 2 * DV + from + c)) = x;
    else *(typename Vec<T>::v4*)(to + out * DV + c) = __builtin_convertvector(x, typename Vec<T>::v4);
  };
  if (wave < NP) {
    const T* kp = (const T*)a.k + s.b * a.k_sb + s.hk * a.k_sh + (long)kr * a.k_ss;
    v8 kf[2][KQ];
#pragma unroll
    for (int k = 0; k < KQ; ++k) {
      kf[0][k] = *(const v8*)(kp + 16 * k + 8 * h);
      kf[1][k] = *(const v8*)(kp + a.k_sc + 16 * k + 8 * h);
    }
    f32x16 dv[NO];
#pragma unroll
    for (int j = 0; j < NO; ++j) dv[j] = 0.f;
    ColScale<T> fit;               // P_1 - lam P_2 of a key: up to 1 + |lam|, and as small as the key is far from all rows
    const uint32_t gcol = col_base<T, DV>(tiles[0] + 64 * D, lane);
    int cur = 0;
    for (int rb = r0; rb < r1; rb += 32, cur ^= 1) {
      tile_ready();
      if (rb + 32 < r1) stage(rb + 32, cur ^ 1, std::false_type());
      const T* qs = tiles[cur];
      const float* st = stats[cur];
      // a row below the diagonal of the pair's last key, or a key behind the end, needs the mask
      const bool edge = kw + 32 > s.kl || (a.causal && rb / a.G + s.kl - s.ql < kw + 31);
      f32x16 pc, sc[2];
      sc[0] = sc[1] = 0.f;
#pragma unroll
      for (int k = 0; k < KQ; ++k) {
        sc[0] = Mfma<T>::run(frag_row<T, D>(qs, k, lane), kf[0][k], sc[0]);
        sc[1] = Mfma<T>::run(frag_row<T, D>(qs + 32 * D, k, lane), kf[1][k], sc[1]);
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 ls = *(const f32x4*)(st + 32 * (c ? RS_L2 : RS_L1) + 8 * r4 + 4 * h);
#pragma unroll
          for (int j = 0; j < 4; ++j) sc[c][4 * r4 + j] = __builtin_amdgcn_exp2f(fmaf(sc[c][4 * r4 + j], a.c, -ls[j]));
        }
      if (edge) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const i32x4 lim = *(const i32x4*)(st + 32 * RS_LIM + 8 * r4 + 4 * h);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            sc[0][4 * r4 + j] = key < lim[j] ? sc[0][4 * r4 + j] : 0.f;
            sc[1][4 * r4 + j] = key < lim[j] ? sc[1][4 * r4 + j] : 0.f;
          }
        }
      }
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x4 lam = *(const f32x4*)(st + 32 * RS_LAM + 8 * r4 + 4 * h);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          f32x4 p;
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = sc[c][4 * r4 + j];
          probs[pair][c][r4][lane] = p;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) pc[4 * r4 + j] = fmaf(-lam[j], sc[1][4 * r4 + j], sc[0][4 * r4 + j]);
      }
      const float down = fit.fit(top_of<T>(pc));
      if (__any(down != 1.f)) {
#pragma unroll
        for (int j = 0; j < NO; ++j) dv[j] *= down;
      }
      if constexpr (HALF) pc *= fit.f;
      const v8 pf[2] = {pack<T>(pc, 0), pack<T>(pc, 1)};
      lds_barrier();
      add_cols<T, DV>(gcol + cur * TILE * sizeof(T), pf, dv);
    }
    if (key >= a.S) return;
    const float f = 1.f / fit.f;
#pragma unroll
    for (int j = 0; j < NO; ++j)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = dv[j][4 * r4 + r] * f;
        put((T*)a.dv, DV, 32 * j + 8 * r4 + 4 * h, x);
      }
  } else {
    const T* vp = (const T*)a.v + s.b * a.v_sb + s.hk * a.v_sh + (long)kr * a.v_ss;
    v8 vf[KV];
#pragma unroll
    for (int k = 0; k < KV; ++k) vf[k] = *(const v8*)(vp + 16 * k + 8 * h);
    f32x16 dk[2][NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) dk[0][j] = dk[1][j] = 0.f;
    ColScale<T> fit;
    const uint32_t qcol = col_base<T, D>(tiles[0], lane);
    int cur = 0;
    for (int rb = r0; rb < r1; rb += 32, cur ^= 1) {
      tile_ready();
      if (rb + 32 < r1) stage(rb + 32, cur ^ 1, std::false_type());
      const T* gs = tiles[cur] + 64 * D;
      const float* st = stats[cur];
      f32x16 dp = 0.f;
#pragma unroll
      for (int k = 0; k < KV; ++k) dp = Mfma<T>::run(frag_row<T, DV>(gs, k, lane), vf[k], dp);
      // dP of a masked place may be anything (a value behind the end): its dS is 0
      const bool edge = kw + 32 > s.kl;
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dp[r] = key < s.kl ? dp[r] : 0.f;
      }
      lds_barrier();
      f32x16 ds[2];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int at = 8 * r4 + 4 * h;
        const f32x4 d1 = *(const f32x4*)(st + 32 * RS_D1 + at), d2 = *(const f32x4*)(st + 32 * RS_LD2 + at),
                    lam = *(const f32x4*)(st + 32 * RS_LAM + at);
        const f32x4 p1 = probs[pair][0][r4][lane], p2 = probs[pair][1][r4][lane];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * r4 + j;
          ds[0][r] = p1[j] * (dp[r] - d1[j]);
          ds[1][r] = p2[j] * fmaf(-lam[j], dp[r], d2[j]);
        }
      }
      const float down = fit.fit(top_of<T>(ds[1], top_of<T>(ds[0])));
      if (__any(down != 1.f)) {
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int j = 0; j < NQ; ++j) dk[c][j] *= down;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if constexpr (HALF) ds[c] *= fit.f;
        const v8 df[2] = {pack<T>(ds[c], 0), pack<T>(ds[c], 1)};
        add_cols<T, D>(qcol + (cur * TILE + c * 32 * D) * sizeof(T), df, dk[c]);
      }
    }
    if (key >= a.S) return;
    const float f = a.scale / fit.f;
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          f32x4 x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = dk[c][j][4 * r4 + r] * f;
          put((T*)a.dk, 0, c * D + 32 * j + 8 * r4 + 4 * h, x);
        }
  }
}

// sums the row splits' dK and dV in order: a thread takes four elements of a key's 2 D + 2 D
template <typename T, int D>
__global__ __launch_bounds__(256) void da_kv_join(const DaArgs a) {
  constexpr int DV = 2 * D;
  const long n = (long)a.B * a.S * a.Hkv * (2 * DV), i = ((long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  f32x4 v = *(const f32x4*)(a.kvpart + i);
  for (int s = 1; s < a.splits; ++s) v += *(const f32x4*)(a.kvpart + s * n + i);
  const long key = i / (2 * DV);
  const int c = (int)(i - key * (2 * DV));
  *(typename Vec<T>::v4*)((T*)(c < DV ? a.dk : a.dv) + key * DV + (c < DV ? c : c - DV)) = __builtin_convertvector(v, typename Vec<T>::v4);
}

// ------------------------------------------------------------------------------------------------ host side
// Two pairs of waves share a key tile where the rows fill them; a few rows over many keys are one pair.
bool da_wide(long rows) { return rows > 32; }

// Key splits that give every compute unit two workgroups of four waves, or of two as many as its LDS takes, with at least 128
// keys each
int da_splits(const ctr_diffattn_t* p) {
  const long R = (long)p->T * (p->H / p->Hkv);
  const bool wide = da_wide(R);
  const long blocks = (long)cdiv(R, wide ? 64 : 32) * p->B * p->Hkv;
  return (int)std::max<long>(1, std::min<long>((wide || p->D == 128 ? 512 : 1024) / std::max<long>(1, blocks), p->S / 128));
}

constexpr int da_pairs(int D) { return D == 128 ? 4 : 2; }

// Row splits of the dK / dV kernel: eight workgroups a compute unit in all, so that the causal differences of their lengths
// even out, with at least eight row tiles each; a split costs its fp32 part of dK and dV, written and read once.
int da_kv_splits(const ctr_diffattn_t* p) {
  const long blocks = (long)cdiv(p->S, 32 * da_pairs(p->D)) * p->B * p->Hkv, tiles = cdiv((long)p->T * (p->H / p->Hkv), 32);
  return (int)std::max<long>(1, std::min<long>({8, 2048 / std::max<long>(1, blocks), tiles / 8}));
}
size_t da_rowstat_bytes(const ctr_diffattn_t* p) {
  return (size_t)p->B * p->Hkv * cdiv((long)p->T * (p->H / p->Hkv), 32) * RS_LINES * 32 * sizeof(float);
}

// elements from the first to the last head of a group
long da_span(long sh, long G) { return G == 1 ? 0 : sh > (1L << 40) ? sh : sh * (G - 1); }

int da_check(const ctr_diffattn_t* p, bool bwd) {
  CTR_REQUIRE(p, "null argument");
  CTR_REQUIRE(p->type == TY_BF16 || p->type == TY_F16, "type (1 bf16, 2 fp16)");
  CTR_REQUIRE(p->D == 32 || p->D == 64 || p->D == 128, "map width D in {32, 64, 128}");
  CTR_REQUIRE(p->B >= 0 && p->T >= 0 && p->S >= 0 && p->H >= 1 && p->Hkv >= 1 && p->H % p->Hkv == 0, "sizes");
  CTR_REQUIRE((long)p->T * (p->H / p->Hkv) < (1L << 30) && p->S < (1 << 30) && p->H / p->Hkv < (1 << 15), "sizes");
  CTR_REQUIRE((long)p->B * p->Hkv * cdiv((long)p->T * (p->H / p->Hkv), 32) < (1L << 31) &&
                  (long)p->B * p->Hkv * cdiv(p->S, 32) < (1L << 31) && (long)p->B * p->H * p->T < (1L << 31), "sizes");
  CTR_REQUIRE(p->scale > 0.f && std::isfinite(p->scale), "scale > 0");
  if ((long)p->B * p->T == 0 && !(bwd && (long)p->B * p->S > 0)) return 0;
  CTR_REQUIRE(p->lam, "null lam");
  // a tile's byte offsets are 32 bits wide: those of 32 positions and those of a group's heads are held to 2^30 each
  const auto ok = [](const void* q, std::initializer_list<long> st, long row, long head) {
    if (!q || (uintptr_t)q % 16) return false;
    for (long s : st)
      if (s % 8 || s < 0) return false;
    return row < (1L << 24) && head < (1L << 29);
  };
  const long G = p->H / p->Hkv;
  CTR_REQUIRE((long)p->B * p->T == 0 || ok(p->q, {p->q_sb, p->q_st, p->q_sh, p->q_sc}, p->q_st, da_span(p->q_sh, G)), "q: 16-byte aligned rows");
  CTR_REQUIRE((long)p->B * p->S == 0 || ok(p->k, {p->k_sb, p->k_ss, p->k_sh, p->k_sc}, p->k_ss, 0), "k: 16-byte aligned rows");
  CTR_REQUIRE((long)p->B * p->S == 0 || ok(p->v, {p->v_sb, p->v_ss, p->v_sh}, p->v_ss, 0), "v: 16-byte aligned rows");
  CTR_REQUIRE((long)p->B * p->T == 0 || (p->o && (uintptr_t)p->o % 16 == 0 && (uintptr_t)p->o2 % 16 == 0 && (uintptr_t)p->ol % 16 == 0 && !p->o2 == !p->ol), "output");
  return 0;
}

DaArgs da_args(const ctr_diffattn_t* p) {
  DaArgs a = {};
  a.q = p->q; a.k = p->k; a.v = p->v; a.lam = p->lam;
  a.o = p->o; a.o2 = p->o2; a.ol = p->ol; a.stat = p->stat;
  a.q_lens = p->q_lens; a.kv_lens = p->kv_lens;
  a.q_sb = p->q_sb; a.q_st = p->q_st; a.q_sh = p->q_sh; a.q_sc = p->q_sc;
  a.k_sb = p->k_sb; a.k_ss = p->k_ss; a.k_sh = p->k_sh; a.k_sc = p->k_sc;
  a.v_sb = p->v_sb; a.v_ss = p->v_ss; a.v_sh = p->v_sh;
  a.scale = p->scale;
  a.c = p->scale * 1.44269504088896341f;
  a.B = p->B; a.T = p->T; a.S = p->S; a.H = p->H; a.Hkv = p->Hkv; a.G = p->H / p->Hkv; a.R = p->T * a.G;
  a.rows = (long)p->B * p->Hkv * a.R;
  a.plane = a.rows * 2 * p->D;
  a.causal = p->causal;
  a.splits = 1;
  return a;
}

template <typename T, int D>
int da_run_fwd(DaArgs a, hipStream_t s) {
  const long bh = (long)a.B * a.Hkv;
  const bool wide = da_wide(a.R);
  a.tiles = cdiv(a.R, wide ? 64 : 32);
  const long blocks = a.tiles * bh * a.splits;
  if (wide) da_fwd<T, D, 2><<<(unsigned)blocks, 256, 0, s>>>(a);
  else da_fwd<T, D, 1><<<(unsigned)blocks, 128, 0, s>>>(a);
  if (a.splits > 32) da_join<T, D, 32><<<dim3((unsigned)a.rows, 2 * D / 32), 1024, 0, s>>>(a);
  else if (a.splits > 1) da_join<T, D, 4><<<dim3((unsigned)a.rows, 2 * D / 32), 128, 0, s>>>(a);
  return check_launch("diffattn_fwd");
}

template <typename T, int D>
int da_run_bwd(DaArgs a, int kv_splits, hipStream_t s) {
  const long bh = (long)a.B * a.Hkv;
  a.tiles32 = cdiv(a.R, 32);
  if (a.rows > 0) {
    const bool wide = a.R > 64;
    a.tiles = cdiv(a.R, wide ? 128 : 32);
    if (wide) da_bwd_q<T, D, 4><<<(unsigned)(a.tiles * bh), 256, 0, s>>>(a);
    else da_bwd_q<T, D, 1><<<(unsigned)(a.tiles * bh), 64, 0, s>>>(a);
  }
  if (bh * a.S > 0) {
    constexpr int NP = da_pairs(D);
    a.tiles = cdiv(a.S, 32 * NP);
    a.splits = kv_splits;
    da_bwd_kv<T, D, NP><<<(unsigned)(a.tiles * bh * a.splits), 128 * NP, 0, s>>>(a);
    if (a.splits > 1) da_kv_join<T, D><<<(unsigned)cdiv(bh * a.S * 4 * D, 1024), 256, 0, s>>>(a);
  }
  da_dlam<<<a.H, 1024, 0, s>>>(a);
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
  if (!p || p->B <= 0 || p->T <= 0 || p->Hkv <= 0 || p->H < p->Hkv) return 0;
  const int splits = da_kv_splits(p);
  return da_rowstat_bytes(p) + (splits > 1 ? (size_t)splits * p->B * p->S * p->Hkv * 4 * p->D * sizeof(float) : 0);
}

extern "C" int ctr_diffattn_bwd(const ctr_diffattn_t* p, const void* dout, long g_sb, long g_st, long g_sh, void* dq, void* dk,
                                void* dv, float* dlam, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = da_check(p, true)) return rc;
  CTR_REQUIRE(dlam, "null dlam");
  const bool q_on = (long)p->B * p->T > 0, k_on = (long)p->B * p->S > 0;
  CTR_REQUIRE(!q_on || (p->o2 && p->ol && p->stat && dq && dout), "null operand");
  CTR_REQUIRE(!q_on || ((uintptr_t)dout % 16 == 0 && g_sb % 8 == 0 && g_st % 8 == 0 && g_sh % 8 == 0 && g_sb >= 0 &&
                        g_st >= 0 && g_sh >= 0 && g_st < (1L << 24) && da_span(g_sh, p->H / p->Hkv) < (1L << 29)), "dout: 16-byte aligned rows");
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
  a.part = (float*)ws;
  a.kvpart = (float*)((char*)ws + da_rowstat_bytes(p));
  a.dlam = dlam;
#define DA_CALL(T, D) da_run_bwd<T, D>(a, da_kv_splits(p), (hipStream_t)stream)
  DA_TYPES(DA_CALL);
#undef DA_CALL
}
