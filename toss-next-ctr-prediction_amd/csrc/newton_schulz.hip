// Newton-Schulz orthogonalisation of matrices (the direction of a Muon update) and the update around it.
//   X_0 = G / (||G||_F + eps)  (transposed when it has more rows than columns: m <= n below)
//   A = X X^T,   W = a I + b A + c A^2,   X <- W X        (`steps` times)
//
// Arithmetic.  X, A and W are kept as two fp16 planes, hi = fp16(s v) and lo = fp16(s v - hi) with s a power of two as large
// as the planes' range allows (X: 2^12, A and W: 2^10; the host refuses coefficients under which a singular value of X could
// pass 8 or one of W 32): 22 mantissa bits and a sign of lo, which is fp32's step to within a factor of two, for elements of X
// from 2^-15 of its norm up, and an absolute 2^-37 of the norm below, where lo is subnormal (elements under 2^-26 so keep fewer
// bits than a 16-bit input has; in the norm it counts from 65536 x 65536 on).  A product of two such values is hi hi + hi lo + lo hi on v_mfma_f32_32x32x16_f16 with fp32
// accumulation; the lo lo term is 2^-24 of it.  Three fp16 products cost 3/16 of one fp32 matrix instruction's time, so
// this is fp32's accuracy at up to five times its rate.  16-bit accuracy would not do: the polynomial multiplies the error
// of a small singular value by a (3.44) a step, 485 times in five.  Nor would the hi parts do for a bf16 result's last step (2048 x
// 8192: 1815 us instead of 1942): roundings of matrices with structure do not average out, all ones of 150 x 333 came out 1.2 half
// steps of bf16 off before their own rounding.  The squares of the norm are summed in fp64, where no fp32 input overflows or
// vanishes.
#include <algorithm>
#include <atomic>

#include "ctr_hip.h"
#include "vec16.h"

namespace ctr {
namespace {

constexpr float SX = 4096.f, SA = 1024.f;      // the planes' scales of X and of A, W
constexpr int NS_MAXMAT = 20;                  // matrices of one launch (their table rides in the kernel arguments)
constexpr int NS_BK = 32;
constexpr int NS_SUMSQ_BLOCKS = 256;
constexpr int NS_SMALL_LDS = 160 * 1024 - 256;   // of a workgroup, next to its few static bytes

struct NsMat {
  const void* src;
  void* dst;
  long ld_src, ld_dst;
  int rows, cols;          // as given
  int m, n, mp, np;        // m <= n, and both rounded up to the tile
  long off_x, off_a, off_p, off_s;     // bytes into the workspace: X planes (two buffers), A and W planes, partials, sums
  int splits, asplits, type, group;      // shares of K of X X^T and of A A
 
};
struct NsArgs {
  int count;
  int pre[NS_MAXMAT + 1];  // first block of each matrix
  char* ws;
  float a, b, c, eps;
  NsMat mat[NS_MAXMAT];
};

__device__ __forceinline__ int ns_find(const NsArgs& p, int blk) {
  int i = 0;
  while (i + 1 < p.count && blk >= p.pre[i + 1]) ++i;
  return i;
}

__device__ __forceinline__ float ns_load(const NsMat& q, int r, int c) {
  const long o = (long)r * q.ld_src + c;
  return q.type == TY_F32 ? ((const float*)q.src)[o] : q.type == TY_BF16 ? (float)((const __bf16*)q.src)[o]
                                                                         : (float)((const _Float16*)q.src)[o];
}
__device__ __forceinline__ void ns_store(const NsMat& q, int r, int c, float v) {
  const long o = (long)r * q.ld_dst + c;
  if (q.type == TY_F32) ((float*)q.dst)[o] = v;
  else if (q.type == TY_BF16) ((__bf16*)q.dst)[o] = (__bf16)v;
  else ((_Float16*)q.dst)[o] = (_Float16)v;
}

// The planes in the workspace: 32 hi, then the same 32 lo values, so that a K step of a row is one line of 128 bytes (with a
// plane after the other it was half a line of each, and twice the requests).  Where hi of (row, col) stands; lo: 32 further.
__device__ __forceinline__ long at(long row, int col, int ld) { return row * 2 * ld + (col >> 5) * 64 + (col & 31); }

__device__ __forceinline__ void split16(float v, _Float16& hi, _Float16& lo) {
  hi = (_Float16)v;
  lo = (_Float16)(v - (float)hi);
}

__device__ __forceinline__ double block_sum64(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += red[i];
  return s;
}

// C layout of a 32x32 tile: register r of lane l holds row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32
__device__ __forceinline__ int c_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

#define MFMA16(A, B, C) __builtin_amdgcn_mfma_f32_32x32x16_f16(A, B, C, 0, 0, 0)

typedef __attribute__((address_space(3))) f16x4 lds_f16x4;
typedef short s16x4 __attribute__((ext_vector_type(4)));

// Fragment of 32 rows x 16 k from rows with contiguous k: lane l has row l % 32, k = 8 (l / 32) + 0..7
__device__ __forceinline__ f16x8 frag_k(const _Float16* p, int ld, int row, int k, int lane) {
  return *(const f16x8*)(p + (row + (lane & 31)) * ld + k + 8 * (lane >> 5));
}
// The same rows with the k order that frag_t gives: 4 (l / 32) + 0..3, then 8 + 4 (l / 32) + 0..3
__device__ __forceinline__ f16x8 frag_kp(const _Float16* p, int ld, int row, int k, int lane) {
  const _Float16* q = p + (row + (lane & 31)) * ld + k + 4 * (lane >> 5);
  const f16x4 u = *(const f16x4*)q, v = *(const f16x4*)(q + 8);
  return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Fragment of 16 k x 32 columns from rows of contiguous columns, by the LDS transpose read: a group of 16 lanes takes
// 4 k rows of 16 columns, lane i of it the address of row i / 4, columns 4 (i % 4), and gets column i's four k
__device__ __forceinline__ f16x8 frag_t(const _Float16* p, int ld, int k, int col, int lane) {
  const int row = k + 4 * (lane >> 5) + ((lane & 15) >> 2), c = col + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
  auto q = (__attribute__((address_space(3))) s16x4*)(p + row * ld + c);
  auto q8 = (__attribute__((address_space(3))) s16x4*)(p + (row + 8) * ld + c);
  const f16x4 u = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(q));
  const f16x4 v = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(q8));
  return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
}

// ------------------------------------------------------------------------------------------------ large matrices
template <typename T>
__device__ __forceinline__ double ns_rows_sumsq(const NsMat& q) {
  // 8-element pieces of the rows, dealt over all threads; a thread's own sum of 64 squares at a time in fp32 would overflow
  // where the matrix does not, so fp64 from the start
  double s = 0.;
  const int per = (q.cols + 7) / 8;
  const long total = (long)q.rows * per, step = (long)NS_SUMSQ_BLOCKS * 256;
  const int dr = (int)(step / per), dc = (int)(step % per);
  long i = (long)blockIdx.x * 256 + threadIdx.x;
  int r = (int)(i / per), c = (int)(i % per);
  for (; i < total; i += step) {
    const f32x8 v = ld8f((const T*)q.src + (long)r * q.ld_src + c * 8, q.cols - c * 8);
#pragma unroll
    for (int k = 0; k < 8; ++k) s = fma((double)v[k], (double)v[k], s);
    r += dr;
    c += dc;
    if (c >= per) c -= per, ++r;
  }
  return s;
}
__global__ __launch_bounds__(256) void ns_sumsq(const NsArgs p) {
  const NsMat& q = p.mat[blockIdx.y];
  __shared__ double red[4];
  double s = q.type == TY_F32 ? ns_rows_sumsq<float>(q) : q.type == TY_BF16 ? ns_rows_sumsq<__bf16>(q) : ns_rows_sumsq<_Float16>(q);
  s = block_sum64(s, red);
  if (threadIdx.x == 0) ((double*)(p.ws + q.off_s))[blockIdx.x] = s;
}

// X_0's planes, 64 x 64 elements a block, through LDS when transposed
__global__ __launch_bounds__(256) void ns_init(const NsArgs p) {
  const int i = ns_find(p, blockIdx.x);
  const NsMat& q = p.mat[i];
  __shared__ double red[4];
  __shared__ float tile[64][65];
  const double part = threadIdx.x < NS_SUMSQ_BLOCKS ? ((const double*)(p.ws + q.off_s))[threadIdx.x] : 0.;
  const float scale = (float)(SX / (sqrt(block_sum64(part, red)) + (double)p.eps));
  const int id = blockIdx.x - p.pre[i], tc = q.np / 64, m0 = id / tc * 64, n0 = id % tc * 64;
  const bool tall = q.rows > q.cols;
  const int lx = threadIdx.x & 63, ly = threadIdx.x >> 6;
  for (int j = ly; j < 64; j += 4) {
    const int r = tall ? n0 + j : m0 + j, c = tall ? m0 + lx : n0 + lx;
    tile[j][lx] = r < q.rows && c < q.cols ? ns_load(q, r, c) : 0.f;
  }
  __syncthreads();
  _Float16* x = (_Float16*)(p.ws + q.off_x);
  for (int j = ly; j < 64; j += 4) {
    const float v = tall ? tile[lx][j] : tile[j][lx];
    const long o = at(m0 + j, n0 + lx, q.np);
    split16(v * scale, x[o], x[o + 32]);
  }
}

// 64 lanes x 16 bytes to consecutive LDS places.  Nothing comes back in registers and the K loop waits for it by count.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"      // m0 is a reserved register; it is named because it changes
__device__ __forceinline__ void ns_dma16(__amdgpu_buffer_rsrc_t r, uint32_t lds, uint32_t off, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(off), "s"(r), "s"(soff) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void ns_wait() {      // all but the last N loads have landed, in every wave
  static_assert(N <= 63, "vmcnt");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A tile of a product, K from k0 to k1 (multiples of 32): A rows from r0, B rows (NT) or columns (NN) from c0.  Eight waves, WR
// by 8 / WR, of NI x NJ blocks of 32 x 32: two a SIMD, so that one's products run under the other's LDS reads (four waves of
// 64 x 64 took the sum of both, 0.86 us a step).  A K step's planes come by direct loads to one of NST places in LDS, NST - 1
// steps ahead.  2048 x 2048 x 8192, three products: 256 x 256 tiles 186 us (1.1 PFLOP/s, the rate of a large 16-bit product on
// this card is 1.25), 256 x 128 197; its symmetric product, with half as many tiles: 256 x 128 150, 256 x 256 165; below 768
// rows, where a tile's chain of steps is what counts, 128 x 128 (512 x 7552: 20 us, 0.6 PFLOP/s).
// In LDS a row of 128 bytes (A, NT: hi and lo of 32 k) holds its 16-byte chunk c at c ^ (row / 2 % 8), one of 4 C bytes (NN:
// hi and lo of C columns) at c ^ (4 (row % 4) + row / 4 % 4): the row and the transpose reads cover all banks.
template <int WR_, int NI_, int NJ_, int NST_>
struct NsTile {
  static constexpr int WR = WR_, WC = 8 / WR, NI = NI_, NJ = NJ_, NST = NST_, R = 32 * WR * NI, C = 32 * WC * NJ;
  static constexpr int PA = 2 * NS_BK * R, STAGE = 2 * NS_BK * (R + C);      // elements of a step's planes of A, of both
  static constexpr int LDS = std::max(NST * STAGE, 2 * 128 * (C + 8)) * 2;   // bytes, the store of the result included
  using Acc = f32x16[NI][NJ];
};
constexpr int NS_GROUPS = 3;               // matrices that share their tiles
using NsSmall = NsTile<2, 2, 1, 4>;        // 128 x 128
using NsMid = NsTile<4, 2, 2, 3>;          // 256 x 128
using NsLarge = NsTile<2, 4, 2, 2>;        // 256 x 256
template <bool NN, class S>
__device__ __forceinline__ void ns_tile(const _Float16* A, int lda, const _Float16* B, int ldb, int r0, int c0, int k0, int k1,
                                        _Float16* lds, typename S::Acc& acc) {
  constexpr int NI = S::NI, NJ = S::NJ, NST = S::NST, NA = S::R / 64, NB = S::C / 64, LOADS = NA + NB, RPL = 256 / S::C;
  static_assert(S::R % 128 == 0 && (S::C == 128 || S::C == 256), "loads dealt to eight waves");
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wave / S::WC * 32 * NI, wc = wave % S::WC * 32 * NJ;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds;
  // a load is 8 rows of 128 bytes, or RPL of 4 C; a wave takes NA of A and NB of B
  const _Float16* asrc = A + at(r0 + 8 * NA * wave, k0, lda);
  const _Float16* bsrc = B + (NN ? at(k0 + 4 * wave, c0, ldb) : at(c0 + 8 * NB * wave, k0, ldb));
  uint32_t aoff[2], boff[NB];
#pragma unroll
  for (int j = 0; j < 2; ++j) aoff[j] = (lane >> 3) * lda * 4 + ((lane & 7) ^ ((4 * j + (lane >> 4)) & 7)) * 16;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int r = RPL * j + lane / (S::C / 4);        // of the wave's four K rows
    boff[j] = NN ? lane / (S::C / 4) * ldb * 4 + ((lane % (S::C / 4)) ^ ((r & 3) << 2 | (wave & 3))) * 16
                 : (lane >> 3) * ldb * 4 + ((lane & 7) ^ ((4 * j + (lane >> 4)) & 7)) * 16;
  }
  const auto stage = [&](int step, int place) {
    const auto ra = buf_rsrc(asrc + (long)step * 2 * NS_BK, 0x7ffffff0u);
    const auto rb = buf_rsrc(bsrc + (NN ? (long)step * 2 * NS_BK * ldb : (long)step * 2 * NS_BK), 0x7ffffff0u);
    const uint32_t ta = lds0 + (place * S::STAGE + wave * NA * 512) * 2, tb = lds0 + (place * S::STAGE + S::PA + wave * NB * 512) * 2;
#pragma unroll
    for (int j = 0; j < NA; ++j) ns_dma16(ra, ta + j * 1024, aoff[j & 1], j * 32 * lda);
#pragma unroll
    for (int j = 0; j < NB; ++j) ns_dma16(rb, tb + j * 1024, boff[j], j * (NN ? 4 * RPL : 32) * ldb);
  };
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = 0.f;
  const int steps = (k1 - k0) / NS_BK;
#pragma unroll
  for (int i = 0; i < NST - 1; ++i)
    if (i < steps) stage(i, i);
  const int row = lane & 31, h = lane >> 5, turn = (row >> 1) & 7;
  const int arow = (wr + row) * 2 * NS_BK, brow = (wc + row) * 2 * NS_BK;
  const int tk = 8 * h + ((lane & 15) >> 2), tc = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;      // transpose reads: row, column
  struct Frags { f16x8 a[2][NI], b[2][NJ]; };      // [plane][tile]
  const auto read = [&](int place, int kk) {
    const _Float16* s = lds + place * S::STAGE;
    const _Float16* bp = s + S::PA;
    Frags f;
#pragma unroll
    for (int pl = 0; pl < 2; ++pl) {
      const int ch = ((4 * pl + 2 * kk + h) ^ turn) * 8;
#pragma unroll
      for (int i = 0; i < NI; ++i) f.a[pl][i] = *(const f16x8*)(s + arow + 64 * i * NS_BK + ch);
#pragma unroll
      for (int i = 0; i < NJ; ++i) {
        if constexpr (!NN) f.b[pl][i] = *(const f16x8*)(bp + brow + 64 * i * NS_BK + ch);
        else {
          f16x4 u[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = 16 * kk + tk + 4 * half, c = (wc / 32 + i) * 8 + 4 * pl + (tc >> 3);
            const _Float16* q = bp + r * 2 * S::C + (c ^ (((r & 3) << 2) | ((r >> 2) & 3))) * 8 + (tc & 4);
            u[half] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)q));
          }
          f.b[pl][i] = __builtin_shufflevector(u[0], u[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
      }
    }
    return f;
  };
  const auto multiply = [&](const Frags& f) {
#pragma unroll
    for (int pr = 0; pr < 3; ++pr) {    // lo hi, hi lo, hi hi; the accumulators in turn
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = MFMA16(f.a[pr == 0][i], f.b[pr == 1][j], acc[i][j]);
    }
  };
  int place = 0;
  if constexpr (NI * NJ > 4) {      // no registers for a second set of fragments; written out, as read() and multiply() spill here
    for (int k = 0; k < steps; ++k) {
      if (k + NST - 1 <= steps) ns_wait<LOADS * (NST - 2)>();
      else ns_wait<0>();
      if (k + NST - 1 < steps) stage(k + NST - 1, place == 0 ? NST - 1 : place - 1);
      const _Float16* s = lds + place * S::STAGE;
      const _Float16* bp = s + S::PA;
      place = place + 1 == NST ? 0 : place + 1;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        f16x8 fa[2][NI], fb[2][NJ];
#pragma unroll
        for (int pl = 0; pl < 2; ++pl) {
          const int ch = ((4 * pl + 2 * kk + h) ^ turn) * 8;
#pragma unroll
          for (int i = 0; i < NI; ++i) fa[pl][i] = *(const f16x8*)(s + arow + 64 * i * NS_BK + ch);
#pragma unroll
          for (int i = 0; i < NJ; ++i) {
            if constexpr (!NN) fb[pl][i] = *(const f16x8*)(bp + brow + 64 * i * NS_BK + ch);
            else {
              f16x4 u[2];
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const int r = 16 * kk + tk + 4 * half, c = (wc / 32 + i) * 8 + 4 * pl + (tc >> 3);
                const _Float16* q = bp + r * 2 * S::C + (c ^ (((r & 3) << 2) | ((r >> 2) & 3))) * 8 + (tc & 4);
                u[half] = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)q));
              }
              fb[pl][i] = __builtin_shufflevector(u[0], u[1], 0, 1, 2, 3, 4, 5, 6, 7);
            }
          }
        }
#pragma unroll
        for (int pr = 0; pr < 3; ++pr) {
#pragma unroll
          for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j) acc[i][j] = MFMA16(fa[pr == 0][i], fb[pr == 1][j], acc[i][j]);
        }
      }
    }
  } else {
    // Half a step's fragments are read while the half before is multiplied; the barrier, in the middle of a step, is where the
    // next one has landed and the place of the last one is free.
    if (steps >= NST - 1) ns_wait<LOADS * (NST - 2)>();
    else ns_wait<0>();
    Frags f = read(0, 0);
    for (int k = 0; k < steps; ++k) {
      const Frags g = read(place, 1);
      multiply(f);
      if (k + 1 < steps) {
        if (k + NST - 1 <= steps) ns_wait<LOADS * (NST - 3)>();
        else ns_wait<0>();
        if (k + NST - 1 < steps) stage(k + NST - 1, place == 0 ? NST - 1 : place - 1);
        place = place + 1 == NST ? 0 : place + 1;
        f = read(place, 0);
      }
      multiply(g);
    }
  }
}

// tile of the lower triangle, row by row
__device__ __forceinline__ void tri(int id, int& ti, int& tj) {
  ti = (int)((sqrtf(8.f * id + 1.f) - 1.f) * 0.5f);
  while ((ti + 1) * (ti + 2) / 2 <= id) ++ti;
  while (ti * (ti + 1) / 2 > id) --ti;
  tj = id - ti * (ti + 1) / 2;
}

// tiles of S that meet the lower triangle, row by row
template <class S>
__device__ __forceinline__ void tri_tile(int id, int& ti, int& tj) {
  constexpr int W = S::R / S::C;
  tri(id / W, ti, tj);       // row ti has W (ti + 1) of them
  tj = W * tj + id % W;
}
template <class S>
__host__ __device__ inline int tri_tiles(int mp) { return mp / S::R * (mp / S::R + 1) / 2 * (S::R / S::C); }

// partials of X X^T (square = false) or A A over a share of K, lower tiles; the workgroups of an XCD (every eighth) take the
// same share, whose rows so stay in its L2
template <class S>
__global__ __launch_bounds__(512, 2) void ns_gram(const NsArgs p, int buf, bool square) {
  extern __shared__ __align__(16) _Float16 lds[];
  const int i = ns_find(p, blockIdx.x);
  const NsMat& q = p.mat[i];
  const int splits = square ? q.asplits : q.splits, id = blockIdx.x - p.pre[i], K = square ? q.mp : q.np;
  const int tiles = tri_tiles<S>(q.mp), sp = (id >> 3) / tiles * 8 + (id & 7);
  if (sp >= splits) return;
  int ti, tj;
  tri_tile<S>((id >> 3) % tiles, ti, tj);
  const int steps = K / NS_BK, per = (steps + splits - 1) / splits;
  const _Float16* x = square ? (const _Float16*)(p.ws + q.off_a) : (const _Float16*)(p.ws + q.off_x) + (long)buf * 2 * q.mp * K;
  typename S::Acc acc;
  ns_tile<false, S>(x, K, x, K, ti * S::R, tj * S::C, min(steps, sp * per) * NS_BK, min(steps, (sp + 1) * per) * NS_BK, lds, acc);
  float* out = (float*)(p.ws + q.off_p) + (long)sp * q.mp * q.mp;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / S::WC * 32 * S::NI, wc = wave % S::WC * 32 * S::NJ;
#pragma unroll
  for (int a = 0; a < S::NI; ++a)
#pragma unroll
    for (int b = 0; b < S::NJ; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        out[(long)(ti * S::R + wr + a * 32 + c_row(r, lane >> 5)) * q.mp + tj * S::C + wc + b * 32 + (lane & 31)] = acc[a][b][r];
}

// the partials of a 32 x 32 block of the lower tiles summed in order (four elements a thread, eight loads in flight), and A
// (square = false) or W = a I + b A + c A A written, both triangles' planes
__global__ __launch_bounds__(256) void ns_join(const NsArgs p, bool square) {
  const int i = ns_find(p, blockIdx.x);
  const NsMat& q = p.mat[i];
  __shared__ float tile[32][33];
  int ti, tj;
  tri(blockIdx.x - p.pre[i], ti, tj);
  const long plane = (long)q.mp * q.mp;
  const _Float16* A = (const _Float16*)(p.ws + q.off_a);
  _Float16* out = (_Float16*)(p.ws + q.off_a) + (square ? 2 * plane : 0);
  const int splits = square ? q.asplits : q.splits;
  const int r = threadIdx.x >> 3, c4 = (threadIdx.x & 7) * 4;
  const float* in = (const float*)(p.ws + q.off_p) + (long)(ti * 32 + r) * q.mp + tj * 32 + c4;
  f32x4 v = 0.f;
  int s = 0;
  for (; s + 8 <= splits; s += 8) {
    f32x4 u[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) u[k] = *(const f32x4*)(in + (s + k) * plane);
#pragma unroll
    for (int k = 0; k < 8; ++k) v += u[k];
  }
  for (; s < splits; ++s) v += *(const f32x4*)(in + s * plane);
  if (square) {
    const _Float16* o = A + at(ti * 32 + r, tj * 32 + c4, q.mp);
    const f32x4 av = __builtin_convertvector(*(const f16x4*)o, f32x4) + __builtin_convertvector(*(const f16x4*)(o + 32), f32x4);
    v = p.b * av + (p.c / SA) * v;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (ti * 32 + r == tj * 32 + c4 + k) v[k] += p.a * SA;
  } else {
    v *= SA / (SX * SX);
  }
  const auto put = [&](int row, int col, const f32x4& x) {
    f16x4 hi, lo;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      _Float16 a, b;
      split16(x[k], a, b);
      hi[k] = a;
      lo[k] = b;
    }
    *(f16x4*)(out + at(row, col, q.mp)) = hi;
    *(f16x4*)(out + at(row, col, q.mp) + 32) = lo;
  };
  put(ti * 32 + r, tj * 32 + c4, v);
  if (ti == tj) return;      // the whole block: it is symmetric by itself
#pragma unroll
  for (int k = 0; k < 4; ++k) tile[c4 + k][r] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = tile[r][c4 + k];
  put(tj * 32 + r, ti * 32 + c4, v);
}

// X' = W X; the last step writes the result in its own type and orientation.  An XCD takes every eighth panel of columns, with
// all row tiles of one together.
template <class S>
__global__ __launch_bounds__(512, 2) void ns_apply(const NsArgs p, int buf, int last) {
  extern __shared__ __align__(16) _Float16 lds[];
  constexpr int NI = S::NI, NJ = S::NJ;
  const int i = ns_find(p, blockIdx.x);
  const NsMat& q = p.mat[i];
  const int id = blockIdx.x - p.pre[i], mt = q.mp / S::R, r0 = (id >> 3) % mt * S::R, c0 = ((id >> 3) / mt * 8 + (id & 7)) * S::C;
  if (c0 >= q.np) return;
  const _Float16* W = (const _Float16*)(p.ws + q.off_a) + 2 * (long)q.mp * q.mp;
  const _Float16* x = (const _Float16*)(p.ws + q.off_x) + (long)buf * 2 * q.mp * q.np;
  _Float16* y = (_Float16*)(p.ws + q.off_x) + (long)(buf ^ 1) * 2 * q.mp * q.np;
  typename S::Acc acc;
  ns_tile<true, S>(W, q.mp, x, q.np, r0, c0, 0, q.mp, lds, acc);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / S::WC * 32 * NI, wc = wave % S::WC * 32 * NJ;
  const bool tall = q.rows > q.cols;
  if (last) {
#pragma unroll
    for (int a = 0; a < NI; ++a)
#pragma unroll
      for (int b = 0; b < NJ; ++b) {
        const int c = c0 + wc + b * 32 + (lane & 31);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = r0 + wr + a * 32 + c_row(r, lane >> 5);
          if (row < q.m && c < q.n) ns_store(q, tall ? c : row, tall ? row : c, acc[a][b][r] * (1.f / (SA * SX)));
        }
      }
    return;
  }
  // the planes go out through LDS, 128 rows at a time, 16 bytes a lane along a row
  constexpr int LD = S::C + 8, PL = 128 * LD, CPR = S::C / 8;
  static_assert(128 % (32 * NI) == 0, "a wave's rows lie in one pass");
#pragma unroll
  for (int pass = 0; pass < S::R / 128; ++pass) {
    __syncthreads();
    if (wr / 128 == pass) {
#pragma unroll
      for (int a = 0; a < NI; ++a)
#pragma unroll
        for (int b = 0; b < NJ; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int o = (wr % 128 + a * 32 + c_row(r, lane >> 5)) * LD + wc + b * 32 + (lane & 31);
            split16(acc[a][b][r] * (1.f / SA), lds[o], lds[PL + o]);
          }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2 * 128 * CPR / 512; ++k) {
      const int e = threadIdx.x + k * 512, c = e % CPR, row = e / CPR % 128, pl = e / CPR / 128;
      *(f16x8*)(y + at(r0 + pass * 128 + row, c0 + c * 8, q.np) + pl * 32) = *(const f16x8*)(lds + pl * PL + row * LD + c * 8);
    }
  }
}

// ------------------------------------------------------------------------------------------------ small matrices
// One workgroup of eight waves holds a matrix: X's planes, and A's (W's after it, in the same place), stay in LDS for all
// steps, so a list of encoder matrices is one launch.  Bound by the latency of a chain, not by a rate: of a step's phases (A, A A,
// W X and the planes' stores) each waits for the last, six barriers a step up to 64 rows and five above, and A A's one tile of
// 32 rows keeps one wave of the eight busy: 36 us for five steps of twelve matrices of 32 x 32 to 384 x 32, one compute unit each
// (over 1 us a barrier, so it is not the barriers alone; the phases were not timed apart).
struct NsSmallArgs {
  float a, b, c, eps;
  int steps;
  NsMat mat[NS_MAXMAT];
};

constexpr int ns_small_splits(int mt) { return mt == 1 ? 8 : mt == 2 ? 2 : 1; }      // of the Gram matrix's columns
inline size_t ns_small_lds(int mp, int np) {
  const int mt = mp / 32, sp = ns_small_splits(mt);
  return (size_t)4 * mp * (np + 8) + (size_t)4 * mp * (mp + 8) + (sp > 1 ? (size_t)sp * mt * mt * 4096 : 0);
}
inline bool ns_is_small(int mp, int np) {
  return mp / 32 <= 4 && (mp / 32) * (np / 32) <= 32 && ns_small_lds(mp, np) <= NS_SMALL_LDS;
}

// a 32 x 32 tile of a product over [k0, k1): rows of A, and rows (NT) or columns (NN) of B; every operand two planes
template <bool NN>
__device__ __forceinline__ f32x16 small_tile(const _Float16* Ah, const _Float16* Al, int lda, int r0, const _Float16* Bh,
                                             const _Float16* Bl, int ldb, int c0, int k0, int k1, int lane) {
  f32x16 acc = 0.f;
#pragma unroll 2
  for (int k = k0; k < k1; k += 16) {
    const f16x8 ah = NN ? frag_kp(Ah, lda, r0, k, lane) : frag_k(Ah, lda, r0, k, lane),
                al = NN ? frag_kp(Al, lda, r0, k, lane) : frag_k(Al, lda, r0, k, lane);
    const f16x8 bh = NN ? frag_t(Bh, ldb, k, c0, lane) : frag_k(Bh, ldb, c0, k, lane),
                bl = NN ? frag_t(Bl, ldb, k, c0, lane) : frag_k(Bl, ldb, c0, k, lane);
    acc = MFMA16(al, bh, acc);
    acc = MFMA16(ah, bl, acc);
    acc = MFMA16(ah, bh, acc);
  }
  return acc;
}

template <typename T, int MT>
__device__ __forceinline__ void ns_small_run(const NsSmallArgs& p, const NsMat& q, _Float16* lds, double* red) {
  constexpr int MP = 32 * MT, LDA = MP + 8, SPLITS = ns_small_splits(MT), UNITS = MT * MT * SPLITS, NA = (MT * MT + 7) / 8;
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int np = q.np, ldx = np + 8, nt = np / 32;
  _Float16 *Xh = lds, *Xl = Xh + MP * ldx, *Ah = Xl + MP * ldx, *Al = Ah + MP * LDA;
  float* part = (float*)(Al + MP * LDA);
  const bool tall = q.rows > q.cols;
  const T* src = (const T*)q.src;
  // the whole matrix in registers (at most 64 elements a thread), all loads in flight at once; e / cols is the upper half of
  // e ceil(2^32 / cols), exact for e cols < 2^32
  const int total = q.rows * q.cols;
  const uint32_t magic = q.cols == 1 ? 0 : (uint32_t)((0x100000000ull + q.cols - 1) / q.cols);
  const auto row_of = [&](int e) { return q.cols == 1 ? e : (int)__umulhi((uint32_t)e, magic); };
  float g[64];
#pragma unroll
  for (int k = 0; k < 64; ++k) {
    const int e = t + 512 * k, r = row_of(e);
    g[k] = e < total ? (float)src[(long)r * q.ld_src + (e - r * q.cols)] : 0.f;
  }
  for (int e = t * 8; e < 2 * MP * ldx; e += 4096) *(f16x8*)(Xh + e) = f16x8{};      // what stands beside it in the planes
  double s = 0.;
#pragma unroll
  for (int k = 0; k < 64; ++k) s = fma((double)g[k], (double)g[k], s);
  const float scale = (float)(SX / (sqrt(block_sum64(s, red)) + (double)p.eps));
#pragma unroll
  for (int k = 0; k < 64; ++k) {
    const int e = t + 512 * k, r = row_of(e), c = e - r * q.cols, o = tall ? c * ldx + r : r * ldx + c;
    if (e < total) split16(g[k] * scale, Xh[o], Xl[o]);
  }
  __syncthreads();
  int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int step = 0; step < p.steps; ++step) {
    asm volatile("" : "+v"(lane));       // else every address of the loop is kept in a register, and those in scratch
    const int h = lane >> 5;
    // A = X X^T: a wave takes (tile, share of the columns) units
#pragma unroll 1
    for (int u = wave; u < UNITS; u += 8) {
      const int tile = u / SPLITS, sp = u % SPLITS, ti = tile / MT, tj = tile % MT;
      const int chunks = np / 16, per = (chunks + SPLITS - 1) / SPLITS;
      const f32x16 acc = small_tile<false>(Xh, Xl, ldx, ti * 32, Xh, Xl, ldx, tj * 32, min(chunks, sp * per) * 16,
                                           min(chunks, (sp + 1) * per) * 16, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = c_row(r, h), c = lane & 31;
        if constexpr (SPLITS > 1) part[u * 1024 + row * 32 + c] = acc[r];
        else {
          const int o = (ti * 32 + row) * LDA + tj * 32 + c;
          split16(acc[r] * (SA / (SX * SX)), Ah[o], Al[o]);
        }
      }
    }
    __syncthreads();
    if constexpr (SPLITS > 1) {
      for (int i = t; i < MT * MT * 1024; i += 512) {
        const int tile = i >> 10, e = i & 1023;
        float v = 0.f;
#pragma unroll
        for (int sp = 0; sp < SPLITS; ++sp) v += part[(tile * SPLITS + sp) * 1024 + e];
        const int o = (tile / MT * 32 + (e >> 5)) * LDA + tile % MT * 32 + (e & 31);
        split16(v * (SA / (SX * SX)), Ah[o], Al[o]);
      }
      __syncthreads();
    }
    // W = a I + b A + c A A, into A's place once all have read it
    f32x16 w[NA];
#pragma unroll
    for (int j = 0; j < NA; ++j) {
      const int tile = wave + 8 * j;
      if (tile >= MT * MT) continue;
      const int ti = tile / MT, tj = tile % MT;
      w[j] = small_tile<false>(Ah, Al, LDA, ti * 32, Ah, Al, LDA, tj * 32, 0, MP, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = ti * 32 + c_row(r, h), c = tj * 32 + (lane & 31);
        const float av = (float)Ah[row * LDA + c] + (float)Al[row * LDA + c];
        w[j][r] = p.b * av + (p.c / SA) * w[j][r] + (row == c ? p.a * SA : 0.f);
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NA; ++j) {
      const int tile = wave + 8 * j;
      if (tile >= MT * MT) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int o = (tile / MT * 32 + c_row(r, h)) * LDA + tile % MT * 32 + (lane & 31);
        split16(w[j][r], Ah[o], Al[o]);
      }
    }
    __syncthreads();
    // X' = W X, up to four tiles a wave, written once all have read X
    f32x16 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int tile = wave + 8 * j;
      if (tile < MT * nt) x[j] = small_tile<true>(Ah, Al, LDA, tile % MT * 32, Xh, Xl, ldx, tile / MT * 32, 0, MP, lane);
    }
    __syncthreads();
    const bool last = step + 1 == p.steps;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int tile = wave + 8 * j;
      if (tile >= MT * nt) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = tile % MT * 32 + c_row(r, h), c = tile / MT * 32 + (lane & 31);
        const float v = x[j][r] * (1.f / SA);
        if (!last) split16(v, Xh[row * ldx + c], Xl[row * ldx + c]);
        else if (row < q.m && c < q.n) ((T*)q.dst)[tall ? (long)c * q.ld_dst + row : (long)row * q.ld_dst + c] = (T)(v * (1.f / SX));
      }
    }
    __syncthreads();
  }
}

template <typename T>
__global__ __launch_bounds__(512, 2) void ns_small(const NsSmallArgs p) {
  extern __shared__ __align__(16) _Float16 lds[];
  __shared__ double red[8];
  const NsMat& q = p.mat[blockIdx.x];
  switch (q.mp / 32) {
    case 1: ns_small_run<T, 1>(p, q, lds, red); break;
    case 2: ns_small_run<T, 2>(p, q, lds, red); break;
    case 3: ns_small_run<T, 3>(p, q, lds, red); break;
    default: ns_small_run<T, 4>(p, q, lds, red); break;
  }
}

// ------------------------------------------------------------------------------------------------ the update around it
constexpr int MUON_MAXMAT = 64;
struct MuonArgs {
  const float* coef;       // the clip's multiplier of the gradients, on the device
  float mu, lr, decay;
  int nesterov;
  ctr_muon_mat_t mat[MUON_MAXMAT];
};
// buf = mu buf + coef g;  u = coef g + mu buf (Nesterov) or buf
__global__ __launch_bounds__(256) void muon_momentum(const MuonArgs a) {
  const ctr_muon_mat_t& q = a.mat[blockIdx.y];
  const float c = *a.coef;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < q.n; i += (long)gridDim.x * 256) {
    const float g = c * q.g[i], b = fmaf(a.mu, q.buf[i], g);
    q.buf[i] = b;
    q.u[i] = a.nesterov ? fmaf(a.mu, b, g) : b;
  }
}
// p = (1 - lr decay) p - lr scale u
__global__ __launch_bounds__(256) void muon_apply(const MuonArgs a) {
  const ctr_muon_mat_t& q = a.mat[blockIdx.y];
  const float keep = 1.f - a.lr * a.decay, f = -a.lr * q.scale;
  for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < q.n; i += (long)gridDim.x * 256) q.p[i] = fmaf(f, q.u[i], keep * q.p[i]);
}

// ------------------------------------------------------------------------------------------------ host side
// Layout of a matrix of the large form in the workspace; returns the bytes used.
size_t ns_layout(NsMat& q, size_t off) {
  const auto take = [&](size_t n) { const size_t o = off; off = (off + n + 255) / 256 * 256; return (long)o; };
  q.off_x = take((size_t)8 * q.mp * q.np);         // two buffers of two planes
  q.off_a = take((size_t)8 * q.mp * q.mp);         // A and W
  q.off_p = take((size_t)4 * std::max(q.splits, q.asplits) * q.mp * q.mp);
  q.off_s = take((size_t)8 * NS_SUMSQ_BLOCKS);
  return off;
}

void ns_dims(NsMat& q, const ctr_ns_mat_t& g, int type) {
  q = NsMat{};
  q.src = g.src;
  q.dst = g.dst;
  q.ld_src = g.ld_src;
  q.ld_dst = g.ld_dst;
  q.rows = g.rows;
  q.cols = g.cols;
  q.type = type;
  q.m = std::min(g.rows, g.cols);
  q.n = std::max(g.rows, g.cols);
  q.mp = cdiv(q.m, 32) * 32;
  q.np = cdiv(q.n, 32) * 32;
}

// Shares of K of a symmetric product: as many as give every compute unit a workgroup, a whole number of times as nearly as may
// be, each with at least four K steps; a share costs its partial sums, written and read once.
int ns_splits(int tiles, int K) {
  const int most = std::max(1, std::min(K / (4 * NS_BK), 32));
  int best = 1;
  double cost = 1e30;
  for (int s = 1; s <= most; ++s) {
    const double c = (double)cdiv((long)tiles * s, 256) / s * 256. / tiles + 0.02 * s;
    if (c < cost) cost = c, best = s;
  }
  return best;
}

bool ns_large_dims(NsMat& q) {
  if (ns_is_small(q.mp, q.np)) return false;
  // 256 x 256 tiles where they are three for every four compute units or more
  q.group = q.m <= 768 ? 0 : (long)cdiv(q.m, 256) * cdiv(q.n, 256) < 192 ? 1 : 2;
  const int r = q.group ? 256 : 128, c = q.group == 2 ? 256 : 128;
  q.mp = cdiv(q.m, r) * r;
  q.np = std::max(cdiv(q.n, c) * c, q.mp);
  const int tiles = q.group ? tri_tiles<NsMid>(q.mp) : tri_tiles<NsSmall>(q.mp);
  q.splits = ns_splits(tiles, q.np);
  q.asplits = ns_splits(tiles, q.mp);
  return true;
}

// The largest singular value r that X can reach, and W: with u the square of one, W's is p(u) = a + b u + c u^2 and X's next
// sqrt(u) p(u); over [0, r^2] both are largest at an end or where 2 c u + b = 0, 5 c u^2 + 3 b u + a = 0.
bool ns_in_range(int steps, double a, double b, double c) {
  if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
  const auto p = [=](double u) { return std::fabs(a + u * (b + u * c)); };
  double at[5] = {0., 0., -1., -1., -1.};
  if (c != 0.) {
    at[2] = -b / (2. * c);
    const double d = 9. * b * b - 20. * a * c;
    if (d >= 0.) {
      const double q = -0.5 * (3. * b + std::copysign(std::sqrt(d), b));      // the roots q / (5 c) and a / q, without cancelling
      at[3] = q / (5. * c);
      if (q != 0.) at[4] = a / q;
    }
  } else if (b != 0.) at[3] = -a / (3. * b);
  double r = 1.;
  for (int s = 0; s < steps; ++s) {
    at[1] = r * r;
    double w = 0., next = 0.;
    for (const double u : at) {
      if (!(u >= 0. && u <= r * r)) continue;
      w = std::max(w, p(u));
      next = std::max(next, std::sqrt(u) * p(u));
    }
    if (!(w <= 32.) || !(next <= 7.5)) return false;
    r = next * 1.001;
  }
  return true;
}

// the kernels' LDS beyond 64 KB, once for each device
bool ns_allow_lds() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load() & bit) return true;
  const auto allow = [](const void* f, int n) {
    return hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, n) == hipSuccess;
  };
  if (!allow((const void*)ns_gram<NsSmall>, NsSmall::LDS) || !allow((const void*)ns_apply<NsSmall>, NsSmall::LDS) ||
      !allow((const void*)ns_gram<NsMid>, NsMid::LDS) || !allow((const void*)ns_apply<NsMid>, NsMid::LDS) ||
      !allow((const void*)ns_apply<NsLarge>, NsLarge::LDS) ||
      !allow((const void*)ns_small<float>, NS_SMALL_LDS) ||
      !allow((const void*)ns_small<__bf16>, NS_SMALL_LDS) || !allow((const void*)ns_small<_Float16>, NS_SMALL_LDS))
    return false;
  done.fetch_or(bit);
  return true;
}

}  // namespace
}  // namespace ctr

using namespace ctr;

extern "C" size_t ctr_newton_schulz_ws_size(const ctr_ns_mat_t* mats, int count) {
  size_t most = 0, off[NS_GROUPS] = {};
  int in[NS_GROUPS] = {};
  for (int i = 0; mats && i < count; ++i) {
    if (mats[i].rows <= 0 || mats[i].cols <= 0) continue;
    NsMat q;
    ns_dims(q, mats[i], 0);
    if (!ns_large_dims(q)) continue;
    const int g = q.group;
    if (in[g] == NS_MAXMAT) in[g] = 0, off[g] = 0;
    off[g] = ns_layout(q, off[g]);
    ++in[g];
    most = std::max(most, off[g]);
  }
  return most;
}

extern "C" int ctr_newton_schulz(const ctr_ns_mat_t* mats, int count, int steps, float a, float b, float c, float eps,
                                 int type, void* ws, size_t ws_bytes, void* stream) {
  CTR_REQUIRE(count >= 0 && (count == 0 || mats), "matrix list");
  CTR_REQUIRE(type >= TY_F32 && type <= TY_F16, "type (0 fp32, 1 bf16, 2 fp16)");
  CTR_REQUIRE(steps >= 1 && steps <= 64, "steps in [1, 64]");
  CTR_REQUIRE(eps >= 0.f && std::isfinite(eps), "eps");
  CTR_REQUIRE(ns_in_range(steps, a, b, c), "coefficients: a singular value could pass 7.5, or one of a I + b A + c A^2 32");
  for (int i = 0; i < count; ++i) {
    const ctr_ns_mat_t& g = mats[i];
    CTR_REQUIRE(g.rows >= 0 && g.cols >= 0 && g.rows <= 65536 && g.cols <= 65536, "matrix sides in [0, 65536]");
    if (g.rows == 0 || g.cols == 0) continue;
    CTR_REQUIRE(g.src && g.dst, "null matrix");
    CTR_REQUIRE((g.rows == 1 || g.ld_src >= g.cols) && (g.rows == 1 || g.ld_dst >= g.cols), "row strides");
  }
  CTR_REQUIRE(ws_bytes >= ctr_newton_schulz_ws_size(mats, count), "workspace too small");
  hipStream_t s = (hipStream_t)stream;

  bool any = false;
  for (int i = 0; i < count; ++i) any |= mats[i].rows > 0 && mats[i].cols > 0;
  if (!any) return 0;
  CTR_REQUIRE(ns_allow_lds(), "LDS size attribute");
  NsSmallArgs small = {a, b, c, eps, steps, {}};
  int ns = 0;
  size_t small_lds = 0;
  const auto flush_small = [&] {
    if (ns && type == TY_F32) ns_small<float><<<ns, 512, small_lds, s>>>(small);
    else if (ns && type == TY_BF16) ns_small<__bf16><<<ns, 512, small_lds, s>>>(small);
    else if (ns) ns_small<_Float16><<<ns, 512, small_lds, s>>>(small);
    ns = 0;
    small_lds = 0;
  };
  NsArgs large[NS_GROUPS] = {};
  size_t off[NS_GROUPS] = {};
  for (NsArgs& g : large) {
    g.ws = (char*)ws;
    g.a = a;
    g.b = b;
    g.c = c;
    g.eps = eps;
  }
  const auto flush_large = [&](int w) {
    NsArgs& g = large[w];
    if (g.count == 0) return;
    const auto prefix = [&](auto blocks) {
      int n = 0;
      for (int i = 0; i < g.count; ++i) {
        g.pre[i] = n;
        n += blocks(g.mat[i]);
      }
      g.pre[g.count] = n;
      return n;
    };
    ns_sumsq<<<dim3(NS_SUMSQ_BLOCKS, g.count), 256, 0, s>>>(g);
    const int ni = prefix([](const NsMat& q) { return q.mp / 64 * (q.np / 64); });
    ns_init<<<ni, 256, 0, s>>>(g);
    for (int k = 0; k < steps; ++k) {
      for (int square = 0; square < 2; ++square) {
        const int ng = prefix([&](const NsMat& q) { return cdiv(square ? q.asplits : q.splits, 8) * 8 * (w ? tri_tiles<NsMid>(q.mp) : tri_tiles<NsSmall>(q.mp)); });
        if (w) ns_gram<NsMid><<<ng, 512, NsMid::LDS, s>>>(g, k & 1, square);
        else ns_gram<NsSmall><<<ng, 512, NsSmall::LDS, s>>>(g, k & 1, square);
        const int nj = prefix([](const NsMat& q) { return (q.mp / 32) * (q.mp / 32 + 1) / 2; });
        ns_join<<<nj, 256, 0, s>>>(g, square);
      }
      const int tr = w ? 256 : 128, tc = w == 2 ? 256 : 128;
      const int na = prefix([&](const NsMat& q) { return q.mp / tr * (cdiv(q.np / tc, 8) * 8); });
      if (w == 2) ns_apply<NsLarge><<<na, 512, NsLarge::LDS, s>>>(g, k & 1, k + 1 == steps);
      else if (w) ns_apply<NsMid><<<na, 512, NsMid::LDS, s>>>(g, k & 1, k + 1 == steps);
      else ns_apply<NsSmall><<<na, 512, NsSmall::LDS, s>>>(g, k & 1, k + 1 == steps);
    }
    g.count = 0;
    off[w] = 0;
  };
  for (int i = 0; i < count; ++i) {
    if (mats[i].rows == 0 || mats[i].cols == 0) continue;
    NsMat q;
    ns_dims(q, mats[i], type);
    if (ns_large_dims(q)) {
      const int w = q.group;
      if (large[w].count == NS_MAXMAT) flush_large(w);
      off[w] = ns_layout(q, off[w]);
      large[w].mat[large[w].count++] = q;
    } else {
      if (ns == NS_MAXMAT) flush_small();
      small_lds = std::max(small_lds, ns_small_lds(q.mp, q.np));
      small.mat[ns++] = q;
    }
  }
  flush_small();
  for (int w = 0; w < NS_GROUPS; ++w) flush_large(w);
  return check_launch("newton_schulz");
}

extern "C" int ctr_muon_update(const ctr_muon_mat_t* mats, int count, int apply, const float* coef, float mu, int nesterov, float lr,
                               float weight_decay, void* stream) {
  CTR_REQUIRE(count >= 0 && (count == 0 || mats), "matrix list");
  CTR_REQUIRE(apply || coef, "null coefficient");
  MuonArgs a = {coef, mu, lr, weight_decay, nesterov, {}};
  for (int i = 0; i < count; i += MUON_MAXMAT) {
    const int n = std::min(MUON_MAXMAT, count - i);
    long most = 0;
    for (int k = 0; k < n; ++k) {
      a.mat[k] = mats[i + k];
      CTR_REQUIRE(a.mat[k].n >= 0 && a.mat[k].u && (apply ? (bool)a.mat[k].p : a.mat[k].g && a.mat[k].buf), "null matrix");
      most = std::max(most, a.mat[k].n);
    }
    const dim3 grid(std::max(1, std::min(256, cdiv(most, 1024))), n);
    if (apply) muon_apply<<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else muon_momentum<<<grid, 256, 0, (hipStream_t)stream>>>(a);
  }
  return check_launch("muon_update");
}
