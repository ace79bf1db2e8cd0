// Layer norm over rows of fp32 / bf16 / fp16, forward and backward, with the weight and bias gradients reduced:
//   y = (x - mean) rstd w + b,   rstd = 1 / sqrt(var + eps),   xhat = (x - mean) rstd,   g = dy w
//   dx = rstd (g - mean_n(g) - xhat mean_n(g xhat)),   dw = sum_m dy xhat,   db = sum_m dy
// Statistics, sums and partial gradients are fp32 whatever the rows' type; the variance is of the centred values, which
// stay in registers, so no E[x^2] - mean^2 cancels.  Bound by HBM: the forward pass reads x and writes y, the backward
// reads x and dy and writes dx, each once up to 16384 columns (wider rows are read again for each sum).  The backward also writes
// and reads 16 N bytes a workgroup of partial weight gradients: nothing beside many rows, but more than the rows themselves
// where wide rows are few (1024 x 4096 bf16: 67 MB written and read beside 25).
//
// TPR threads own a row, thread t its 8-element vectors t, t + TPR, ... (V of them): 16 bytes a lane for the 16-bit
// types, at whatever alignment the row has (a row of odd width starts at any element).  TPR is the smallest of
// 4 .. 64 that covers the row with one vector, then a wave with up to four, then a block: a narrow row never idles
// a wave and a wide one never spills.  Rows beyond 16384 elements stream (ln_*_wide).
// Measured: 32768 x 4096 bf16 forward 134 us (4.0 TB/s), backward with the join 168 us (4.8 TB/s), a large copy reaching 4.65;
// 245760 x 32 bf16 9 and 13 + 4 us (3.5 and 3.6 TB/s); 4099 x 1001 fp16, every row at another alignment, 7.2 us (2.3 TB/s).
// Small calls (64 x 256: forward and backward in two launches, 23 us) are bound by the host.
// Weight gradients: a thread keeps its columns' sums over all rows of its block in registers, the block joins its
// row groups in a fixed order and writes one partial row, ln_reduce adds the partial rows in a fixed order: no atomics,
// the same bits every time.
#include <algorithm>

#include "ctr_hip.h"
#include "vec16.h"

namespace ctr {
namespace {

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (TPR <= 64) return group_sum<TPR>(v);
  else return block_sum(v, red);
}

// b may be null
template <typename T, typename W, int TPR, int V>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_fwd(const T* __restrict__ x, long ldx, long M, int N,
                                                                const W* __restrict__ w, const W* __restrict__ b,
                                                                float eps, T* __restrict__ y, long ldy,
                                                                float* __restrict__ mean, float* __restrict__ rstd) {
  constexpr int BT = TPR > 256 ? TPR : 256, RPB = BT / TPR;
  __shared__ float red[BT / 64];
  const int t = threadIdx.x % TPR;
  const float inv_n = 1.0f / (float)N;
  for (long m = (long)blockIdx.x * RPB + threadIdx.x / TPR; m < M; m += (long)gridDim.x * RPB) {
    f32x8 v[V];
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * TPR + t) * 8;
      v[k] = ld8f(x + m * ldx + c, N - c);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[k][i];
    }
    const float mu = row_sum<TPR>(s, red) * inv_n;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * TPR + t) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[k][i] -= mu;
        q = fmaf(c + i < N ? v[k][i] : 0.f, v[k][i], q);
      }
    }
    const float rs = 1.0f / sqrtf(row_sum<TPR>(q, red) * inv_n + eps);
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * TPR + t) * 8;
      if (c >= N) continue;
      const f32x8 wv = ld8f(w + c, N - c);
      f32x8 o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = v[k][i] * rs * wv[i];
      if (b) o += ld8f(b + c, N - c);
      st8f(y + m * ldy + c, o, N - c);
    }
    if (t == 0) {
      mean[m] = mu;
      rstd[m] = rs;
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_fwd_wide(const T* __restrict__ x, long ldx, long M, int N,
                                                    const W* __restrict__ w, const W* __restrict__ b, float eps,
                                                    T* __restrict__ y, long ldy, float* __restrict__ mean,
                                                    float* __restrict__ rstd) {
  __shared__ float red[16];
  const float inv_n = 1.0f / (float)N;
  for (long m = blockIdx.x; m < M; m += gridDim.x) {
    const T* r = x + m * ldx;
    float s = 0.f;
    for (long c = threadIdx.x * 8L; c < N; c += 8192) {
      const f32x8 v = ld8f(r + c, (int)(N - c));
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
    const float mu = block_sum(s, red) * inv_n;
    float q = 0.f;
    for (long c = threadIdx.x * 8L; c < N; c += 8192) {
      const f32x8 v = ld8f(r + c, (int)(N - c));
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = c + i < N ? v[i] - mu : 0.f;
        q = fmaf(d, d, q);
      }
    }
    const float rs = 1.0f / sqrtf(block_sum(q, red) * inv_n + eps);
    for (long c = threadIdx.x * 8L; c < N; c += 8192) {
      const int n = (int)(N - c);
      f32x8 o = (ld8f(r + c, n) - mu) * rs * ld8f(w + c, n);
      if (b) o += ld8f(b + c, n);
      st8f(y + m * ldy + c, o, n);
    }
    if (threadIdx.x == 0) {
      mean[m] = mu;
      rstd[m] = rs;
    }
  }
}

// part: (2, nb, N) fp32 partial rows of dw and db; dw_out != null (one block): the gradients themselves
template <typename T, typename W, int TPR, int V>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void ln_bwd(const T* __restrict__ dy, long lddy,
                                                                const T* __restrict__ x, long ldx,
                                                                const float* __restrict__ mean,
                                                                const float* __restrict__ rstd,
                                                                const W* __restrict__ w, long M, int N,
                                                                T* __restrict__ dx, long lddx, float* __restrict__ part,
                                                                W* __restrict__ dw_out, W* __restrict__ db_out) {
  constexpr int BT = TPR > 256 ? TPR : 256, RPB = BT / TPR, NW = BT / 64;
  __shared__ float red[NW];
  const int t = threadIdx.x % TPR;
  const float inv_n = 1.0f / (float)N;
  f32x8 wv[V], aw[V], ab[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int c = (k * TPR + t) * 8;
    wv[k] = ld8f(w + c, N - c);
    aw[k] = 0.f;
    ab[k] = 0.f;
  }
  for (long m = (long)blockIdx.x * RPB + threadIdx.x / TPR; m < M; m += (long)gridDim.x * RPB) {
    const float rs = rstd[m], mu = mean[m];
    f32x8 g[V], xh[V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * TPR + t) * 8;
      xh[k] = ld8f(x + m * ldx + c, N - c);
      g[k] = ld8f(dy + m * lddy + c, N - c);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * TPR + t) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        xh[k][i] = c + i < N ? (xh[k][i] - mu) * rs : 0.f;
        aw[k][i] = fmaf(g[k][i], xh[k][i], aw[k][i]);
        ab[k][i] += g[k][i];
        g[k][i] *= wv[k][i];
        s1 = fmaf(g[k][i], xh[k][i], s1);
        s2 += g[k][i];
      }
    }
    const float c1 = row_sum<TPR>(s1, red) * inv_n, c2 = row_sum<TPR>(s2, red) * inv_n;
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int c = (k * TPR + t) * 8;
      f32x8 o;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = rs * (g[k][i] - c2 - xh[k][i] * c1);
      if (c < N) st8f(dx + m * lddx + c, o, N - c);
    }
  }
  // join the block's row groups: lanes of a wave first, then the waves
  __shared__ float join[TPR <= 64 ? NW * TPR * V * 8 : 1];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    f32x8* a = which ? ab : aw;
    W* out = which ? db_out : dw_out;
    float* pr = part + ((long)which * gridDim.x + blockIdx.x) * N;
    if constexpr (TPR <= 64) {
      const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
      for (int k = 0; k < V; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float v = a[k][i];
#pragma unroll
          for (int o = TPR; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
          if (lane < TPR) join[wave * TPR * V * 8 + (k * TPR + t) * 8 + i] = v;
        }
      __syncthreads();
      for (int c = threadIdx.x; c < N; c += BT) {
        float v = 0.f;
#pragma unroll
        for (int j = 0; j < NW; ++j) v += join[j * TPR * V * 8 + c];
        if (dw_out) { if (out) out[c] = (W)v; }
        else pr[c] = v;
      }
      __syncthreads();
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int c = (k * TPR + t) * 8;
        if (c >= N) continue;
        if (dw_out) { if (out) st8f(out + c, a[k], N - c); }
        else st8f(pr + c, a[k], N - c);
      }
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(1024) void ln_bwd_wide(const T* __restrict__ dy, long lddy, const T* __restrict__ x,
                                                    long ldx, const float* __restrict__ mean,
                                                    const float* __restrict__ rstd, const W* __restrict__ w, long M,
                                                    int N, T* __restrict__ dx, long lddx) {
  __shared__ float red[16];
  const float inv_n = 1.0f / (float)N;
  for (long m = blockIdx.x; m < M; m += gridDim.x) {
    const float rs = rstd[m], mu = mean[m];
    float s1 = 0.f, s2 = 0.f;
    for (long c = threadIdx.x * 8L; c < N; c += 8192) {
      const int n = (int)(N - c);
      const f32x8 g = ld8f(dy + m * lddy + c, n) * ld8f(w + c, n), xh = (ld8f(x + m * ldx + c, n) - mu) * rs;
#pragma unroll
      for (int i = 0; i < 8; ++i) {      // g is 0 behind the row's end
        s1 = fmaf(g[i], xh[i], s1);
        s2 += g[i];
      }
    }
    const float c1 = block_sum(s1, red) * inv_n, c2 = block_sum(s2, red) * inv_n;
    for (long c = threadIdx.x * 8L; c < N; c += 8192) {
      const int n = (int)(N - c);
      const f32x8 g = ld8f(dy + m * lddy + c, n) * ld8f(w + c, n), xh = (ld8f(x + m * ldx + c, n) - mu) * rs;
      st8f(dx + m * lddx + c, rs * (g - c2 - xh * c1), n);
    }
  }
}

// the wide rows' weight gradients: block (j, p) takes 2048 columns of the rows p, p + np, ...
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_cols(const T* __restrict__ dy, long lddy, const T* __restrict__ x, long ldx,
                                                   const float* __restrict__ mean, const float* __restrict__ rstd, long M,
                                                   int N, float* __restrict__ part) {
  const long c = ((long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (c >= N) return;
  const int n = (int)(N - c);
  f32x8 aw = 0.f, ab = 0.f;
  for (long m = blockIdx.y; m < M; m += gridDim.y) {
    const f32x8 g = ld8f(dy + m * lddy + c, n);
    aw += g * ((ld8f(x + m * ldx + c, n) - mean[m]) * rstd[m]);
    ab += g;
  }
  st8f(part + (long)blockIdx.y * N + c, aw, n);
  st8f(part + ((long)gridDim.y + blockIdx.y) * N + c, ab, n);
}

// out[c] = sum_p part[p][c], 32 columns a block, the partial rows dealt over 32 threads each and joined in order
template <typename W>
__global__ __launch_bounds__(1024) void ln_reduce(const float* __restrict__ part, int np, int N, W* __restrict__ dw,
                                                  W* __restrict__ db) {
  __shared__ float s[32][33];
  const int cl = threadIdx.x & 31, r = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  W* out = blockIdx.y ? db : dw;
  if (!out) return;
  const float* p = part + (long)blockIdx.y * np * N;
  float v = 0.f;
  if (c < N) {
#pragma unroll 16                 // as many loads in flight
    for (int i = r; i < np; i += 32) v += p[(long)i * N + c];
  }
  s[r][cl] = v;
  __syncthreads();
  for (int o = 16; o > 0; o >>= 1) {
    if (r < o) s[r][cl] += s[r + o][cl];
    __syncthreads();
  }
  if (r == 0 && c < N) out[c] = (W)s[0][cl];
}

constexpr int LN_WIDE = 16384;

int ln_tpr(int N) {
  for (int t = 4; t < 64; t <<= 1)
    if (N <= t * 8) return t;
  return N <= 1024 ? 64 : N <= 8192 ? 256 : 1024;
}

// partial rows of the backward (= its blocks).  One block joins its own rows and writes the gradients itself.
int ln_parts(long M, int N) {
  if (N > LN_WIDE) return (int)std::min<long>(std::max<long>(M, 1), 64);
  const int tpr = ln_tpr(N), rpb = std::max(256, tpr) / tpr;
  // Rows in turn in one block, or a row at a time and a join.  The launch saved is 2.5 us of the host's (a call in a loop 12.7 us
  // against 15.2 at every size); the kernels alone take, in us, for 4 / 8 / 16 rows in turn (and with a join): 32 columns 6.7 / 9.0 /
  // 13.7 (6.9), 256: 6.0 / 8.8 / 14.4 (6.2), 512: 5.4 / 8.4 / 14.4 (5.6), 1024: 7.7 / 12.4 / 21.6 (6.6)
  if (tpr <= 64 && M <= (N <= 512 ? 8L : 4L) * rpb) return 1;
  return (int)std::min<long>(std::max<long>(1, (M + rpb - 1) / rpb), tpr > 256 ? 512 : 1024);
}

template <typename T, typename W>
int run_fwd(const T* x, long ldx, long M, int N, const W* w, const W* b, float eps, T* y, long ldy, float* mean,
            float* rstd, hipStream_t s) {
#define LN_F(TPR, V)                                                                                       \
  ln_fwd<T, W, TPR, V><<<(int)std::min<long>((M + (TPR > 256 ? 1 : 256 / TPR) - 1) / (TPR > 256 ? 1 : 256 / TPR), 1 << 20), \
                         TPR > 256 ? TPR : 256, 0, s>>>(x, ldx, M, N, w, b, eps, y, ldy, mean, rstd)
  if (N > LN_WIDE) ln_fwd_wide<T, W><<<(int)std::min<long>(M, 1 << 20), 1024, 0, s>>>(x, ldx, M, N, w, b, eps, y, ldy, mean, rstd);
  else switch (ln_tpr(N)) {
    case 4: LN_F(4, 1); break;
    case 8: LN_F(8, 1); break;
    case 16: LN_F(16, 1); break;
    case 32: LN_F(32, 1); break;
    case 64: if (N <= 512) LN_F(64, 1); else LN_F(64, 2); break;
    case 256: if (N <= 2048) LN_F(256, 1); else if (N <= 4096) LN_F(256, 2); else LN_F(256, 4); break;
    default: LN_F(1024, 2); break;
  }
#undef LN_F
  return check_launch("ln_fwd");
}

template <typename T, typename W>
int run_bwd(const T* dy, long lddy, const T* x, long ldx, const float* mean, const float* rstd, const W* w, long M, int N,
            T* dx, long lddx, W* dw, W* db, float* ws, hipStream_t s) {
  const int nb = M > 0 ? ln_parts(M, N) : 0;
  const bool direct = nb == 1 && N <= LN_WIDE && dw;
  W* dwo = direct ? dw : nullptr;
  W* dbo = direct ? db : nullptr;
#define LN_B(TPR, V) \
  ln_bwd<T, W, TPR, V><<<nb, TPR > 256 ? TPR : 256, 0, s>>>(dy, lddy, x, ldx, mean, rstd, w, M, N, dx, lddx, ws, dwo, dbo)
  if (nb == 0) {
  } else if (N > LN_WIDE) {
    ln_bwd_wide<T, W><<<(int)std::min<long>(M, 1 << 20), 1024, 0, s>>>(dy, lddy, x, ldx, mean, rstd, w, M, N, dx, lddx);
    ln_bwd_cols<T><<<dim3(cdiv(N, 2048), nb), 256, 0, s>>>(dy, lddy, x, ldx, mean, rstd, M, N, ws);
  } else switch (ln_tpr(N)) {
    case 4: LN_B(4, 1); break;
    case 8: LN_B(8, 1); break;
    case 16: LN_B(16, 1); break;
    case 32: LN_B(32, 1); break;
    case 64: if (N <= 512) LN_B(64, 1); else LN_B(64, 2); break;
    case 256: if (N <= 2048) LN_B(256, 1); else if (N <= 4096) LN_B(256, 2); else LN_B(256, 4); break;
    default: LN_B(1024, 2); break;
  }
#undef LN_B
  if (!direct) ln_reduce<W><<<dim3(cdiv(N, 32), 2), 1024, 0, s>>>(ws, nb, N, dw, db);
  return check_launch("ln_bwd");
}

}  // namespace
}  // namespace ctr

using namespace ctr;

#define LN_TYPES(CALL)                                                                                    \
  if (xt == TY_F32 && wt == TY_F32) return CALL(float, float);                                            \
  if (xt == TY_BF16 && wt == TY_F32) return CALL(__bf16, float);                                          \
  if (xt == TY_BF16 && wt == TY_BF16) return CALL(__bf16, __bf16);                                        \
  if (xt == TY_F16 && wt == TY_F32) return CALL(_Float16, float);                                         \
  if (xt == TY_F16 && wt == TY_F16) return CALL(_Float16, _Float16);                                      \
  CTR_REQUIRE(false, "types: the weight is fp32 or of the rows' type (0 fp32, 1 bf16, 2 fp16)")

extern "C" int ctr_ln_fwd(const void* x, long ldx, long M, int N, const void* w, const void* b, float eps, void* y,
                          long ldy, float* mean, float* rstd, int xt, int wt, void* stream) {
  CTR_REQUIRE(M >= 0 && N >= 1 && N <= (1 << 30), "sizes");
  CTR_REQUIRE(M <= 1 || (ldx >= 0 && ldy >= N), "row strides");
  if (M == 0) return 0;
  CTR_REQUIRE(x && w && y && mean && rstd, "null operand");
#define LN_CALL(T, W) \
  run_fwd((const T*)x, ldx, M, N, (const W*)w, (const W*)b, eps, (T*)y, ldy, mean, rstd, (hipStream_t)stream)
  LN_TYPES(LN_CALL);
#undef LN_CALL
}

extern "C" size_t ctr_ln_bwd_ws_size(long M, int N) {
  return M <= 0 || N <= 0 ? 0 : (size_t)2 * ln_parts(M, N) * N * sizeof(float);
}

extern "C" int ctr_ln_bwd(const void* dy, long lddy, const void* x, long ldx, const float* mean, const float* rstd,
                          const void* w, long M, int N, void* dx, long lddx, void* dw, void* db, void* ws, size_t ws_bytes,
                          int xt, int wt, void* stream) {
  CTR_REQUIRE(M >= 0 && N >= 1 && N <= (1 << 30), "sizes");
  CTR_REQUIRE(M <= 1 || (ldx >= 0 && lddy >= 0 && lddx >= N), "row strides");
  CTR_REQUIRE(dw, "null operand");
  CTR_REQUIRE(M == 0 || (dy && x && mean && rstd && w && dx), "null operand");
  CTR_REQUIRE(ws_bytes >= ctr_ln_bwd_ws_size(M, N), "workspace too small");
#define LN_CALL(T, W)                                                                                              \
  run_bwd((const T*)dy, lddy, (const T*)x, ldx, mean, rstd, (const W*)w, M, N, (T*)dx, lddx, (W*)dw, (W*)db, (float*)ws, \
          (hipStream_t)stream)
  LN_TYPES(LN_CALL);
#undef LN_CALL
}
