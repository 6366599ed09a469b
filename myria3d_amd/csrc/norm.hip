// Layer norm over the last dimension, forward and backward (gfx950).
//
//   mu = mean_c x,  var = mean_c (x - mu)^2,  r = 1 / sqrt(var + eps),  xh = (x - mu) r,  z = xh w + b,  y = z > 0 ? z : slope z
//   g = dy (z > 0 ? 1 : slope);  dx = r (g w - mean_c(g w) - xh mean_c(g w xh));  dw = sum_rows g xh;  db = sum_rows g
//
// (slope = 1: no activation.)  About 8 operations an element forward and 20 backward against 4 to 12 bytes: the memory bounds
// both, so a row is read ONCE and stays in registers — forward for the mean, the squared deviations from it and the result,
// backward for the two row sums and the result.
//
// The mean is held as two floats.  A first sum over cols is rounded to a float, mu1, off by its additions' roundings (3e-4 of a deviation
// where rows lie 3 000 of them from zero, and the mean of a constant row need not be that constant).  The deviations from mu1 are
// exact or nearly so; their own mean is what mu1 is off by, mu2.  Both sums of the second step go across the row together:
//   sum (x - mu)^2 = sum (x - mu1)^2 - mu2 sum (x - mu1),      xh = ((x - mu1) - mu2) r
// so a common offset costs no digits, and the backward pass, from the pair, finds the same bits of xh and the same side of the activation.
//
// A row belongs to TPR lanes, each with NE vectors of 16 bytes (4 fp32 or 8 half-precision elements) and, where the width is not
// a multiple of a vector, one element of the rest.  Up to 64 lanes the row sits inside a wave (narrow rows: several rows a wave,
// sums by lane swaps, no LDS); above, a workgroup of 128 to 1 024 threads takes a row (sums over its waves through LDS).  The
// columns of a lane are the same for every row it meets: w and b are read once per lane (where they fit), and the backward pass
// keeps dw and db of its columns in registers over all its rows (in 32 bits: at 1.6 M x 64 a lane meets 100 rows and the sums are
// off by 2e-7; 64 bits would take twice the registers).  At the end the waves of a workgroup are added up through LDS in a fixed order,
// the workgroups leave one row of partial sums each, and a second kernel adds these in 64 bits: no atomics, the same bits every time.
// Vectors are loaded with the alignment of their element, so rows of any stride take this path.
//
// Bound by memory (6.1 TB/s is what a large scaling reaches here): 1 638 400 x 64 fp32 forward 147 us, 5.7 TB/s, backward 207 + 5 us,
// 6.0 TB/s; 8 192 x 8 192 bf16 54 us, 5.0 TB/s, and 75 + 7 us, 4.9 TB/s.  The next row's loads are issued before the present row's
// sums: without that the latter took 74 and 118 us.
#include "m3d_common.h"
#include "../../include/m3d_hip.h"

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short h8u __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned short h4u __attribute__((ext_vector_type(4), aligned(2)));

struct NormArgs {
  const void *x, *dy, *w, *b;
  void *y, *dx;
  float *mean, *rstd;   // forward: written (nullable); backward: read; mean: two values a row, whose sum it is
  float* parts;         // backward: [gridDim.x][2][cols], or null: no weight gradients
  int64_t rows, ldx, lddy;
  int32_t cols, wtype;  // type of w and b
  float eps, slope, inv;
};

template <int TYPE> struct Vec { static constexpr int N = TYPE == M3D_TYPE_F32 ? 4 : 8; };
template <int TYPE>
__device__ __forceinline__ float el_load(const void* base, int64_t e) {
  if constexpr (TYPE == M3D_TYPE_F32) return ((const float*)base)[e];
  else if constexpr (TYPE == M3D_TYPE_BF16) return bf16_to_f32(((const unsigned short*)base)[e]);
  else return (float)((const _Float16*)base)[e];
}
template <int TYPE>
__device__ __forceinline__ void el_store(void* base, int64_t e, float v) {
  if constexpr (TYPE == M3D_TYPE_F32) ((float*)base)[e] = v;
  else if constexpr (TYPE == M3D_TYPE_BF16) ((unsigned short*)base)[e] = f32_to_bf16(v);
  else ((_Float16*)base)[e] = (_Float16)v;
}
typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(2)));
// a lane's part of a row as it lies in memory: NE vectors of 16 bytes and one element of the rest
template <int NE> struct Raw { u4u v[NE]; float rest; };
// (ONCE: past the caches, see M3D_CACHE_BYTES)
template <int TYPE, int NE, bool ONCE>
__device__ __forceinline__ Raw<NE> raw_load(const void* base, int64_t row_at, int lane, int lanes, int nv, int rest, bool has_rest) {
  Raw<NE> r;
#pragma unroll
  for (int i = 0; i < NE; ++i) {
    const int q = lane + i * lanes;
    r.v[i] = u4u{0u, 0u, 0u, 0u};
    if (q < nv) {
      const u4u* at = (const u4u*)((const char*)base + (row_at + (int64_t)q * Vec<TYPE>::N) * (16 / Vec<TYPE>::N));
      if constexpr (ONCE) r.v[i] = __builtin_nontemporal_load(at);
      else r.v[i] = *at;
    }
  }
  r.rest = has_rest ? el_load<TYPE>(base, row_at + rest) : 0.f;
  return r;
}
template <int TYPE, int NE>
__device__ __forceinline__ void raw_values(const Raw<NE>& r, float* x) {
  constexpr int V = Vec<TYPE>::N;
#pragma unroll
  for (int i = 0; i < NE; ++i)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (TYPE == M3D_TYPE_F32) x[i * V + j] = __uint_as_float(r.v[i][j]);
      else {
        const unsigned short u = (unsigned short)(r.v[i][j >> 1] >> (16 * (j & 1)));
        x[i * V + j] = TYPE == M3D_TYPE_BF16 ? __uint_as_float(j & 1 ? r.v[i][j >> 1] & 0xffff0000u : r.v[i][j >> 1] << 16)
                                             : (float)__builtin_bit_cast(_Float16, u);
      }
    }
  x[NE * V] = r.rest;
}
template <int TYPE, bool ONCE>
__device__ __forceinline__ void vec_store(void* base, int64_t e, const float* v) {
  if constexpr (TYPE == M3D_TYPE_F32) {
    f4u t;
#pragma unroll
    for (int j = 0; j < 4; ++j) t[j] = v[j];
    if constexpr (ONCE) __builtin_nontemporal_store(t, (f4u*)((float*)base + e));
    else *(f4u*)((float*)base + e) = t;
  } else {
    h8u t;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if constexpr (TYPE == M3D_TYPE_BF16) {
        const unsigned p = pack_bf16(v[j], v[j + 1]);
        t[j] = (unsigned short)(p & 0xffffu);
        t[j + 1] = (unsigned short)(p >> 16);
      } else {
        t[j] = __builtin_bit_cast(unsigned short, (_Float16)v[j]);
        t[j + 1] = __builtin_bit_cast(unsigned short, (_Float16)v[j + 1]);
      }
    }
    if constexpr (ONCE) __builtin_nontemporal_store(t, (h8u*)((unsigned short*)base + e));
    else *(h8u*)((unsigned short*)base + e) = t;
  }
}
__device__ __forceinline__ float w_load(const void* base, int64_t e, int type, float none) {
  if (!base) return none;
  return type == M3D_TYPE_F32 ? el_load<M3D_TYPE_F32>(base, e) : type == M3D_TYPE_BF16 ? el_load<M3D_TYPE_BF16>(base, e) : el_load<M3D_TYPE_F16>(base, e);
}
// the weights of a lane's columns: a vector of V elements (vector q of the row's nv; shift: 0), all NE of them and the one of the rest
template <int V>
__device__ __forceinline__ void w_vector(const void* base, int type, float none, int q, int nv, float* w, uint32_t shift = 0u) {
#pragma unroll
  for (int j = 0; j < V; j += 4) {
    float* o = w + j;
    o[0] = o[1] = o[2] = o[3] = q < nv ? none : 0.f;
    if (base && q < nv) {
      if (type == M3D_TYPE_F32) {
        const f4u t = *(const f4u*)((const float*)base + ((uint32_t)(q * V + j) + shift));
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = t[k];
      } else {
        const h4u t = *(const h4u*)((const unsigned short*)base + ((uint32_t)(q * V + j) + shift));
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = type == M3D_TYPE_BF16 ? bf16_to_f32(t[k]) : (float)__builtin_bit_cast(_Float16, (unsigned short)t[k]);
      }
    }
  }
}
template <int V, int NE>
__device__ __forceinline__ void w_loads(const void* base, int type, float none, int lane, int lanes, int nv, int rest, bool has_rest, float* w) {
#pragma unroll
  for (int i = 0; i < NE; ++i) w_vector<V>(base, type, none, lane + i * lanes, nv, w + i * V);
  w[NE * V] = has_rest ? w_load(base, rest, type, none) : 0.f;
}

template <int CTRL>
__device__ __forceinline__ float dpp_f(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}
// sum over groups of TPR lanes, in every lane of the group
template <int TPR>
__device__ __forceinline__ float group_sum(float v) {
  v += dpp_f<0xB1>(v);                          // quad_perm [1,0,3,2]
  v += dpp_f<0x4E>(v);                          // quad_perm [2,3,0,1]
  if constexpr (TPR >= 8) v += dpp_f<0x141>(v);   // row_half_mirror: 8 lanes
  if constexpr (TPR >= 16) v += dpp_f<0x140>(v);  // row_mirror: 16 lanes
  float a, b;
  if constexpr (TPR >= 32) { xgroup_pair16(v, a, b); v = a + b; }
  if constexpr (TPR >= 64) { xgroup_pair32(v, a, b); v = a + b; }
  return v;
}
// the lanes at the same place of every group of TPR lanes of a wave, added up
template <int TPR>
__device__ __forceinline__ float across_groups(float v) {
  float a, b;
  if constexpr (TPR <= 32) { xgroup_pair32(v, a, b); v = a + b; }
  if constexpr (TPR <= 16) { xgroup_pair16(v, a, b); v = a + b; }
  if constexpr (TPR <= 8) v += dpp_f<0x128>(v);  // row_ror:8
  if constexpr (TPR <= 4) v += dpp_f<0x124>(v);  // row_ror:4
  return v;
}
// a row over a whole workgroup: wave sums through LDS; `flip` alternates the two halves of red, so that one barrier a sum is enough
template <int S, int W, typename T>
__device__ __forceinline__ void wg_sums(T (&v)[S], T (*red)[16][W], int& flip) {
  static_assert(S <= W, "sums of a row");
  const int waves = blockDim.x >> 6;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (sizeof(T) == 8) v[s] = wave_sum_d(v[s]);
    else v[s] = group_sum<64>(v[s]);
  }
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int s = 0; s < S; ++s) red[flip][threadIdx.x >> 6][s] = v[s];
  }
  __syncthreads();
  // (16 lanes read a value each and add them up by lane swaps: one read of LDS a wave and sum, not one for every other wave)
  const int wave = threadIdx.x & 15;
#pragma unroll
  for (int s = 0; s < S; ++s) v[s] = wave < waves ? red[flip][wave][s] : (T)0;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if constexpr (sizeof(T) == 8) v[s] = row16_sum_d(v[s]);
    else v[s] = group_sum<16>(v[s]);
  }
  flip ^= 1;
}
// a value of the row: the same in all lanes, and held once a wave, where the row is the workgroup's
template <bool IN>
__device__ __forceinline__ float row_value(float v) {
  if constexpr (IN) return v;
  else return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v)));
}
// s / n by the reciprocal of n (inv, rounded) and the remainder of that quotient, which is exact: a quotient that is a float comes out exactly
__device__ __forceinline__ float over(float s, float n, float inv) {
  const float t = s * inv;
  return fmaf(fmaf(-t, n, s), inv, t);
}

// TPR = 0: a workgroup a row (TPR = 1 024: one of that many threads, whose lanes have half the registers)
#define NORM_THREADS(TPR) ((TPR) == 0 ? 512 : (TPR) == 1024 ? 1024 : 256)
template <int TYPE, int TPR, int NE, bool ONCE>
__global__ __launch_bounds__(NORM_THREADS(TPR)) void layer_norm_kernel(const NormArgs A) {
  constexpr int V = Vec<TYPE>::N;
  constexpr bool IN = TPR > 0 && TPR <= 64;  // the row sits inside a wave
  constexpr int G = IN ? TPR : 64;
  __shared__ float red[2][16][2];
  const int lanes = IN ? G : blockDim.x, lane = IN ? threadIdx.x & (G - 1) : threadIdx.x;
  const int nv = A.cols / V, rest = nv * V + lane;  // full vectors of a row; this lane's element behind them
  const bool has_rest = rest < A.cols;
  float w[NE * V + 1], b[NE * V + 1];
  const int per = IN ? 256 / G : 1;  // rows a workgroup holds at a time
  const int64_t step = (int64_t)gridDim.x * per;
  int64_t row = (int64_t)blockIdx.x * per + (IN ? threadIdx.x / G : 0);
  const int64_t turns = (A.rows - (int64_t)blockIdx.x * per + step - 1) / step;  // (the same for all lanes: they swap values)
  Raw<NE> next = raw_load<TYPE, NE, ONCE>(A.x, row * A.ldx, lane, lanes, row < A.rows ? nv : 0, rest, row < A.rows && has_rest);
  w_loads<V, NE>(A.w, A.wtype, 1.f, lane, lanes, nv, rest, has_rest, w);
  w_loads<V, NE>(A.b, A.wtype, 0.f, lane, lanes, nv, rest, has_rest, b);
  int flip = 0;
  for (int64_t turn = 0; turn < turns; ++turn, row += step) {
    const bool on = row < A.rows;
    float x[NE * V + 1];
    raw_values<TYPE, NE>(next, x);
    {  // the next row is on its way while this one is summed
      const bool more = row + step < A.rows;
      next = raw_load<TYPE, NE, ONCE>(A.x, (row + step) * A.ldx, lane, lanes, more ? nv : 0, rest, more && has_rest);
    }
    float s[1] = {x[NE * V]};
#pragma unroll
    for (int e = 0; e < NE * V; ++e) s[0] += x[e];
    if constexpr (IN) s[0] = group_sum<G>(s[0]);
    else wg_sums(s, red, flip);
    const float mean = row_value<IN>(over(s[0], (float)A.cols, A.inv));
    float q[2] = {0.f, 0.f};  // sums of the deviations from that, and of their squares
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const float from = lane + i * lanes < nv ? mean : 0.f;  // (past the end x is 0)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float d = x[i * V + j] - from;
        x[i * V + j] = d;
        q[0] += d;
        q[1] = fmaf(d, d, q[1]);
      }
    }
    x[NE * V] = has_rest ? x[NE * V] - mean : 0.f;
    q[0] += x[NE * V];
    q[1] = fmaf(x[NE * V], x[NE * V], q[1]);
    if constexpr (IN) {
      q[0] = group_sum<G>(q[0]);
      q[1] = group_sum<G>(q[1]);
    } else wg_sums(q, red, flip);
    const float low = row_value<IN>(over(q[0], (float)A.cols, A.inv)), squares = fmaf(-low, q[0], q[1]);
    const float rstd = row_value<IN>(1.f / sqrtf((squares < 0.f ? 0.f : squares) * A.inv + A.eps));  // (a NaN stays one)
    if (!on) continue;
    if (lane == 0 && A.mean) { A.mean[2 * row] = mean; A.mean[2 * row + 1] = low; A.rstd[row] = rstd; }
    const int64_t yo = row * A.cols;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int q = lane + i * lanes;
      if (q < nv) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float z = fmaf((x[i * V + j] - low) * rstd, w[i * V + j], b[i * V + j]);
          o[j] = z > 0.f ? z : z * A.slope;
        }
        vec_store<TYPE, ONCE>(A.y, yo + q * V, o);
      }
    }
    if (has_rest) {
      const float z = fmaf((x[NE * V] - low) * rstd, w[NE * V], b[NE * V]);
      el_store<TYPE>(A.y, yo + rest, z > 0.f ? z : z * A.slope);
    }
  }
}

template <int TYPE, int TPR, int NE, bool ACT, bool ONCE>
__global__ __launch_bounds__(NORM_THREADS(TPR)) void layer_norm_bwd_kernel(const NormArgs A) {
  constexpr int V = Vec<TYPE>::N, E = NE * V + 1;
  constexpr bool IN = TPR > 0 && TPR <= 64;  // the row sits inside a wave
  constexpr int G = IN ? TPR : 64;
  __shared__ float red[2][16][2];
  extern __shared__ __attribute__((aligned(16))) float sums[];  // IN: the waves' dw and db
  const int lanes = IN ? G : TPR == 1024 ? 1024 : blockDim.x, lane = IN ? threadIdx.x & (G - 1) : threadIdx.x;
  const int nv = A.cols / V, rest = nv * V + lane;
  const bool has_rest = rest < A.cols;
  float w[E], b[E], dw[E], db[E];  // (b only to find the sign of z again)
  const int per = IN ? 256 / G : 1;
  const int64_t step = (int64_t)gridDim.x * per;
  int64_t row = (int64_t)blockIdx.x * per + (IN ? threadIdx.x / G : 0);
  const int64_t turns = (A.rows - (int64_t)blockIdx.x * per + step - 1) / step;
  // 1 024 threads with 16 elements each have 128 registers a lane: none for a row ahead (6 000 x 8 199 fp32, both passes: 510 us with one),
  // nor for w and b, which are read again with every row (with the activation 265 us where they were kept and went to scratch
  // memory, 237 now; without it 233 and 228).
  constexpr bool AHEAD = TPR != 1024 || NE * V < 16;
  Raw<NE> nx, ng;
  float nmean = 0.f, nlow = 0.f, nrstd = 0.f;
  if constexpr (AHEAD) {
    nx = raw_load<TYPE, NE, ONCE>(A.x, row * A.ldx, lane, lanes, row < A.rows ? nv : 0, rest, row < A.rows && has_rest);
    ng = raw_load<TYPE, NE, ONCE>(A.dy, row * A.lddy, lane, lanes, row < A.rows ? nv : 0, rest, row < A.rows && has_rest);
    nmean = row < A.rows ? A.mean[2 * row] : 0.f;
    nlow = row < A.rows ? A.mean[2 * row + 1] : 0.f;
    nrstd = row < A.rows ? A.rstd[row] : 0.f;
  }
  if constexpr (AHEAD) {
    w_loads<V, NE>(A.w, A.wtype, 1.f, lane, lanes, nv, rest, has_rest, w);
    if constexpr (ACT) w_loads<V, NE>(A.b, A.wtype, 0.f, lane, lanes, nv, rest, has_rest, b);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) dw[e] = db[e] = 0.f;
  int flip = 0;
  for (int64_t turn = 0; turn < turns; ++turn, row += step) {
    const bool on = row < A.rows;
    if constexpr (!AHEAD) {
      nx = raw_load<TYPE, NE, ONCE>(A.x, row * A.ldx, lane, lanes, on ? nv : 0, rest, on && has_rest);
      ng = raw_load<TYPE, NE, ONCE>(A.dy, row * A.lddy, lane, lanes, on ? nv : 0, rest, on && has_rest);
      nmean = on ? A.mean[2 * row] : 0.f;
      nlow = on ? A.mean[2 * row + 1] : 0.f;
      nrstd = on ? A.rstd[row] : 0.f;
    }
    float x[E], g[E];
    raw_values<TYPE, NE>(nx, x);
    raw_values<TYPE, NE>(ng, g);
    const float mean = row_value<IN>(nmean), low = row_value<IN>(nlow), rstd = row_value<IN>(nrstd);
    if constexpr (AHEAD) {
      const bool more = row + step < A.rows;
      nx = raw_load<TYPE, NE, ONCE>(A.x, (row + step) * A.ldx, lane, lanes, more ? nv : 0, rest, more && has_rest);
      ng = raw_load<TYPE, NE, ONCE>(A.dy, (row + step) * A.lddy, lane, lanes, more ? nv : 0, rest, more && has_rest);
      nmean = more ? A.mean[2 * (row + step)] : 0.f;
      nlow = more ? A.mean[2 * (row + step) + 1] : 0.f;
      nrstd = more ? A.rstd[row + step] : 0.f;
    }
    float s[2] = {0.f, 0.f};
    uint32_t zero = 0u;
    if constexpr (!AHEAD) asm volatile("" : "+s"(zero));  // (or the compiler would keep the addresses of w and b, 40 registers, over the rows)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if constexpr (!AHEAD) {
        if (e == E - 1) {
          const uint32_t at = (uint32_t)(nv * V + lane) + zero;
          w[e] = has_rest ? w_load(A.w, at, A.wtype, 1.f) : 0.f;
          if constexpr (ACT) b[e] = has_rest ? w_load(A.b, at, A.wtype, 0.f) : 0.f;
        } else if (e % 4 == 0) {
          const int q = (lane + (e / V) * lanes) * (V / 4) + e % V / 4;
          w_vector<4>(A.w, A.wtype, 1.f, q, nv * (V / 4), w + e, zero);
          if constexpr (ACT) w_vector<4>(A.b, A.wtype, 0.f, q, nv * (V / 4), b + e, zero);
        }
      }
      const bool there = e == E - 1 ? on && has_rest : on && lane + (e / V) * lanes < nv;
      const float xh = there ? (x[e] - mean - low) * rstd : 0.f;  // (a lane past the end adds nothing, also where the mean is not finite)
      if constexpr (ACT) g[e] = fmaf(xh, w[e], b[e]) > 0.f ? g[e] : g[e] * A.slope;
      const float gw = g[e] * w[e];
      s[0] += gw;
      s[1] = fmaf(gw, xh, s[1]);
      dw[e] = fmaf(g[e], xh, dw[e]);
      db[e] += g[e];
      x[e] = xh;
      g[e] = gw;
    }
    if constexpr (IN) {
      s[0] = group_sum<G>(s[0]);
      s[1] = group_sum<G>(s[1]);
    } else wg_sums(s, red, flip);
    if (!on || !A.dx) continue;
    const float m0 = row_value<IN>(s[0] * A.inv), m1 = row_value<IN>(s[1] * A.inv);
    const int64_t yo = row * A.cols;
#pragma unroll
    for (int i = 0; i < NE; ++i) {
      const int q = lane + i * lanes;
      if (q < nv) {
        float o[V];
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = rstd * (g[i * V + j] - m0 - x[i * V + j] * m1);
        vec_store<TYPE, ONCE>(A.dx, yo + q * V, o);
      }
    }
    if (has_rest) el_store<TYPE>(A.dx, yo + rest, rstd * (g[E - 1] - m0 - x[E - 1] * m1));
  }
  if (!A.parts) return;
  float* out = A.parts + (int64_t)blockIdx.x * 2 * A.cols;
  if constexpr (IN) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      dw[e] = across_groups<G>(dw[e]);
      db[e] = across_groups<G>(db[e]);
    }
    const int ld = (A.cols + 3) & ~3;  // [4 waves][dw, db][ld]: every wave its own part, added in the order of the waves
    float* mine = sums + (threadIdx.x >> 6) * 2 * ld;
    if ((threadIdx.x & 63) < G) {
#pragma unroll
      for (int i = 0; i < NE; ++i)
#pragma unroll
        for (int j = 0; j < V; j += 4) {
          const int q = lane + i * lanes, e = i * V + j;
          if (q < nv) {
            *(float4*)(mine + q * V + j) = make_float4(dw[e], dw[e + 1], dw[e + 2], dw[e + 3]);
            *(float4*)(mine + ld + q * V + j) = make_float4(db[e], db[e + 1], db[e + 2], db[e + 3]);
          }
        }
      if (has_rest) {
        mine[rest] = dw[E - 1];
        mine[ld + rest] = db[E - 1];
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < A.cols; c += 256) {
      float w4[4], b4[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) { w4[k] = sums[k * 2 * ld + c]; b4[k] = sums[(k * 2 + 1) * ld + c]; }
      out[c] = ((w4[0] + w4[1]) + w4[2]) + w4[3];
      out[A.cols + c] = ((b4[0] + b4[1]) + b4[2]) + b4[3];
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = e == E - 1 ? rest : (lane + (e / V) * lanes) * V + e % V;
      if (e == E - 1 ? has_rest : c < nv * V) { out[c] = dw[e]; out[A.cols + c] = db[e]; }
    }
  }
}

// Rows too wide for the registers of 1 024 threads: the row is read again (from cache) for every step.  A thread adds up cols / 1 024
// elements one after the other, so the row's sums are in 64 bits.
template <int TYPE>
__global__ __launch_bounds__(1024) void layer_norm_wide_kernel(const NormArgs A) {
  __shared__ double red[2][16][1];
  int flip = 0;
  for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
    const int64_t xo = row * A.ldx;
    double s[1] = {0.0}, q[1] = {0.0};
    for (int c = threadIdx.x; c < A.cols; c += 1024) s[0] += (double)el_load<TYPE>(A.x, xo + c);
    wg_sums(s, red, flip);
    const double m = s[0] / (double)A.cols;
    const float mean = (float)m, low = (float)(m - (double)mean);
    for (int c = threadIdx.x; c < A.cols; c += 1024) {
      const double d = (double)(el_load<TYPE>(A.x, xo + c) - mean - low);
      q[0] = fma(d, d, q[0]);
    }
    wg_sums(q, red, flip);
    const float rstd = (float)(1.0 / sqrt(q[0] / (double)A.cols + (double)A.eps));
    if (threadIdx.x == 0 && A.mean) { A.mean[2 * row] = mean; A.mean[2 * row + 1] = low; A.rstd[row] = rstd; }
    for (int c = threadIdx.x; c < A.cols; c += 1024) {
      const float z = fmaf((el_load<TYPE>(A.x, xo + c) - mean - low) * rstd, w_load(A.w, c, A.wtype, 1.f), w_load(A.b, c, A.wtype, 0.f));
      el_store<TYPE>(A.y, row * A.cols + c, z > 0.f ? z : z * A.slope);
    }
  }
}
// (dw and db: a workgroup owns a run of rows AND walks all columns, adding to its own row of partial sums)
template <int TYPE>
__global__ __launch_bounds__(1024) void layer_norm_wide_bwd_kernel(const NormArgs A) {
  __shared__ double red[2][16][2];
  int flip = 0;
  float* out = A.parts ? A.parts + (int64_t)blockIdx.x * 2 * A.cols : nullptr;
  bool first = true;
  for (int64_t row = blockIdx.x; row < A.rows; row += gridDim.x) {
    const int64_t xo = row * A.ldx, go = row * A.lddy;
    const float mean = A.mean[2 * row], low = A.mean[2 * row + 1], rstd = A.rstd[row];
    double s[2] = {0.0, 0.0};
    for (int c = threadIdx.x; c < A.cols; c += 1024) {
      const float xh = (el_load<TYPE>(A.x, xo + c) - mean - low) * rstd, w = w_load(A.w, c, A.wtype, 1.f);
      float g = el_load<TYPE>(A.dy, go + c);
      if (A.slope != 1.f) g = fmaf(xh, w, w_load(A.b, c, A.wtype, 0.f)) > 0.f ? g : g * A.slope;
      s[0] += (double)(g * w);
      s[1] = fma((double)(g * w), (double)xh, s[1]);
      if (out) {
        out[c] = first ? g * xh : fmaf(g, xh, out[c]);
        out[A.cols + c] = first ? g : out[A.cols + c] + g;
      }
    }
    first = false;
    wg_sums(s, red, flip);
    if (!A.dx) continue;
    const float m0 = (float)(s[0] / (double)A.cols), m1 = (float)(s[1] / (double)A.cols);
    for (int c = threadIdx.x; c < A.cols; c += 1024) {
      const float xh = (el_load<TYPE>(A.x, xo + c) - mean - low) * rstd, w = w_load(A.w, c, A.wtype, 1.f);
      float g = el_load<TYPE>(A.dy, go + c);
      if (A.slope != 1.f) g = fmaf(xh, w, w_load(A.b, c, A.wtype, 0.f)) > 0.f ? g : g * A.slope;
      el_store<TYPE>(A.dx, row * A.cols + c, rstd * (g * w - m0 - xh * m1));
    }
  }
}

// dw and db: the partial rows added up in 64 bits.  16 columns (64 bytes) a workgroup at a time, 64 of its threads to a column.
__global__ __launch_bounds__(1024) void layer_norm_wgrad_kernel(const float* __restrict__ parts, int nparts, int cols, int wtype,
                                                                void* __restrict__ dw, void* __restrict__ db) {
  __shared__ double red[64][17];
  const int tc = threadIdx.x & 15, tr = threadIdx.x >> 4;
  const int64_t ld = 2 * (int64_t)cols;
  for (int64_t c0 = (int64_t)blockIdx.x * 16; c0 < ld; c0 += (int64_t)gridDim.x * 16) {
    const int64_t c = c0 + tc;
    double s = 0.0;
    if (c < ld) {
      int p = tr;
      for (; p + 3 * 64 < nparts; p += 4 * 64) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = parts[(p + u * 64) * ld + c];
#pragma unroll
        for (int u = 0; u < 4; ++u) s += (double)v[u];
      }
      for (; p < nparts; p += 64) s += (double)parts[p * ld + c];
    }
    red[tr][tc] = s;
    __syncthreads();
    for (int h = 32; h > 0; h >>= 1) {
      if (tr < h) red[tr][tc] += red[tr + h][tc];
      __syncthreads();
    }
    if (tr == 0 && c < ld) {  // (red[0][tc] is this thread's own: no barrier before the next columns)
      void* out = c < cols ? dw : db;
      const int64_t k = c < cols ? c : c - cols;
      const float v = (float)red[0][tc];
      if (!out) continue;
      if (wtype == M3D_TYPE_F32) el_store<M3D_TYPE_F32>(out, k, v);
      else if (wtype == M3D_TYPE_BF16) el_store<M3D_TYPE_BF16>(out, k, v);
      else el_store<M3D_TYPE_F16>(out, k, v);
    }
  }
}

// ------------------------------------------------------------------------------------------ host
// How a row is laid over lanes (V elements a vector): as few lanes as hold it in 16 elements each — fewer lanes mean fewer steps in
// the sums and fewer idle ones, more elements a lane would cost the backward pass its occupancy.  From a workgroup a row on, the
// backward pass takes 8 elements a lane: twice the lanes are half the rows of partial sums, which at 8 192 columns and rows weigh
// a tenth of the data (bf16, 8 192 x 8 192: 90 + 7 us against 94 + 7 with 16 and half the workgroups, 102 + 12 with as
// many; forward 53 us with 16, 77 with 8).  Rows of up to four vectors take four lanes (2 M x 32 bf16: forward 50 us with four, 86 with eight).
// tpr = 0 or 1024: a workgroup a row; ne = 0: too wide for registers.
struct NormShape { int tpr, ne, threads; };
static NormShape norm_shape(int32_t cols, int32_t type, bool bwd) {
  const int V = type == M3D_TYPE_F32 ? 4 : 8, most = 16 / V, nv = cols / V;
  if (nv <= 4 && cols % V <= 4) return {4, 1, 256};
  for (int ne = 1; ne <= most; ne *= 2)
    if (nv <= 8 * ne) return {8, ne, 256};
  for (int tpr = 16; tpr <= 64; tpr *= 2)
    if (nv <= tpr * most) return {tpr, most, 256};
  const int wide = bwd ? most / 2 : most;
  for (int threads = 128; threads <= 1024; threads *= 2)
    if (nv <= threads * wide) return {threads == 1024 ? 1024 : 0, wide, threads};
  if (nv <= 1024 * most) return {1024, most, 1024};
  return {0, 0, 1024};
}
static int norm_per(const NormShape& s) { return s.tpr && s.tpr <= 64 ? 256 / s.tpr : 1; }
// Workgroups: at most 16 waves on each of the 256 compute units (8 in the backward pass with several rows a wave, whose registers
// allow little more and whose ends, w, b, dw and db, cost more than they hide: 241 against 259 us at 1.6 M x 64 fp32), each with
// the same number of turns.  Rows of up to 40 bytes: what the registers allow, since only many waves keep some of them in flight (20 M x 3
// fp32, both passes: 882 -> 547 us, 12 M x 7: 661 -> 533; but 6 M x 15: 450 -> 556).
static int64_t norm_grid(const NormShape& s, int64_t rows, int32_t cols, int32_t type, bool bwd) {
  const bool few = cols <= (type == M3D_TYPE_F32 ? 10 : 20);
  const int per_unit = few ? (bwd ? 5 : 8) : bwd && s.threads == 256 && norm_per(s) > 1 ? 2 : 1024 / s.threads;
  const int64_t most = 256 * per_unit, need = m3d_cdiv(rows, norm_per(s));
  return need <= most ? need : m3d_cdiv(need, m3d_cdiv(need, most));
}
static bool norm_once(int64_t rows, int32_t cols, int32_t type, int matrices) {
  return (double)rows * cols * (type == M3D_TYPE_F32 ? 4 : 2) * matrices > (double)M3D_CACHE_BYTES;
}

template <int TYPE, int TPR, int NE, bool ONCE>
static void launch_norm(const NormArgs& A, const NormShape& s, int64_t grid, bool bwd, hipStream_t st) {
  const dim3 g((unsigned)grid), t(s.threads);
  constexpr int most = 16 / Vec<TYPE>::N;
  if (!bwd) {
    if constexpr ((TPR > 0 && TPR <= 64) || NE == most) hipLaunchKernelGGL((layer_norm_kernel<TYPE, TPR, NE, ONCE>), g, t, 0, st, A);
    return;
  }
  if constexpr (TPR != 0 || NE == most / 2) {
    const size_t lds = TPR > 0 && TPR <= 64 && A.parts ? 4 * 2 * sizeof(float) * (size_t)((A.cols + 3) & ~3) : 0;
    if (A.slope != 1.f) hipLaunchKernelGGL((layer_norm_bwd_kernel<TYPE, TPR, NE, true, ONCE>), g, t, lds, st, A);
    else hipLaunchKernelGGL((layer_norm_bwd_kernel<TYPE, TPR, NE, false, ONCE>), g, t, lds, st, A);
  }
}
template <int TYPE, bool ONCE>
static void launch_norm_shape(const NormArgs& A, const NormShape& s, int64_t grid, bool bwd, hipStream_t st) {
  constexpr int most = 16 / Vec<TYPE>::N;
  if (s.ne == 0) {
    if (bwd) hipLaunchKernelGGL(layer_norm_wide_bwd_kernel<TYPE>, dim3((unsigned)grid), dim3(1024), 0, st, A);
    else hipLaunchKernelGGL(layer_norm_wide_kernel<TYPE>, dim3((unsigned)grid), dim3(1024), 0, st, A);
    return;
  }
  switch (s.tpr) {
    case 4: launch_norm<TYPE, 4, 1, ONCE>(A, s, grid, bwd, st); break;
    case 8:
      if (s.ne == 1) launch_norm<TYPE, 8, 1, ONCE>(A, s, grid, bwd, st);
      else if (s.ne == 2) launch_norm<TYPE, 8, 2, ONCE>(A, s, grid, bwd, st);
      else if constexpr (most == 4) launch_norm<TYPE, 8, 4, ONCE>(A, s, grid, bwd, st);
      break;
    case 16: launch_norm<TYPE, 16, most, ONCE>(A, s, grid, bwd, st); break;
    case 32: launch_norm<TYPE, 32, most, ONCE>(A, s, grid, bwd, st); break;
    case 64: launch_norm<TYPE, 64, most, ONCE>(A, s, grid, bwd, st); break;
    case 1024:
      if (s.ne == most) launch_norm<TYPE, 1024, most, ONCE>(A, s, grid, bwd, st);
      else launch_norm<TYPE, 1024, most / 2, ONCE>(A, s, grid, bwd, st);
      break;
    default:
      if (bwd) launch_norm<TYPE, 0, most / 2, ONCE>(A, s, grid, bwd, st);
      else launch_norm<TYPE, 0, most, ONCE>(A, s, grid, bwd, st);
  }
}
template <int TYPE>
static void launch_norm_type(const NormArgs& A, const NormShape& s, int64_t grid, bool bwd, hipStream_t st) {
  if (norm_once(A.rows, A.cols, TYPE, bwd ? 3 : 2)) launch_norm_shape<TYPE, true>(A, s, grid, bwd, st);
  else launch_norm_shape<TYPE, false>(A, s, grid, bwd, st);
}
static int launch_norm_any(const NormArgs& A, const NormShape& s, int64_t grid, int32_t type, bool bwd, hipStream_t st) {
  if (type == M3D_TYPE_F32) launch_norm_type<M3D_TYPE_F32>(A, s, grid, bwd, st);
  else if (type == M3D_TYPE_BF16) launch_norm_type<M3D_TYPE_BF16>(A, s, grid, bwd, st);
  else launch_norm_type<M3D_TYPE_F16>(A, s, grid, bwd, st);
  M3D_CHECK_LAUNCH();
  return M3D_OK;
}
static bool norm_type_ok(int32_t t) { return t >= M3D_TYPE_F32 && t <= M3D_TYPE_F16; }
static bool element_aligned(const void* p, int32_t type) { return (((uintptr_t)p) & (type == M3D_TYPE_F32 ? 3 : 1)) == 0; }

extern "C" int m3d_layer_norm_fwd(const void* x, int64_t ldx, const void* w, const void* b, int64_t rows, int32_t cols, int32_t type,
                                  int32_t wtype, float eps, float slope, void* y, float* mean, float* rstd, void* stream) {
  if (rows < 0 || cols < 1 || ldx < 0 || !norm_type_ok(type) || !norm_type_ok(wtype) || !(eps >= 0.f)) return M3D_ERR_INVALID;
  if (cols > 1 << 30) return M3D_ERR_UNSUPPORTED;  // (columns are counted in 32 bits)
  if (rows == 0) return M3D_OK;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return M3D_ERR_INVALID;
  if (!element_aligned(x, type) || !element_aligned(y, type) || !element_aligned(w, wtype) || !element_aligned(b, wtype)) return M3D_ERR_INVALID;
  NormArgs A{};
  A.x = x; A.w = w; A.b = b; A.y = y; A.mean = mean; A.rstd = rstd; A.rows = rows; A.ldx = ldx; A.cols = cols; A.wtype = wtype;
  A.eps = eps; A.slope = slope; A.inv = 1.f / (float)cols;
  const NormShape s = norm_shape(cols, type, false);
  return launch_norm_any(A, s, norm_grid(s, rows, cols, type, false), type, false, (hipStream_t)stream);
}

extern "C" size_t m3d_layer_norm_bwd_workspace_bytes(int64_t rows, int32_t cols, int32_t type) {
  if (rows <= 0 || cols < 1 || !norm_type_ok(type)) return 0;
  return (size_t)norm_grid(norm_shape(cols, type, true), rows, cols, type, true) * 2 * (size_t)cols * sizeof(float);
}

extern "C" int m3d_layer_norm_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, const void* b, const float* mean,
                                  const float* rstd, int64_t rows, int32_t cols, int32_t type, int32_t wtype, float slope, void* dx,
                                  void* dw, void* db, void* ws, void* stream) {
  if (rows < 0 || cols < 1 || ldx < 0 || lddy < 0 || !norm_type_ok(type) || !norm_type_ok(wtype)) return M3D_ERR_INVALID;
  if (cols > 1 << 30) return M3D_ERR_UNSUPPORTED;
  if (rows > 0 && (!dy || !x || !mean || !rstd || ((dw || db) && !ws))) return M3D_ERR_INVALID;
  if (!element_aligned(x, type) || !element_aligned(dy, type) || !element_aligned(dx, type) || !element_aligned(w, wtype) ||
      !element_aligned(b, wtype) || !element_aligned(dw, wtype) || !element_aligned(db, wtype) || (((uintptr_t)ws) & 3))
    return M3D_ERR_INVALID;
  hipStream_t st = (hipStream_t)stream;
  NormArgs A{};
  A.x = x; A.dy = dy; A.w = w; A.b = b; A.dx = dx; A.mean = (float*)mean; A.rstd = (float*)rstd; A.rows = rows; A.ldx = ldx; A.lddy = lddy;
  A.cols = cols; A.wtype = wtype; A.slope = slope; A.inv = 1.f / (float)cols;
  A.parts = (dw || db) ? (float*)ws : nullptr;
  const NormShape s = norm_shape(cols, type, true);
  const int64_t grid = norm_grid(s, rows, cols, type, true);
  if (rows > 0 && (dx || A.parts)) {
    const int rc = launch_norm_any(A, s, grid, type, true, st);
    if (rc != M3D_OK) return rc;
  }
  if (dw || db) {  // (no rows: no parts, zeros)
    // (a launch has less than 2^32 threads)
    const int64_t groups = m3d_cdiv(2 * (int64_t)cols, 16), most = 1 << 20;
    hipLaunchKernelGGL(layer_norm_wgrad_kernel, dim3((unsigned)(groups < most ? groups : most)), dim3(1024), 0, st, (const float*)ws,
                       (int)grid, cols, wtype, dw, db);
    M3D_CHECK_LAUNCH();
  }
  return M3D_OK;
}
