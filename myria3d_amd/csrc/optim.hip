// Optimizer-side kernels over MANY tensors at once (gfx950): the global gradient norm, clipping by it, and the AdamW update with
// its moments in 32 or in 8 bits.
//
//   s = sum g^2,  norm = sqrt(s),  k = min(1, max_norm / (norm + 1e-6)),  g' = k g
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Everything here streams: an element costs a handful of operations and 12 (norm + clip, fp32) to 28 bytes (AdamW, fp32), so the
// memory bounds all of it and the design is about few launches and few bytes:
//   * the tensors' pointers travel as KERNEL ARGUMENTS (up to OPT_TENSORS a launch): no table in device memory to upload when a
//     gradient moves, nothing to keep alive, and a captured graph holds its own copy;
//   * a tensor is cut into blocks of 256 elements, numbered through over all tensors; workgroups take runs of up to 32 blocks in
//     turn and find a run's first tensor by a binary search over the arguments (scalar loads).  The moments live in flat buffers in
//     the same numbering (every tensor's slice starts at a multiple of 256);
//   * the norm is two steps without a launch of its own in between: workgroups leave fp64 partial sums, and whoever needs the
//     norm (the clip kernel, the AdamW kernel) adds them up, in a fixed order, at its start;
//   * vectors are loaded with the alignment of their ELEMENT (unaligned 16-byte accesses are fine on this target), so that views
//     at odd offsets take the same path.
#include "m3d_common.h"
#include "../../include/m3d_hip.h"

#define OPT_TENSORS 152   // 24 bytes each: the list stays under 4 KB of kernel arguments (HipRandLANet has 141 tensors: one launch)
#define OPT_BLOCK 256     // elements of a block (and of one 8-bit scale)
#define OPT_PARTS M3D_GRAD_NORM_PARTS
#define OPT_CHUNK 32      // blocks a workgroup takes at a time where there are many: 16 or 32 KB, one run of memory (AdamW, 75 M: 270 us; 64: 290)
#define OPT_DECODE 4      // blocks a wave decodes side by side

struct TensorList {
  void* p[OPT_TENSORS];
  void* g[OPT_TENSORS];             // null: the tensor has no gradient in this step
  uint32_t blk[OPT_TENSORS + 1];    // number of the tensor's first block
  uint32_t info[OPT_TENSORS];       // bits 0-7: elements of its last block (0: 256), bits 8-9: type (0 fp32, 1 bf16, 2 fp16)
  int32_t count, first;             // tensors in the list; number of the first one
};
static_assert(sizeof(TensorList) <= 3800, "kernel arguments");

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short h4u __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned short h8u __attribute__((ext_vector_type(8), aligned(2)));

__device__ __forceinline__ float half_bits_to_f32(unsigned short b) { return (float)__builtin_bit_cast(_Float16, b); }
__device__ __forceinline__ float bits_to_f32(unsigned short b, int type) { return type == 1 ? bf16_to_f32(b) : half_bits_to_f32(b); }
__device__ __forceinline__ unsigned short f32_to_bits(float v, int type) {
  return type == 1 ? f32_to_bf16(v) : __builtin_bit_cast(unsigned short, (_Float16)v);
}
__device__ __forceinline__ float load1(const void* base, int64_t e, int type) {
  return type == 0 ? ((const float*)base)[e] : bits_to_f32(((const unsigned short*)base)[e], type);
}
__device__ __forceinline__ void store1(void* base, int64_t e, int type, float v) {
  if (type == 0) ((float*)base)[e] = v;
  else ((unsigned short*)base)[e] = f32_to_bits(v, type);
}
__device__ __forceinline__ void store4(void* base, int64_t e, int n, int type, const float (&v)[4]) {
  if (n >= 4) {
    if (type == 0) {
      f4u t;
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = v[j];
      *(f4u*)((float*)base + e) = t;
    } else {
      h4u t;
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = f32_to_bits(v[j], type);
      *(h4u*)((unsigned short*)base + e) = t;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) store1(base, e + j, type, v[j]);
  }
}

// the tensor that block b belongs to (blk[0] <= b < blk[count])
__device__ __forceinline__ int tensor_of(const TensorList& L, uint32_t b) {
  int lo = 0, hi = L.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (L.blk[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ int64_t tensor_numel(const TensorList& L, int t) {
  const int last = L.info[t] & 255;
  return (int64_t)(L.blk[t + 1] - L.blk[t]) * OPT_BLOCK - (last ? OPT_BLOCK - last : 0);
}

// sum over the 256 threads of a workgroup, the same bits in every thread
__device__ __forceinline__ double block_sum_d(double v, double* red /* [4] */) {
  v = wave_sum_d(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return red[0] + red[1] + red[2] + red[3];
}
__device__ __forceinline__ double norm_of(const double* __restrict__ parts, int nparts, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < nparts; i += 256) s += parts[i];
  return sqrt(block_sum_d(s, red));
}
__device__ __forceinline__ double clip_factor(double norm, double max_norm) {
  const double k = max_norm / (norm + 1e-6);
  return k > 1.0 ? 1.0 : k;  // (a NaN norm stays a NaN)
}

// ---- s: fp64 partial sums of g^2 (to 2^-53: the factor that follows, and every 8-bit code behind it, does not depend on how
// the work was cut).  Bound by memory: 400 MB fp32 in 80 us, 250 MB bf16 in 55 us where the caches held nothing to write back before.
template <int TYPE>
__device__ __forceinline__ double range_squares(const void* base, int64_t lo, int64_t n) {  // n vectors of 16 bytes from element lo on
  constexpr int N = TYPE == 0 ? 4 : 8;
  double s[2] = {0.0, 0.0};
  auto add = [&](const float (&x)[N]) {
#pragma unroll
    for (int j = 0; j < N; ++j) s[j & 1] = fma((double)x[j], (double)x[j], s[j & 1]);
  };
  auto load = [&](int64_t i, float (&x)[N]) {
    if constexpr (TYPE == 0) {
      const f4u t = *(const f4u*)((const float*)base + lo + i * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = t[j];
    } else {
      const h8u t = *(const h8u*)((const unsigned short*)base + lo + i * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = bits_to_f32(t[j], TYPE);
    }
  };
  int64_t i = threadIdx.x;
  for (; i + (4 - 1) * 256 < n; i += 4 * 256) {
    float x[4][N];
#pragma unroll
    for (int u = 0; u < 4; ++u) load(i + u * 256, x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u) add(x[u]);
  }
  for (; i < n; i += 256) {
    float x[N];
    load(i, x);
    add(x);
  }
  return s[0] + s[1];
}

__global__ __launch_bounds__(256, 8) void grad_norm_kernel(const TensorList L, uint32_t chunk, double* __restrict__ parts, int add) {
  __shared__ double red[4];
  const uint32_t first = L.blk[0], n = L.blk[L.count] - first;
  double s = 0.0;
  for (uint64_t c = (uint64_t)blockIdx.x * chunk; c < n; c += (uint64_t)gridDim.x * chunk) {
    uint32_t b = first + (uint32_t)c;
    const uint32_t c1 = first + (c + chunk < n ? (uint32_t)(c + chunk) : n);
    for (int t = tensor_of(L, b); b < c1; ++t) {
      const uint32_t stop = L.blk[t + 1] < c1 ? L.blk[t + 1] : c1;
      if (L.g[t]) {
        const int type = (L.info[t] >> 8) & 3;
        const int64_t lo = (int64_t)(b - L.blk[t]) * OPT_BLOCK;
        int64_t hi = (int64_t)(stop - L.blk[t]) * OPT_BLOCK;
        const int64_t all = tensor_numel(L, t);
        if (hi > all) hi = all;
        const int64_t per = type == 0 ? 4 : 8, m = (hi - lo) / per, tail = lo + m * per;
        s += type == 0 ? range_squares<0>(L.g[t], lo, m) : type == 1 ? range_squares<1>(L.g[t], lo, m) : range_squares<2>(L.g[t], lo, m);
        if (tail + (int64_t)threadIdx.x < hi) {
          const double x = (double)load1(L.g[t], tail + threadIdx.x, type);
          s = fma(x, x, s);
        }
      }
      b = stop;
    }
  }
  s = block_sum_d(s, red);
  if (threadIdx.x == 0) parts[blockIdx.x] = add ? parts[blockIdx.x] + s : s;
}

// ---- g *= k in place (written also where k = 1).  The runs are taken in the opposite order of the norm's pass: what that pass
// read last is still in the 256 MB cache in front of the memory.  250 MB bf16: 82 us, 6.1 TB/s of reading and writing.
template <int TYPE>
__device__ __forceinline__ void range_scale(void* base, int64_t lo, int64_t n, float k) {  // n vectors of 16 bytes from element lo on
  constexpr int N = TYPE == 0 ? 4 : 8;
  for (int64_t i = threadIdx.x; i < n; i += 4 * 256) {
    f4u f[4];
    h8u h[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * 256 < n) {
        if constexpr (TYPE == 0) f[u] = *(const f4u*)((const float*)base + lo + (i + u * 256) * N);
        else h[u] = *(const h8u*)((const unsigned short*)base + lo + (i + u * 256) * N);
      }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * 256 < n) {
        if constexpr (TYPE == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) f[u][j] *= k;
          *(f4u*)((float*)base + lo + (i + u * 256) * N) = f[u];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) h[u][j] = f32_to_bits(bits_to_f32(h[u][j], TYPE) * k, TYPE);
          *(h8u*)((unsigned short*)base + lo + (i + u * 256) * N) = h[u];
        }
      }
  }
}

__global__ __launch_bounds__(256) void grad_clip_kernel(const TensorList L, uint32_t chunk, const double* __restrict__ parts, int nparts,
                                                        double max_norm, float* __restrict__ norm_out) {
  __shared__ double red[4];
  const double norm = norm_of(parts, nparts, red);
  const float k = (float)clip_factor(norm, max_norm);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const uint32_t first = L.blk[0], n = L.blk[L.count] - first;
  const int64_t chunks = ((int64_t)n + chunk - 1) / chunk;
  for (int64_t q = chunks - 1 - blockIdx.x; q >= 0; q -= gridDim.x) {
    const uint64_t c = (uint64_t)q * chunk;
    uint32_t b = first + (uint32_t)c;
    const uint32_t c1 = first + (c + chunk < n ? (uint32_t)(c + chunk) : n);
    for (int t = tensor_of(L, b); b < c1; ++t) {
      const uint32_t stop = L.blk[t + 1] < c1 ? L.blk[t + 1] : c1;
      if (L.g[t]) {
        const int type = (L.info[t] >> 8) & 3;
        const int64_t lo = (int64_t)(b - L.blk[t]) * OPT_BLOCK;
        int64_t hi = (int64_t)(stop - L.blk[t]) * OPT_BLOCK;
        const int64_t all = tensor_numel(L, t);
        if (hi > all) hi = all;
        const int64_t per = type == 0 ? 4 : 8, m = (hi - lo) / per, tail = lo + m * per;
        if (type == 0) range_scale<0>(L.g[t], lo, m, k);
        else if (type == 1) range_scale<1>(L.g[t], lo, m, k);
        else range_scale<2>(L.g[t], lo, m, k);
        if (tail + (int64_t)threadIdx.x < hi)
          store1(L.g[t], tail + threadIdx.x, type, load1(L.g[t], tail + threadIdx.x, type) * k);
      }
      b = stop;
    }
  }
}

// ------------------------------------------------------------------------------------------
// AdamW.  state (fp32 words): [0] updates done, [1] the master ticket, [2 ..] 64 tickets (uint32, zero between launches); missed[i]:
// updates that tensor i had no gradient in — its own count is state[0] - missed[i], as torch counts per parameter.
// ------------------------------------------------------------------------------------------
struct AdamArgs {
  void *m, *v;
  float *ms, *vs;                // block scales (8 bits)
  float* state;
  int32_t* missed;
  const double* parts;           // gradient norm's partial sums, or null: no clipping
  float* norm_out;
  const float* lr_dev;           // learning rate on the device, or null
  double max_norm, lr, log_b1, log_b2, wd;
  double b1, b2, c1, c2;         // betas and 1 - betas
  float eps;
  int32_t nparts, bump;
  uint32_t chunk;
};

struct AdamStep { float decay, size, root; };  // p *= decay; p -= size * m / (sqrt(v) * root + eps)
// 1 - b^t through expm1: at b = 0.999, t = 1 the plain difference in fp32 is off by 1e-5
__device__ __forceinline__ AdamStep adam_step_of(const AdamArgs& A, double t, double lr) {
  AdamStep s;
  s.decay = (float)(1.0 - lr * A.wd);
  s.size = (float)(lr / -expm1(t * A.log_b1));
  s.root = (float)(1.0 / sqrt(-expm1(t * A.log_b2)));
  return s;
}

// ---- 8 bits.  A value comes as a double over its block's scale.  What is below the fraction's bits decides the rounding, and must
// not be rounded itself before: the upper word's last bit takes in whether anything is below it (the words hold 17 and 16 bits more
// than the codes do).
#define NAN_M 0x7fu
#define NAN_V 0xffu
__device__ __forceinline__ int sticky_word(double x) {
  const uint32_t lo = (uint32_t)__double2loint(x);
  return __double2hiint(x) | (int)(lo < 1u ? lo : 1u);  // (one minimum: the compiler's own form of lo != 0 is a comparison and a select)
}
// decoded, as held: one rounding in 32 bits (the factor 2^-8 is exact: the block's largest magnitude has code 256)
__device__ __forceinline__ void decode_m4(uint32_t c, float s, float (&m)[4]) {
  const float k = 0.00390625f;  // (the conversion scales by powers of two)
  const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, k, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(c, k, true);
  m[0] = a[0] * s; m[1] = a[1] * s; m[2] = b[0] * s; m[3] = b[1] * s;
}
// u(c) = 2^((c >> 3) - 31) (1 + (c & 7) / 8): the code is the upper part of a float with its exponent moved
__device__ __forceinline__ void decode_v4(uint32_t q, float s, float (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t c = (q >> (8 * j)) & 255u;
    v[j] = c ? __uint_as_float((c << 20) + ((127u - 31u) << 23)) * s : 0.f;
  }
  if (((~q - 0x01010101u) & q & 0x80808080u) != 0u) {  // (a byte of ones)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (((q >> (8 * j)) & 255u) == NAN_V) v[j] = __builtin_nanf("");
  }
}
// the largest of a wave's values, in every lane; the bits of floats that are not negative are ordered as the floats are
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false); }
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = umax(v, dpp_u<0xB1>(v));
  v = umax(v, dpp_u<0x4E>(v));
  v = umax(v, dpp_u<0x141>(v));
  v = umax(v, dpp_u<0x140>(v));
  const m3d_u2 a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = umax(a[0], a[1]);
  const m3d_u2 b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(umax(b[0], b[1]));
}

// one wave's block of new moments (mf, vf: rounded to 32 bits) -> codes and scales; every lane: four consecutive elements
__device__ __forceinline__ void encode_block(const double (&m)[4], const double (&v)[4], const float (&mf)[4], const float (&vf)[4],
                                             uint32_t& cm, uint32_t& cv, float& sm, float& sv) {
  const uint32_t inf = 0x7f800000u;
  uint32_t mx = 0u, vx = 0u;  // (rounding keeps the order: the largest one's rounding is the scale)
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    mx = umax(mx, __float_as_uint(mf[j]) & 0x7fffffffu);
    vx = umax(vx, __float_as_uint(vf[j]));  // (with its sign: what is negative here is no second moment, and counts as not finite)
  }
  mx = wave_umax(mx);
  vx = wave_umax(vx);
  const bool odd = mx >= inf || vx >= inf;  // something is not finite: the scale is the largest of the rest
  if (odd) {
    asm volatile("" ::: );  // (a branch, not selects: here and below)
    mx = vx = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = __float_as_uint(mf[j]) & 0x7fffffffu, b = __float_as_uint(vf[j]);
      mx = umax(mx, a < inf ? a : 0u);
      vx = umax(vx, b < inf ? b : 0u);
    }
    mx = wave_umax(mx);
    vx = wave_umax(vx);
  }
  mx = mx < 0x00800000u ? 0u : mx;  // under 2^-126
  vx = vx < 0x00800000u ? 0u : vx;
  sm = __uint_as_float(mx);
  sv = __uint_as_float(vx);
  // Quotients by the reciprocal: off by two units in the last place at most, which matters for a code only where the quotient's lower
  // word is next to zero.  There (one value in 2^29) the division itself decides.  A scale of zero makes everything zero.
  const double dm = (double)sm * 0.00390625, dv = (double)sv, im = mx ? 1.0 / dm : 0.0, iv = vx ? 1.0 / dv : 0.0;
  double qm[4], qv[4];
  bool near = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    qm[j] = m[j] * im;
    qv[j] = v[j] * iv;
    near |= (uint32_t)__double2loint(qm[j]) + 4u < 8u && m[j] != 0.0;
    near |= (uint32_t)__double2loint(qv[j]) + 4u < 8u && v[j] != 0.0;
  }
  if (__ballot(near) != 0ull) {  // (a branch of the wave: the compiler would divide everywhere and select)
    asm volatile("" ::: );
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      qm[j] = mx ? m[j] / dm : 0.0;
      qv[j] = vx ? v[j] / dv : 0.0;
    }
  }
  float r[4];
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    r[j] = (float)__hiloint2double(sticky_word(qm[j]), 0);  // (exact; the conversion below rounds to nearest even)
    const uint32_t u = (uint32_t)sticky_word(qv[j]);
    const int k = (int)((u + 0xffffu + ((u >> 17) & 1u)) >> 17) - ((1023 - 31) << 3);  // nearest even at three bits of fraction
    const int least = (int)(u < 1u ? u : 1u);  // what is above zero stays above it
    c[j] = (uint32_t)(k < least ? least : k);
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], w, true);
  cm = (uint32_t)w;
  if (odd) {
    asm volatile("" ::: );
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if ((__float_as_uint(mf[j]) & 0x7fffffffu) >= inf) cm = (cm & ~(0xffu << (8 * j))) | (NAN_M << (8 * j));
      if (__float_as_uint(vf[j]) >= inf) c[j] = NAN_V;  // (the others are 248 at most)
    }
  }
  cv = c[0] | (c[1] << 8) | (c[2] << 16) | (c[3] << 24);
}

// sqrt and quotient by the instructions (each within one unit in the last place; the update is a small part of the parameter):
// what the compiler makes of sqrtf and / costs 25 instructions an element.  The square root's argument is kept out of the denormals.
// Beside an eps of 2^-40 or more the root of a denormal number, under 2^-63, says nothing, whatever the instruction makes of it.
__device__ __forceinline__ void quick_roots(const float (&v)[4], float eps, float (&r)[4]) {
  if (eps >= 0x1p-40f) {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = __builtin_amdgcn_sqrtf(v[j]);
  } else {
    asm volatile("" ::: );  // (a branch)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool tiny = v[j] < 0x1p-96f;
      const float t = __builtin_amdgcn_sqrtf(tiny ? v[j] * 0x1p64f : v[j]);
      r[j] = tiny ? t * 0x1p-32f : t;
    }
  }
}

// a lane's four elements as they lie in memory
struct Raw { uint32_t w[4]; };
typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u2u __attribute__((ext_vector_type(2), aligned(2)));
template <bool ONCE>
__device__ __forceinline__ Raw raw_load(const void* base, int64_t e, int n, int type) {
  Raw r{};
  if (n >= 4) {
    if (type == 0) {
      const u4u* at = (const u4u*)((const float*)base + e);
      u4u t;
      if constexpr (ONCE) t = __builtin_nontemporal_load(at);
      else t = *at;
      r.w[0] = t[0]; r.w[1] = t[1]; r.w[2] = t[2]; r.w[3] = t[3];
    } else {
      const u2u* at = (const u2u*)((const unsigned short*)base + e);
      u2u t;
      if constexpr (ONCE) t = __builtin_nontemporal_load(at);
      else t = *at;
      r.w[0] = t[0]; r.w[1] = t[1];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j)
      if (j < n) {
        if (type == 0) r.w[j] = ((const uint32_t*)base)[e + j];
        else r.w[j >> 1] |= (uint32_t)((const unsigned short*)base)[e + j] << (16 * (j & 1));
      }
  }
  return r;
}
__device__ __forceinline__ void raw_values(const Raw& r, int type, float (&v)[4]) {
  if (type == 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(r.w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = bits_to_f32((unsigned short)(r.w[j >> 1] >> (16 * (j & 1))), type);
  }
}

// A workgroup walks chunks of up to 32 blocks, its four waves take a chunk's blocks in turn, a lane four consecutive elements (16-byte
// accesses in fp32); all workgroups together walk one window of memory, and a chunk's 8-bit scales, one line of cache, have one writer
// (with single blocks dealt out to the waves of all workgroups: 590 against 440 us for 100 M parameters with 8-bit moments).
//   32 bits: bound by memory.  The next block is on its way while the present one is computed (320 us without).  75 M bf16 parameters
//     (22 bytes each): 270 us, 6.1 TB/s, what a large scaling reaches here; 3 M fp32 (28 bytes): 19.5 us.
//   8 bits: 85 vector instructions an element, a third of them in 64 bits, beside 16 bytes: the vector units are busy 71 % of the
//     time (SQ counters) and 100 M fp32 parameters take 340 us, 4.7 TB/s; 100 M bf16, 10 bytes an element, 333 us.  Six or seven waves
//     on a SIMD instead of five change nothing; fetching ahead costs more in registers than it hides (389 us).
// ONCE: past the caches (see M3D_CACHE_BYTES), but for what is written of the parameters, which the forward pass reads next.
template <int BITS, bool ONCE>
__global__ __launch_bounds__(256, 5) void adamw_kernel(const TensorList L, const AdamArgs A) {
  constexpr bool AHEAD = BITS == 32;
  __shared__ double red[4];
  const int lane = threadIdx.x & 63;
  const double done = (double)__hip_atomic_load(&A.state[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  double k = 1.0;
  bool go = true;
  if (A.parts) {
    const double norm = norm_of(A.parts, A.nparts, red);
    k = clip_factor(norm, A.max_norm);
    go = norm <= 1.7e308;  // a norm that is not finite: the step is not taken (neither counted)
    if (A.norm_out && blockIdx.x == 0 && threadIdx.x == 0) *A.norm_out = (float)norm;
  }
  const uint32_t first = L.blk[0], n = L.blk[L.count] - first, chunk = A.chunk;
  // (chunks from the end on: against the order of the norm's pass, whose last reads are still in cache)
  const int64_t chunks = ((int64_t)n + chunk - 1) / chunk;
  int64_t q = chunks - 1 - blockIdx.x;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  uint32_t o = wave;  // block of the chunk
  auto there = [&]() { return q >= 0 && o < chunk && (uint64_t)q * chunk + o < n; };
  if (!there()) q -= gridDim.x;  // (the last chunk may hold less than a block for every wave; all others hold one)
  if (go && there()) {
    const double lr = A.lr_dev ? (double)A.lr_dev[0] : A.lr;
    const float kf = (float)k, b1 = (float)A.b1, b2 = (float)A.b2, d1 = (float)A.c1, d2 = (float)A.c2;
    AdamStep S{};
    int at = -1;
    struct Block { int t, type, n; uint32_t b; int64_t e; bool on; } cur, nxt;
    struct Data { Raw g, p; f32x4 m, v; uint32_t qm, qv; float sm, sv; } dc, dn;
    auto find = [&](int t) {
      Block r;
      r.b = first + (uint32_t)(q * chunk + o);
      if (t < 0 || r.b < L.blk[t] || r.b >= L.blk[t + 1]) t = tensor_of(L, r.b);
      r.t = t;
      r.type = (L.info[t] >> 8) & 3;
      const int last = L.info[t] & 255;
      r.e = (int64_t)(r.b - L.blk[t]) * OPT_BLOCK + lane * 4;
      const int n = (r.b + 1 == L.blk[t + 1] && last ? last : OPT_BLOCK) - lane * 4;
      r.n = n > 4 ? 4 : n;
      r.on = L.g[t] != nullptr;
      return r;
    };
    auto fetch = [&](const Block& r, Data& d) {
      if (!r.on) return;
      d.g = d.p = Raw{};
      if (r.n > 0) {
        d.g = raw_load<ONCE>(L.g[r.t], r.e, r.n, r.type);
        d.p = raw_load<ONCE>(L.p[r.t], r.e, r.n, r.type);
      }
      const int64_t s = (int64_t)r.b * 64 + lane;  // the lane's four elements in the flat moments
      if constexpr (BITS == 32) {
        if constexpr (ONCE) {
          d.m = __builtin_nontemporal_load(&((const f32x4*)A.m)[s]);
          d.v = __builtin_nontemporal_load(&((const f32x4*)A.v)[s]);
        } else {
          d.m = ((const f32x4*)A.m)[s];
          d.v = ((const f32x4*)A.v)[s];
        }
      } else {
        d.qm = ((const uint32_t*)A.m)[s];
        d.qv = ((const uint32_t*)A.v)[s];
        d.sm = A.ms[r.b];
        d.sv = A.vs[r.b];
      }
    };
    cur = find(-1);
    fetch(cur, dc);
    while (true) {
      o += 4;
      if (!there()) {
        o = wave;
        q -= gridDim.x;
      }
      const bool more = there();
      if (AHEAD && more) {
        nxt = find(cur.t);
        fetch(nxt, dn);
      }
      if (!cur.on) {
        if (cur.b == L.blk[cur.t] && lane == 0) A.missed[L.first + cur.t] += 1;
      } else {
        if (cur.t != at) {
          at = cur.t;
          S = adam_step_of(A, done + 1.0 - (double)A.missed[L.first + at], lr);
        }
        const int64_t s = (int64_t)cur.b * 64 + lane;
        float p[4], gv[4], mf[4], vf[4];
        raw_values(dc.g, cur.type, gv);
        raw_values(dc.p, cur.type, p);
        if constexpr (BITS == 32) {
          f32x4 mo, vo;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float x = gv[j] * kf;
            mf[j] = mo[j] = b1 * dc.m[j] + d1 * x;
            vf[j] = vo[j] = b2 * dc.v[j] + d2 * x * x;
          }
          if constexpr (ONCE) {
            __builtin_nontemporal_store(mo, &((f32x4*)A.m)[s]);
            __builtin_nontemporal_store(vo, &((f32x4*)A.v)[s]);
          } else {
            ((f32x4*)A.m)[s] = mo;
            ((f32x4*)A.v)[s] = vo;
          }
        } else {
          float om[4], ov[4];
          double m[4], v[4];
          decode_m4(dc.qm, dc.sm, om);
          decode_v4(dc.qv, dc.sv, ov);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // In 64 bits, every operation rounded by itself: with decimal betas the sums (9 a + b) / 10 hit the borders of 32 bits (the
            // scale's) one time in ten, and which side they fall to must not depend on what the compiler contracts.
#pragma clang fp contract(off)
            const double x = (double)gv[j] * k;
            m[j] = A.b1 * (double)om[j] + A.c1 * x;
            v[j] = A.b2 * (double)ov[j] + A.c2 * (x * x);
            mf[j] = (float)m[j];
            vf[j] = (float)v[j];
          }
          uint32_t cm, cv;
          float nm, nv;
          encode_block(m, v, mf, vf, cm, cv, nm, nv);
          ((uint32_t*)A.m)[s] = cm;
          ((uint32_t*)A.v)[s] = cv;
          if (lane == 0) { A.ms[cur.b] = nm; A.vs[cur.b] = nv; }
        }
        float root[4];
        quick_roots(vf, A.eps, root);
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = p[j] * S.decay - S.size * mf[j] * __builtin_amdgcn_rcpf(root[j] * S.root + A.eps);
        if (cur.n > 0) store4(L.p[cur.t], cur.e, cur.n, cur.type, p);
      }
      if (!more) break;
      if (!AHEAD) {
        nxt = find(cur.t);
        fetch(nxt, dn);
      }
      cur = nxt;
      dc = dn;
    }
  }
  if (!A.bump) return;
  __syncthreads();  // every thread of this workgroup has used its copy of the count
  if (threadIdx.x == 0) {  // two levels of tickets: one address takes ~15 ns an arrival
    unsigned* tk = (unsigned*)&A.state[1];
    const unsigned sub = blockIdx.x % 64, members = gridDim.x / 64 + (sub < gridDim.x % 64 ? 1u : 0u);
    if (atomicAdd(&tk[1 + sub], 1u) == members - 1) {
      tk[1 + sub] = 0u;
      const unsigned groups = gridDim.x < 64 ? gridDim.x : 64;
      if (atomicAdd(&tk[0], 1u) == groups - 1) {
        if (go) __hip_atomic_store(&A.state[0], (float)(done + 1.0), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        tk[0] = 0u;
      }
    }
  }
}

// ---- 8-bit moments <-> 32 bits (checkpoints, inspection).  200 M elements decoded: 361 us, 5.5 TB/s, mostly writes (383 with 2 048
// workgroups that go on, 424 with one block a wave at a time).
__global__ __launch_bounds__(256) void moments_decode_kernel(const uint32_t* __restrict__ qm, const uint32_t* __restrict__ qv,
                                                             const float* __restrict__ sm, const float* __restrict__ sv,
                                                             f32x4* __restrict__ m, f32x4* __restrict__ v, int64_t blocks) {
  const int lane = threadIdx.x & 63;
  for (int64_t b = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * OPT_DECODE; b < blocks; b += (int64_t)gridDim.x * 4 * OPT_DECODE) {
    uint32_t cm[OPT_DECODE], cv[OPT_DECODE];
    float fm[OPT_DECODE], fv[OPT_DECODE];
#pragma unroll
    for (int u = 0; u < OPT_DECODE; ++u) {  // (a wave: four blocks side by side, all on their way before the first is stored)
      const int64_t k = b + u < blocks ? b + u : blocks - 1;
      cm[u] = qm[k * 64 + lane]; cv[u] = qv[k * 64 + lane];
      fm[u] = sm[k]; fv[u] = sv[k];
    }
#pragma unroll
    for (int u = 0; u < OPT_DECODE; ++u) {
      if (b + u >= blocks) break;
      float a[4], c[4];
      decode_m4(cm[u], fm[u], a);
      decode_v4(cv[u], fv[u], c);
      m[(b + u) * 64 + lane] = f32x4{a[0], a[1], a[2], a[3]};
      v[(b + u) * 64 + lane] = f32x4{c[0], c[1], c[2], c[3]};
    }
  }
}
__global__ __launch_bounds__(256) void moments_encode_kernel(const f32x4* __restrict__ m, const f32x4* __restrict__ v,
                                                             uint32_t* __restrict__ qm, uint32_t* __restrict__ qv,
                                                             float* __restrict__ sm, float* __restrict__ sv, int64_t blocks) {
  const int lane = threadIdx.x & 63;
  for (int64_t b = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); b < blocks; b += (int64_t)gridDim.x * 4) {
    const f32x4 a = m[b * 64 + lane], c = v[b * 64 + lane];
    const float mf[4] = {a[0], a[1], a[2], a[3]}, vf[4] = {c[0], c[1], c[2], c[3]};
    const double md[4] = {a[0], a[1], a[2], a[3]}, vd[4] = {c[0], c[1], c[2], c[3]};
    uint32_t cm, cv;
    float nm, nv;
    encode_block(md, vd, mf, vf, cm, cv, nm, nv);
    qm[b * 64 + lane] = cm;
    qv[b * 64 + lane] = cv;
    if (lane == 0) { sm[b] = nm; sv[b] = nv; }
  }
}

// ------------------------------------------------------------------------------------------ host
static int check_tensors(void* const* ptrs, const int64_t* numel, const int32_t* types, int32_t count, int64_t* blocks) {
  if (count < 0 || (count > 0 && (!ptrs || !numel || !types)) ) return M3D_ERR_INVALID;
  int64_t b = 0;
  for (int32_t i = 0; i < count; ++i) {
    if (numel[i] < 0 || types[i] < 0 || types[i] > 2) return M3D_ERR_INVALID;
    if (((uintptr_t)ptrs[i]) & (types[i] == 0 ? 3 : 1)) return M3D_ERR_INVALID;
    if (numel[i] > ((int64_t)1 << 39)) return M3D_ERR_UNSUPPORTED;
    b += m3d_cdiv(numel[i], OPT_BLOCK);
    if (b > 0xfffffff0ll) return M3D_ERR_UNSUPPORTED;  // (blocks are numbered in 32 bits)
  }
  *blocks = b;
  return M3D_OK;
}
// the tensors from `from` on that fit one launch (tensors without elements take no blocks and stay out of the search); the next one
static int32_t fill_list(TensorList& L, void* const* params, void* const* grads, const int64_t* numel, const int32_t* types, int32_t from,
                         int32_t count, uint32_t block) {
  int32_t n = 0, i = from;
  L.first = from;
  for (; i < count && n < OPT_TENSORS; ++i, ++n) {
    L.p[n] = params ? params[i] : nullptr;
    L.g[n] = grads[i];
    L.blk[n] = block;
    L.info[n] = (uint32_t)((numel[i] & 255) | ((int64_t)types[i] << 8));
    block += (uint32_t)m3d_cdiv(numel[i], OPT_BLOCK);
  }
  L.blk[n] = block;
  L.count = n;
  return i;
}
// blocks a workgroup takes at a time: one where there are few (every unit then has some), up to 32, which is 16 or 32 KB
static uint32_t chunk_of(int64_t blocks, int64_t most) {
  const int64_t c = m3d_cdiv(blocks, most);
  return (uint32_t)(c < 1 ? 1 : c > OPT_CHUNK ? OPT_CHUNK : c);
}
static int64_t grid_of(int64_t blocks, uint32_t chunk, int64_t most) {
  const int64_t g = m3d_cdiv(blocks, chunk);
  return g < most ? g : most;
}

// Workgroups of the update: what the registers let run at once (five waves on a SIMD; more would run behind the first ones, alone:
// 100 M parameters with 8-bit moments take 350 us with 1 280 and 410 with 1 792).  With 32-bit moments four are enough to keep the memory
// busy (75 M bf16 parameters: 270 us with 1 024, 276 with 1 280, 330 with 1 536).
static int64_t adamw_grid(int32_t bits) { return bits == 32 ? 1024 : 1280; }

extern "C" int m3d_grad_norm(void* const* grads, const int64_t* numel, const int32_t* types, int32_t count, double* parts, int32_t* nparts,
                             void* stream) {
  int64_t blocks = 0;
  const int rc = check_tensors(grads, numel, types, count, &blocks);
  if (rc != M3D_OK) return rc;
  if (!parts || !nparts) return M3D_ERR_INVALID;
  TensorList L;
  // the first launch leaves a value in every part
  uint32_t grid = 1;
  for (int32_t i = 0; i < count;) {
    i = fill_list(L, nullptr, grads, numel, types, i, count, 0);
    const int64_t n = L.blk[L.count], w = grid_of(n, chunk_of(n, OPT_PARTS), OPT_PARTS);
    if (w > grid) grid = (uint32_t)w;
  }
  int32_t i = 0, add = 0;
  do {
    i = count ? fill_list(L, nullptr, grads, numel, types, i, count, 0) : 0;
    if (!count) { L.count = 0; L.blk[0] = 0; L.first = 0; }
    const int64_t n = L.blk[L.count];
    const uint32_t chunk = chunk_of(n, OPT_PARTS);
    const uint32_t gx = add ? (uint32_t)grid_of(n, chunk, OPT_PARTS) : grid;
    if (gx > 0) hipLaunchKernelGGL(grad_norm_kernel, dim3(gx), dim3(256), 0, (hipStream_t)stream, L, chunk, parts, add);
    M3D_CHECK_LAUNCH();
    add = 1;
  } while (i < count);
  *nparts = (int32_t)grid;
  return M3D_OK;
}

extern "C" int m3d_clip_grads(void* const* grads, const int64_t* numel, const int32_t* types, int32_t count, const double* parts,
                              int32_t nparts, double max_norm, float* norm_out, void* stream) {
  int64_t blocks = 0;
  const int rc = check_tensors(grads, numel, types, count, &blocks);
  if (rc != M3D_OK) return rc;
  if (!parts || nparts < 1 || nparts > OPT_PARTS || !(max_norm >= 0.0)) return M3D_ERR_INVALID;
  TensorList L;
  for (int32_t lists = (int32_t)m3d_cdiv(count, OPT_TENSORS), l = lists > 0 ? lists - 1 : 0; l >= 0; --l) {  // (last list first, see the kernel)
    if (count) fill_list(L, nullptr, grads, numel, types, l * OPT_TENSORS, count, 0);
    else { L.count = 0; L.blk[0] = 0; L.first = 0; }
    const int64_t n = L.blk[L.count];
    const uint32_t chunk = chunk_of(n, 2048);
    const int64_t gx = grid_of(n, chunk, 2048);
    if (gx == 0 && l > 0) continue;  // (the last launch writes the norm)
    hipLaunchKernelGGL(grad_clip_kernel, dim3((unsigned)(gx > 0 ? gx : 1)), dim3(256), 0, (hipStream_t)stream, L, chunk, parts, nparts, max_norm,
                       l == 0 ? norm_out : nullptr);
    M3D_CHECK_LAUNCH();
  }
  return M3D_OK;
}

extern "C" int m3d_adamw_step(const M3DAdamW* a, void* stream) {
  if (!a) return M3D_ERR_INVALID;
  int64_t blocks = 0, same = 0;
  int rc = check_tensors(a->params, a->numel, a->types, a->count, &blocks);
  if (rc == M3D_OK) rc = check_tensors(a->grads, a->numel, a->types, a->count, &same);
  if (rc != M3D_OK) return rc;
  if (!a->state || (a->count > 0 && !a->missed)) return M3D_ERR_INVALID;
  if (a->state_bits != 32 && a->state_bits != 8) return M3D_ERR_UNSUPPORTED;
  if (blocks > 0 && (!a->exp_avg || !a->exp_avg_sq || (a->state_bits == 8 && (!a->scale_avg || !a->scale_avg_sq)))) return M3D_ERR_INVALID;
  if ((((uintptr_t)a->exp_avg) | ((uintptr_t)a->exp_avg_sq)) & 15) return M3D_ERR_INVALID;
  for (int32_t i = 0; i < a->count; ++i)
    if (a->numel[i] > 0 && !a->params[i]) return M3D_ERR_INVALID;
  if (!(a->eps >= 0.0) || (a->state_bits == 8 && a->eps == 0.0)) return M3D_ERR_INVALID;
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0)) return M3D_ERR_INVALID;
  if (a->parts && (a->nparts < 1 || a->nparts > OPT_PARTS || !(a->max_norm >= 0.0))) return M3D_ERR_INVALID;
  AdamArgs A{};
  A.m = a->exp_avg; A.v = a->exp_avg_sq; A.ms = a->scale_avg; A.vs = a->scale_avg_sq;
  A.state = a->state; A.missed = a->missed; A.parts = a->parts; A.nparts = a->nparts; A.lr_dev = a->lr_dev;
  A.max_norm = a->max_norm; A.lr = a->lr; A.wd = a->weight_decay;
  // (the reciprocal instruction takes what is under 2^-126 for zero; an eps of zero stays one, as in the formula)
  A.eps = a->eps > 0.0 && a->eps < 0x1p-126 ? 0x1p-126f : (float)a->eps;
  A.b1 = a->beta1; A.b2 = a->beta2; A.c1 = 1.0 - a->beta1; A.c2 = 1.0 - a->beta2;
  A.log_b1 = log(a->beta1); A.log_b2 = log(a->beta2);
  double bytes = 0.0;
  for (int32_t i = 0; i < a->count; ++i)
    if (a->grads[i]) bytes += (double)a->numel[i] * (3 * (a->types[i] == M3D_TYPE_F32 ? 4 : 2) + (a->state_bits == 32 ? 16 : 4));
  const bool once = bytes > (double)M3D_CACHE_BYTES;
  TensorList L;
  const int32_t lists = (int32_t)m3d_cdiv(a->count > 0 ? a->count : 1, OPT_TENSORS);
  for (int32_t l = lists - 1; l >= 0; --l) {  // (last list first: against the order of the norm's pass)
    uint32_t start = 0;
    for (int32_t i = 0; i < l * OPT_TENSORS; ++i) start += (uint32_t)m3d_cdiv(a->numel[i], OPT_BLOCK);
    if (a->count) fill_list(L, a->params, a->grads, a->numel, a->types, l * OPT_TENSORS, a->count, start);
    else { L.count = 0; L.blk[0] = 0; L.first = 0; }
    const int64_t n = (int64_t)L.blk[L.count] - L.blk[0];
    A.bump = l == 0;
    A.norm_out = l == 0 ? a->norm_out : nullptr;
    const int64_t most = adamw_grid(a->state_bits);
    A.chunk = chunk_of(n, most);
    if (A.chunk < 4) A.chunk = 4;  // (a block for every wave)
    const int64_t gx = grid_of(n, A.chunk, most);
    if (gx == 0 && l > 0) continue;
    const dim3 grid((unsigned)(gx > 0 ? gx : 1));  // (the last launch counts the step)
    if (a->state_bits == 32) {
      if (once) hipLaunchKernelGGL((adamw_kernel<32, true>), grid, dim3(256), 0, (hipStream_t)stream, L, A);
      else hipLaunchKernelGGL((adamw_kernel<32, false>), grid, dim3(256), 0, (hipStream_t)stream, L, A);
    } else {
      if (once) hipLaunchKernelGGL((adamw_kernel<8, true>), grid, dim3(256), 0, (hipStream_t)stream, L, A);
      else hipLaunchKernelGGL((adamw_kernel<8, false>), grid, dim3(256), 0, (hipStream_t)stream, L, A);
    }
    M3D_CHECK_LAUNCH();
  }
  return M3D_OK;
}

extern "C" int m3d_moments_decode(const void* exp_avg, const void* exp_avg_sq, const float* scale_avg, const float* scale_avg_sq,
                                  float* avg_out, float* avg_sq_out, int64_t blocks, void* stream) {
  if (blocks < 0) return M3D_ERR_INVALID;
  if (blocks == 0) return M3D_OK;
  if (!exp_avg || !exp_avg_sq || !scale_avg || !scale_avg_sq || !avg_out || !avg_sq_out) return M3D_ERR_INVALID;
  if ((((uintptr_t)exp_avg) | ((uintptr_t)exp_avg_sq)) & 3 || (((uintptr_t)avg_out) | ((uintptr_t)avg_sq_out)) & 15) return M3D_ERR_INVALID;
  int64_t gx = m3d_cdiv(blocks, 4 * OPT_DECODE);
  if (gx > 1 << 20) gx = 1 << 20;
  hipLaunchKernelGGL(moments_decode_kernel, dim3((unsigned)gx), dim3(256), 0, (hipStream_t)stream, (const uint32_t*)exp_avg,
                     (const uint32_t*)exp_avg_sq, scale_avg, scale_avg_sq, (f32x4*)avg_out, (f32x4*)avg_sq_out, blocks);
  M3D_CHECK_LAUNCH();
  return M3D_OK;
}
extern "C" int m3d_moments_encode(const float* avg, const float* avg_sq, void* exp_avg, void* exp_avg_sq, float* scale_avg,
                                  float* scale_avg_sq, int64_t blocks, void* stream) {
  if (blocks < 0) return M3D_ERR_INVALID;
  if (blocks == 0) return M3D_OK;
  if (!exp_avg || !exp_avg_sq || !scale_avg || !scale_avg_sq || !avg || !avg_sq) return M3D_ERR_INVALID;
  if ((((uintptr_t)exp_avg) | ((uintptr_t)exp_avg_sq)) & 3 || (((uintptr_t)avg) | ((uintptr_t)avg_sq)) & 15) return M3D_ERR_INVALID;
  int64_t gx = m3d_cdiv(blocks, 4);
  if (gx > 4096) gx = 4096;
  hipLaunchKernelGGL(moments_encode_kernel, dim3((unsigned)gx), dim3(256), 0, (hipStream_t)stream, (const f32x4*)avg, (const f32x4*)avg_sq,
                     (uint32_t*)exp_avg, (uint32_t*)exp_avg_sq, scale_avg, scale_avg_sq, blocks);
  M3D_CHECK_LAUNCH();
  return M3D_OK;
}
