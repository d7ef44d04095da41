// Rows of 8-bit floats: e4m3 codes with an f32 scale per block of 128 columns, from plain rows, from silu(gate) * up, and from an
// RMSNorm with the residual's addition.
//
// With a = the block's largest magnitude: scale = a / 448, code = e4m3(v * (448 / a)), rounded to nearest even. a is taken as at least
// 7 * 2^-120, so that both quotients are normal numbers (a block of zeros has codes of zero); a block with a value that is not finite
// has a NaN for its scale and for every code.
//
// Bound: HBM (each input read once, one byte written per value and four per block). A lane holds 16 bytes of an input, so a
// block of 128 columns is 32 lanes of f32 or 16 lanes of 16-bit values, and its maximum takes five or four shuffles.
#include <cuda_fp8.h>

#include <cmath>

#include "qgemv_common.cuh"

namespace {

constexpr int F8_BLOCK = 128;
constexpr float F8_TOP = 448.f, F8_LEAST = 0x7p-120f;
constexpr int NORM_MAX_COLS = 32768;

template <typename T>
constexpr int PER_LANE = 16 / (int)sizeof(T);

__device__ __forceinline__ float f8_float(float v) { return v; }
__device__ __forceinline__ float f8_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float f8_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ void f8_unpack(const uint4& r, float (&v)[4], float) {
  v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
}
__device__ __forceinline__ void f8_unpack(const uint4& r, float (&v)[8], __half) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x; v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void f8_unpack(const uint4& r, float (&v)[8], __nv_bfloat16) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
}

// The lane's values from column c on, as f32; columns from n on are zero. vec: 16-byte loads are aligned. Coherent loads: a sum may be
// written where its operand was read.
template <typename T>
__device__ __forceinline__ void f8_load(const T* row, int c, int n, bool vec, float (&v)[PER_LANE<T>]) {
  if (vec && c + PER_LANE<T> <= n) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(row + c) : "memory");
    f8_unpack(r, v, T());
  } else {
#pragma unroll
    for (int i = 0; i < PER_LANE<T>; ++i) v[i] = c + i < n ? f8_float(row[c + i]) : 0.f;
  }
}

// Codes and scale of a block whose values are spread over 128 / E neighbouring lanes, E from column c on in each; every lane of the
// warp calls it. code_row and scale_row begin at the row's first column and block; a lane without a column writes nothing.
template <int E>
__device__ __forceinline__ void f8_emit(const float (&v)[E], int c, int n, uint8_t* code_row, float* scale_row) {
  constexpr int LANES = F8_BLOCK / E;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < E; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);  // in the order of magnitudes, NaN above all
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (c >= n) return;
  const bool finite = top < 0x7F800000u;
  const float a = fmaxf(__uint_as_float(top), F8_LEAST), nan = __uint_as_float(0x7FFFFFFFu);
  const float r = finite ? F8_TOP / a : nan;
  if ((threadIdx.x & (LANES - 1)) == 0) scale_row[c / F8_BLOCK] = finite ? a / F8_TOP : nan;
  uint32_t q[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i)
    q[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i] * r, v[4 * i + 1] * r), __NV_SATFINITE, __NV_E4M3) |
           (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2] * r, v[4 * i + 3] * r), __NV_SATFINITE, __NV_E4M3) << 16;
  if (c + E <= n) {  // rows of codes begin on 16 bytes
    if (E == 8) *reinterpret_cast<uint2*>(code_row + c) = make_uint2(q[0], q[E / 4 - 1]);
    else *reinterpret_cast<uint32_t*>(code_row + c) = q[0];
  } else {
    for (int i = 0; c + i < n; ++i) code_row[c + i] = (uint8_t)(q[i >> 2] >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ float f8_silu_mul(float g, float u) { return g / (1.0f + expf(-g)) * u; }

// Blocks by themselves: a warp takes STEPS x 32 x PER_LANE columns of a row, `wpr` warps of a CTA stand side by side in a row.
constexpr int ROW_WARPS = 8, STEPS = 4;

template <typename T, bool GATED>
__global__ void __launch_bounds__(ROW_WARPS * 32)
quantize_f8_kernel(const T* x, size_t ldx, const T* gate, size_t ldg, bool vec, size_t rows, int n, int wpr, uint8_t* codes, size_t ld,
                   float* scales) {
  constexpr int E = PER_LANE<T>, SPAN = 32 * E;
  pdl_launch_dependents_small();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, side = warp % wpr;
  const size_t row = (size_t)blockIdx.x * (ROW_WARPS / wpr) + warp / wpr;
  const int c0 = ((int)blockIdx.y * wpr + side) * (STEPS * SPAN) + lane * E;
  if (row >= rows || c0 - lane * E >= n) return;
  const T* xr = x + row * ldx;
  const T* gr = GATED ? gate + row * ldg : nullptr;
  float v[STEPS][E], g[GATED ? STEPS : 1][E];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    f8_load(xr, c0 + s * SPAN, n, vec, v[s]);
    if (GATED) f8_load(gr, c0 + s * SPAN, n, vec, g[GATED ? s : 0]);
  }
  uint8_t* code_row = codes + row * ld;
  float* scale_row = scales + row * (size_t)((n + F8_BLOCK - 1) / F8_BLOCK);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    if (GATED)
#pragma unroll
      for (int i = 0; i < E; ++i) v[s][i] = f8_silu_mul(g[GATED ? s : 0][i], v[s][i]);
    f8_emit(v[s], c0 + s * SPAN, n, code_row, scale_row);
  }
}

__device__ __forceinline__ void f8_store(float* row, int c, int n, bool vec, const float (&v)[4]) {
  if (vec && c + 4 <= n) *reinterpret_cast<float4*>(row + c) = make_float4(v[0], v[1], v[2], v[3]);
  else
    for (int i = 0; i < 4; ++i)
      if (c + i < n) row[c + i] = v[i];
}
__device__ __forceinline__ uint32_t f8_pair(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t f8_pair(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
__device__ __forceinline__ void f8_store(T* row, int c, int n, bool vec, const float (&v)[8]) {
  uint32_t q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) q[i] = f8_pair(v[2 * i], v[2 * i + 1], T());
  if (vec && c + 8 <= n) *reinterpret_cast<uint4*>(row + c) = make_uint4(q[0], q[1], q[2], q[3]);
  else
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < n) reinterpret_cast<uint16_t*>(row)[c + i] = (uint16_t)(q[i >> 1] >> (16 * (i & 1)));
}
// E values of an f32 vector of n from column c on, zeros behind it
template <int E>
__device__ __forceinline__ void f8_vector(const float* w, int c, int n, bool vec, float (&v)[E]) {
  if (vec && c + E <= n) {
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const float4 f = *reinterpret_cast<const float4*>(w + c + 4 * i);
      v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = c + i < n ? w[c + i] : 0.f;
  }
}

template <typename T>
struct NormArgs {
  const T *x, *res;
  T* sum;
  const float *w, *b;
  size_t ldx, ldr, lds, ld;
  uint8_t* codes;
  float* scales;
  float eps;
  int n;
  bool vec, wvec;
};

// A row per CTA, kept in registers between its sum of squares and its norm: CHUNKS x PER_LANE values a thread. The sum of squares and
// the norm are of the unrounded sum x + residual; sum_dev gets it rounded to the type of x, once.
template <typename T, int CHUNKS>
__global__ void __launch_bounds__(1024)
rms_norm_f8_kernel(const NormArgs<T> a) {
  constexpr int E = PER_LANE<T>;
  __shared__ float sh[32];
  pdl_launch_dependents_small();
  pdl_wait();
  const size_t row = blockIdx.x;
  const int tid = threadIdx.x, threads = blockDim.x;
  const T* xr = a.x + row * a.ldx;
  float v[CHUNKS][E];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) f8_load(xr, (i * threads + tid) * E, a.n, a.vec, v[i]);
  if (a.res) {
    const T* rr = a.res + row * a.ldr;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      float r[E];
      f8_load(rr, (i * threads + tid) * E, a.n, a.vec, r);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] += r[e];
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) ss = fmaf(v[i][e], v[i][e], ss);
  if (a.sum) {
    T* sr = a.sum + row * a.lds;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) f8_store(sr, (i * threads + tid) * E, a.n, a.vec, v[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
  if ((tid & 31) == 0) sh[tid >> 5] = ss;
  __syncthreads();
  ss = 0.f;
  for (int i = 0; i < (threads >> 5); ++i) ss += sh[i];
  const float inv = 1.0f / sqrtf(ss / (float)a.n + a.eps);
  uint8_t* code_row = a.codes + row * a.ld;
  float* scale_row = a.scales + row * (size_t)((a.n + F8_BLOCK - 1) / F8_BLOCK);
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = (i * threads + tid) * E;
    float w[E];
    f8_vector(a.w, c, a.n, a.wvec, w);
#pragma unroll
    for (int e = 0; e < E; ++e) v[i][e] = v[i][e] * inv * w[e];
    if (a.b) {
      f8_vector(a.b, c, a.n, a.wvec, w);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] += w[e];
    }
    f8_emit(v[i], c, a.n, code_row, scale_row);
  }
}

template <typename T>
bool f8_aligned(const void* p, size_t ld) { return !p || ((uintptr_t)p % 16 == 0 && ld * sizeof(T) % 16 == 0); }

template <typename T, bool GATED>
int launch_quantize(fb200_device* dev, const void* x, size_t ldx, const void* gate, size_t ldg, size_t rows, size_t n, uint8_t* codes, size_t ld,
                    float* scales) {
  const int span = STEPS * 32 * PER_LANE<T>, spans = (int)((n + span - 1) / span);
  int wpr = 1;
  while (wpr < ROW_WARPS && wpr < spans) wpr *= 2;
  const dim3 grid((unsigned)((rows + ROW_WARPS / wpr - 1) / (ROW_WARPS / wpr)), (unsigned)((spans + wpr - 1) / wpr));
  const bool vec = f8_aligned<T>(x, ldx) && f8_aligned<T>(gate, ldg);
  return fb200_launch(dev, quantize_f8_kernel<T, GATED>, grid, dim3(ROW_WARPS * 32), 0, true, (const T*)x, ldx, (const T*)gate, ldg, vec, rows,
                      (int)n, wpr, codes, ld, scales);
}

template <typename T, int CHUNKS>
int launch_norm_chunks(fb200_device* dev, const NormArgs<T>& a, size_t rows) {
  const int per = CHUNKS * PER_LANE<T>, threads = ((a.n + per - 1) / per + 31) / 32 * 32;
  return fb200_launch(dev, rms_norm_f8_kernel<T, CHUNKS>, dim3((unsigned)rows), dim3((unsigned)threads), 0, true, a);
}

template <typename T>
int launch_norm(fb200_device* dev, const NormArgs<T>& a, size_t rows) {
  constexpr int E = PER_LANE<T>;
  // 16 values a thread, or more where a row would take over 1024 threads
  if (a.n <= 1024 * 16) return launch_norm_chunks<T, 16 / E>(dev, a, rows);
  return launch_norm_chunks<T, 32 / E>(dev, a, rows);
}

// What the operations on rows have in common: n columns a row, codes that begin on 16 bytes in every row
int check_rows(fb200_device* dev, const char* op, size_t rows, size_t n, uint32_t type, const uint8_t* codes, size_t ld, const float* scales) {
  if (type != FB200_F32 && type != FB200_F16 && type != FB200_BF16)
    return fb200_fail(dev, FB200_ERR_UNSUPPORTED_DTYPE, "%s: rows of type %u (F32, F16 or BF16)", op, type);
  if (rows >= (1ull << 31) || n > (1ull << 27)) return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "%s: %zu rows of %zu are too many", op, rows, n);
  if (!codes || !scales) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "%s: null output", op);
  if (ld < n || ld % 16 || (uintptr_t)codes % 16 || (uintptr_t)scales % 4)
    return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "%s: rows of %zu codes every %zu bytes (a multiple of 16, from a multiple of 16 on)", op, n, ld);
  return FB200_OK;
}
int check_input(fb200_device* dev, const char* op, const char* what, const void* p, size_t ld, size_t n, uint32_t type) {
  if (!p) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "%s: %s is null", op, what);
  if (ld < n || (uintptr_t)p % (type == FB200_F32 ? 4 : 2))
    return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "%s: %s has rows of %zu values every %zu, or is not aligned to them", op, what, n, ld);
  return FB200_OK;
}

template <bool GATED>
int quantize(fb200_device* dev, const char* op, const void* x, size_t ldx, const void* gate, size_t ldg, uint32_t type, size_t rows, size_t n,
             uint8_t* codes, size_t ld, float* scales) {
  const double size = type == FB200_F32 ? 4 : 2;
  fb200_op_trace scope(dev, op, (double)rows * (double)n * (size * (GATED ? 2 : 1) + 1.03125));
  if (type == FB200_F32) return launch_quantize<float, GATED>(dev, x, ldx, gate, ldg, rows, n, codes, ld, scales);
  if (type == FB200_F16) return launch_quantize<__half, GATED>(dev, x, ldx, gate, ldg, rows, n, codes, ld, scales);
  return launch_quantize<__nv_bfloat16, GATED>(dev, x, ldx, gate, ldg, rows, n, codes, ld, scales);
}

template <typename T>
int norm(fb200_device* dev, const void* x, size_t ldx, const void* res, size_t ldr, void* sum, size_t lds, const float* w, const float* b, float eps,
         size_t rows, size_t n, uint8_t* codes, size_t ld, float* scales) {
  NormArgs<T> a = {(const T*)x, (const T*)res, (T*)sum, w, b, ldx, ldr, lds, ld, codes, scales, eps, (int)n, false, false};
  a.vec = f8_aligned<T>(x, ldx) && f8_aligned<T>(res, ldr) && f8_aligned<T>(sum, lds);
  a.wvec = (uintptr_t)w % 16 == 0 && (uintptr_t)b % 16 == 0;
  return launch_norm(dev, a, rows);
}

}  // namespace

extern "C" {

int fb200_quantize_f8(fb200_device* dev, const void* x_dev, size_t ldx, uint32_t type, size_t rows, size_t n, uint8_t* codes_dev, size_t ld,
                      float* scales_dev) {
  int rc = fb200_bind(dev);
  if (rc || (rc = check_rows(dev, "quantize_f8", rows, n, type, codes_dev, ld, scales_dev)) ||
      (rc = check_input(dev, "quantize_f8", "x", x_dev, ldx, n, type)))
    return rc;
  if (rows == 0 || n == 0) return FB200_OK;
  return quantize<false>(dev, "quantize_f8", x_dev, ldx, nullptr, 0, type, rows, n, codes_dev, ld, scales_dev);
}

int fb200_silu_mul_f8(fb200_device* dev, const void* gate_dev, size_t ldgate, const void* up_dev, size_t ldup, uint32_t type, size_t rows, size_t n,
                      uint8_t* codes_dev, size_t ld, float* scales_dev) {
  int rc = fb200_bind(dev);
  if (rc || (rc = check_rows(dev, "silu_mul_f8", rows, n, type, codes_dev, ld, scales_dev)) ||
      (rc = check_input(dev, "silu_mul_f8", "gate", gate_dev, ldgate, n, type)) || (rc = check_input(dev, "silu_mul_f8", "up", up_dev, ldup, n, type)))
    return rc;
  if (rows == 0 || n == 0) return FB200_OK;
  return quantize<true>(dev, "silu_mul_f8", up_dev, ldup, gate_dev, ldgate, type, rows, n, codes_dev, ld, scales_dev);
}

int fb200_rms_norm_f8(fb200_device* dev, const void* x_dev, size_t ldx, const void* residual_dev, size_t ldres, void* sum_dev, size_t ldsum,
                      uint32_t type, const float* weight_dev, const float* bias_dev, float eps, size_t rows, size_t n, uint8_t* codes_dev, size_t ld,
                      float* scales_dev) {
  int rc = fb200_bind(dev);
  if (rc || (rc = check_rows(dev, "rms_norm_f8", rows, n, type, codes_dev, ld, scales_dev)) ||
      (rc = check_input(dev, "rms_norm_f8", "x", x_dev, ldx, n, type)) ||
      (residual_dev && (rc = check_input(dev, "rms_norm_f8", "residual", residual_dev, ldres, n, type))) ||
      (sum_dev && (rc = check_input(dev, "rms_norm_f8", "sum", sum_dev, ldsum, n, type))))
    return rc;
  if (!weight_dev || (uintptr_t)weight_dev % 4 || (uintptr_t)bias_dev % 4)
    return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "rms_norm_f8: the weight is null, or weight or bias is not aligned");
  if (n > NORM_MAX_COLS) return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "rms_norm_f8: rows of %zu values (at most %d)", n, NORM_MAX_COLS);
  if (rows == 0 || n == 0) return FB200_OK;
  const double size = type == FB200_F32 ? 4 : 2;
  fb200_op_trace scope(dev, "rms_norm_f8", (double)rows * (double)n * (size * (1 + (residual_dev != nullptr) + (sum_dev != nullptr)) + 1.03125));
  if (type == FB200_F32)
    return norm<float>(dev, x_dev, ldx, residual_dev, ldres, sum_dev, ldsum, weight_dev, bias_dev, eps, rows, n, codes_dev, ld, scales_dev);
  if (type == FB200_F16)
    return norm<__half>(dev, x_dev, ldx, residual_dev, ldres, sum_dev, ldsum, weight_dev, bias_dev, eps, rows, n, codes_dev, ld, scales_dev);
  return norm<__nv_bfloat16>(dev, x_dev, ldx, residual_dev, ldres, sum_dev, ldsum, weight_dev, bias_dev, eps, rows, n, codes_dev, ld, scales_dev);
}

}  // extern "C"
