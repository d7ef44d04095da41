// Rows of 8-bit floats: e4m3 codes with an f32 scale per block of 128 columns, from plain rows, from silu(gate) * up, and from an
// RMSNorm with the residual's addition.
//
// With a = the block's largest magnitude: scale = a / 448, code = e4m3(v * (448 / a)), rounded to nearest even. a is taken as at least
// 7 * 2^-120, so that both quotients are normal numbers (a block of zeros has codes of zero); a block with a value that is not finite
// has a NaN for its scale and for every code.
//
// Bound: HBM (each input read once, one byte written per value and four per block), and for 16-bit inputs instruction issue next to it:
// a lane holds 32 bytes of an input, so that a block of 128 columns is 16 lanes of f32 or 8 lanes of 16-bit values and what is done once
// per lane and block (maximum, quotients) counts for 8 or 16 values.
#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "qgemv_common.cuh"
#include "state_columns.cuh"

namespace {

constexpr int F8_BLOCK = 128;
constexpr float F8_TOP = 448.f, F8_LEAST = 0x7p-120f;
constexpr int NORM_MAX_COLS = 32768, NORM_PIECE = 8;

// A lane's piece of a row: E values as they are held
template <typename T, int E>
struct Piece {
  static constexpr int WORDS = E * (int)sizeof(T) / 4;
  uint32_t w[WORDS];
};

template <typename T, int E>
__device__ __forceinline__ void f8_unpack(const Piece<T, E>& r, float (&v)[E]) {
#pragma unroll
  for (int i = 0; i < Piece<T, E>::WORDS; ++i) {
    if (sizeof(T) == 4) {
      v[i] = __uint_as_float(r.w[i]);
    } else if (std::is_same<T, __half>::value) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
      v[2 * i % E] = f.x; v[(2 * i + 1) % E] = f.y;
    } else {
      v[2 * i % E] = __uint_as_float(r.w[i] << 16); v[(2 * i + 1) % E] = __uint_as_float(r.w[i] & 0xFFFF0000u);
    }
  }
}

// The lane's piece of a row from column c on; columns from n on are zero. vec: 16-byte loads are aligned. Coherent loads: a sum may be
// written where its operand was read.
template <int E, typename T>
__device__ __forceinline__ Piece<T, E> f8_load(const T* row, int c, int n, bool vec) {
  constexpr int WORDS = Piece<T, E>::WORDS;
  Piece<T, E> r;
  if (vec && c + E <= n) {
#pragma unroll
    for (int h = 0; h < WORDS; h += 4)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.w[h]), "=r"(r.w[h + 1]), "=r"(r.w[h + 2]), "=r"(r.w[h + 3]) : "l"(row + c + h * (4 / sizeof(T))) : "memory");
    return r;
  }
#pragma unroll
  for (int i = 0; i < WORDS; ++i) r.w[i] = 0;
  if (c < n) {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (c + i < n) {
        if (sizeof(T) == 4) r.w[i % WORDS] = reinterpret_cast<const uint32_t*>(row)[c + i];
        else r.w[i / 2 % WORDS] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[c + i] << (16 * (i & 1));
      }
  }
  return r;
}

// The largest magnitude of a lane's values as f32 bits; these order magnitudes, with what is not finite above all. f32 values are compared
// three at a time (a NaN wins), 16-bit values two at a time as they are.
template <int E>
__device__ __forceinline__ uint32_t f8_top(const float (&v)[E]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < E; i += 2) asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(v[i]), "f"(v[i + 1]));
  return __float_as_uint(top) & 0x7FFFFFFFu;
}
template <typename T, int E>
__device__ __forceinline__ uint32_t f8_top_packed(const Piece<T, E>& r) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < Piece<T, E>::WORDS; ++i) top = __vmaxu2(top, r.w[i] & 0x7FFF7FFFu);
  const uint32_t one = max(top >> 16, top & 0xFFFFu);
  return std::is_same<T, __half>::value ? __float_as_uint(__half2float(__ushort_as_half((unsigned short)one))) : one << 16;
}

// a / b from an approximate reciprocal y of b: one correction by the exact remainder (Markstein 1990)
__device__ __forceinline__ float f8_quotient(float a, float b, float y) {
  const float q = a * y;
  return fmaf(fmaf(-q, b, a), y, q);
}

// Codes and scale of a block whose values are spread over 128 / E neighbouring lanes, E from column c on in each, with the lane's own
// largest magnitude; every lane of the warp calls it. code_row and scale_row begin at the row's first column and block; a lane without a
// column writes nothing.
template <int E>
__device__ __forceinline__ void f8_emit(const float (&v)[E], uint32_t top, int c, int n, uint8_t* code_row, float* scale_row) {
  constexpr int LANES = F8_BLOCK / E;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if (c >= n) return;
  const bool finite = top < 0x7F800000u;
  const float a = fmaxf(__uint_as_float(top), F8_LEAST), nan = __uint_as_float(0x7FFFFFFFu);
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(a));
  const float r = finite ? f8_quotient(F8_TOP, a, y) : nan;
  if ((threadIdx.x & (LANES - 1)) == 0) scale_row[c / F8_BLOCK] = finite ? f8_quotient(a, F8_TOP, 1.0f / F8_TOP) : nan;
  uint32_t q[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i) {
    const float2 lo = mul2(make_float2(v[4 * i], v[4 * i + 1]), make_float2(r, r)), hi = mul2(make_float2(v[4 * i + 2], v[4 * i + 3]), make_float2(r, r));
    q[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) | (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16;
  }
  if (c + E <= n) {  // rows of codes begin on 16 bytes
    if (E == 16) *reinterpret_cast<uint4*>(code_row + c) = make_uint4(q[0], q[1], q[E / 4 - 2], q[E / 4 - 1]);
    else *reinterpret_cast<uint2*>(code_row + c) = make_uint2(q[0], q[1]);
  } else {
    for (int i = 0; c + i < n; ++i) code_row[c + i] = (uint8_t)(q[i >> 2] >> (8 * (i & 3)));
  }
}

// silu(g) u = g u / (1 + exp(-g)), with the fast exponential (2 + 1.2 |g| units of its last place) and quotient (2 units): a code keeps
// four bits. Divisors above 2^126 (g below -87.3) give 0.
__device__ __forceinline__ float f8_silu_mul(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

// Blocks by themselves: a warp takes STEPS x 32 x PER_LANE columns of a row, `wpr` warps stand side by side in a row. Its pieces
// stay packed until their turn.
constexpr int ROW_WARPS = 8, STEPS = 2;
template <typename T>
constexpr int PER_LANE = 32 / (int)sizeof(T);

template <typename T, bool GATED>
__global__ void __launch_bounds__(ROW_WARPS * 32)
quantize_f8_kernel(const T* x, size_t ldx, const T* gate, size_t ldg, bool vec, size_t rows, int n, int wpr, uint8_t* codes, size_t ld,
                   float* scales) {
  constexpr int E = PER_LANE<T>, SPAN = 32 * E;
  pdl_launch_dependents_small();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, above = warp / wpr;
  const size_t row = (size_t)blockIdx.x * (blockDim.x / 32 / wpr) + above;
  const int c0 = ((int)blockIdx.y * wpr + warp - above * wpr) * (STEPS * SPAN) + lane * E;
  if (row >= rows || c0 - lane * E >= n) return;
  const T* xr = x + row * ldx;
  const T* gr = GATED ? gate + row * ldg : nullptr;
  Piece<T, E> xs[STEPS], gs[GATED ? STEPS : 1];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    xs[s] = f8_load<E>(xr, c0 + s * SPAN, n, vec);
    if (GATED) gs[GATED ? s : 0] = f8_load<E>(gr, c0 + s * SPAN, n, vec);
  }
  uint8_t* code_row = codes + row * ld;
  float* scale_row = scales + row * (size_t)((n + F8_BLOCK - 1) / F8_BLOCK);
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    if (c0 - lane * E + s * SPAN >= n) break;
    float v[E];
    f8_unpack(xs[s], v);
    if (GATED) {
      float g[E];
      f8_unpack(gs[GATED ? s : 0], g);
#pragma unroll
      for (int i = 0; i < E; ++i) v[i] = f8_silu_mul(g[i], v[i]);
    }
    f8_emit(v, GATED || sizeof(T) == 4 ? f8_top(v) : f8_top_packed(xs[s]), c0 + s * SPAN, n, code_row, scale_row);
  }
}

__device__ __forceinline__ uint32_t f8_pair(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t f8_pair(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t f8_pair(float a, float, float) { return __float_as_uint(a); }
template <int E, typename T>
__device__ __forceinline__ void f8_store(T* row, int c, int n, bool vec, const float (&v)[E]) {
  constexpr int WORDS = Piece<T, E>::WORDS, STEP = 4 / (int)sizeof(T);
  uint32_t q[WORDS];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) q[i] = f8_pair(v[STEP * i], v[STEP * i + STEP - 1], T());
  if (vec && c + E <= n) {
#pragma unroll
    for (int h = 0; h < WORDS; h += 4) *reinterpret_cast<uint4*>(row + c + h * STEP) = make_uint4(q[h], q[h + 1], q[h + 2], q[h + 3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (c + i < n) {
      if (sizeof(T) == 4) reinterpret_cast<uint32_t*>(row)[c + i] = q[i % WORDS];
      else reinterpret_cast<uint16_t*>(row)[c + i] = (uint16_t)(q[i / 2 % WORDS] >> (16 * (i & 1)));
    }
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

// A row per CTA at a time, kept in registers between its sum of squares and its norm: CHUNKS pieces a thread. AHEAD: the CTA's next row is
// asked for before this one's sum is complete, and with one piece a thread the weight stays in registers from row to row. The sum of
// squares and the norm are of the unrounded sum x + residual; sum_dev gets it rounded to the type of x, once.
template <typename T, int CHUNKS, bool AHEAD>
__global__ void __launch_bounds__(1024)
rms_norm_f8_kernel(const NormArgs<T> a, size_t rows) {
  constexpr int E = NORM_PIECE;
  __shared__ float sh[2][32];
  pdl_launch_dependents_small();
  pdl_wait();
  const int tid = threadIdx.x, threads = blockDim.x;
  Piece<T, E> xs[CHUNKS], rs[CHUNKS];
  auto fetch = [&](size_t row) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) xs[i] = f8_load<E>(a.x + row * a.ldx, (i * threads + tid) * E, a.n, a.vec);
    if (a.res)
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) rs[i] = f8_load<E>(a.res + row * a.ldr, (i * threads + tid) * E, a.n, a.vec);
  };
  constexpr bool KEEP = AHEAD && CHUNKS == 1;
  if (AHEAD) fetch(blockIdx.x);
  float kept[KEEP ? CHUNKS : 1][E];
  if (KEEP)
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) f8_vector(a.w, (i * threads + tid) * E, a.n, a.wvec, kept[KEEP ? i : 0]);
  int turn = 0;
#pragma unroll 1
  for (size_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    float v[CHUNKS][E];
    float ss = 0.f;
    if (!AHEAD) fetch(row);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      f8_unpack(xs[i], v[i]);
      if (a.res) {
        float r[E];
        f8_unpack(rs[i], r);
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] += r[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(v[i][e], v[i][e], ss);
    }
    if (AHEAD && row + gridDim.x < rows) fetch(row + gridDim.x);
    if (a.sum) {
      T* sr = a.sum + row * a.lds;
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) f8_store(sr, (i * threads + tid) * E, a.n, a.vec, v[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
    if ((tid & 31) == 0) sh[turn][tid >> 5] = ss;
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < (threads >> 5); ++i) ss += sh[turn][i];
    const float inv = 1.0f / sqrtf(ss / (float)a.n + a.eps);
    uint8_t* code_row = a.codes + row * a.ld;
    float* scale_row = a.scales + row * (size_t)((a.n + F8_BLOCK - 1) / F8_BLOCK);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = (i * threads + tid) * E;
      float w[E];
      if (!KEEP) f8_vector(a.w, c, a.n, a.wvec, w);
#pragma unroll
      for (int e = 0; e < E; ++e) v[i][e] = v[i][e] * inv * (KEEP ? kept[KEEP ? i : 0][e] : w[e]);
      if (a.b) {
        f8_vector(a.b, c, a.n, a.wvec, w);
#pragma unroll
        for (int e = 0; e < E; ++e) v[i][e] += w[e];
      }
      f8_emit(v[i], f8_top(v[i]), c, a.n, code_row, scale_row);
    }
  }
}

template <typename T>
bool f8_aligned(const void* p, size_t ld) { return !p || ((uintptr_t)p % 16 == 0 && ld * sizeof(T) % 16 == 0); }

template <typename T, bool GATED>
int launch_quantize(fb200_device* dev, const void* x, size_t ldx, const void* gate, size_t ldg, size_t rows, size_t n, uint8_t* codes, size_t ld,
                    float* scales) {
  const int span = STEPS * 32 * PER_LANE<T>, spans = (int)((n + span - 1) / span);
  const int wpr = spans < ROW_WARPS ? spans : ROW_WARPS, rpc = ROW_WARPS / wpr;  // warps side by side, rows of a CTA
  const dim3 grid((unsigned)((rows + rpc - 1) / rpc), (unsigned)((spans + wpr - 1) / wpr));
  const bool vec = f8_aligned<T>(x, ldx) && f8_aligned<T>(gate, ldg);
  return fb200_launch(dev, quantize_f8_kernel<T, GATED>, grid, dim3(wpr * rpc * 32), 0, true, (const T*)x, ldx, (const T*)gate, ldg, vec, rows,
                      (int)n, wpr, codes, ld, scales);
}

template <typename T, int CHUNKS, bool AHEAD>
int launch_norm_chunks(fb200_device* dev, const NormArgs<T>& a, size_t rows) {
  const int per = CHUNKS * NORM_PIECE, threads = ((a.n + per - 1) / per + 31) / 32 * 32;
  const size_t places = (size_t)dev->sm_count * (size_t)(1024 / threads);  // 64 registers a thread: 1024 threads an SM
  return fb200_launch(dev, rms_norm_f8_kernel<T, CHUNKS, AHEAD>, dim3((unsigned)std::min(rows, places)), dim3((unsigned)threads), 0, true, a, rows);
}

// Values a thread, by what they take with the next row's beside them in 64 registers. 8192 rows of 4096 with a residual: f32 71.7 us with 8,
// 74.9 with 16 (rows of 8192, where 8 leave one CTA to an SM: 83.2 and 74.8 for 4096 rows); bf16 46.2 with 8, 41.9 with 16.
template <typename T>
int launch_norm(fb200_device* dev, const NormArgs<T>& a, size_t rows) {
  if (sizeof(T) == 4 && a.n <= 4096) return launch_norm_chunks<T, 1, true>(dev, a, rows);
  if (a.n <= 1024 * 16) return launch_norm_chunks<T, 2, true>(dev, a, rows);
  return launch_norm_chunks<T, 4, false>(dev, a, rows);
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
