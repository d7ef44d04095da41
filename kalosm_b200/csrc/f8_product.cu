// Products of 8-bit floats: rows of e4m3 codes with an f32 scale per block of 128 columns, times a matrix of e4m3 codes with an f32
// scale per block of 128 x 128.
//
//   y[m, n] = sum over blocks b of 128 columns of  sx[m, b] sw[n / 128, b] * (sum over k in b of x[m, k] w[n, k])   (+ residual or bias)
//
// The inner sum is one accumulation of the tensor cores (tcgen05.mma kind::f8f6f4, f32 in tensor memory): a block of 128 codes is exactly
// one row of a 128-byte swizzled operand and four MMAs. The outer sum is kept in f32 registers: the epilogue warps take each block's
// accumulator out of tensor memory while the tensor cores fill the next one, and add it under its scale.
//
// Three kernels, by the number of rows (f8_product has the rule and what it was measured on):
//  * f8_few_kernel, up to 32: 128 weight rows (in the M role) by 16 or 32 activation rows per CTA, K split over a cluster whose CTAs send
//    their sums to their owner through distributed shared memory. Bound: HBM, N K bytes. One row of 4096 x 4096: 5.4 us (3.1 TB/s, launches
//    one after the other; half of it is set-up and the hand-over of sums), of 28672 x 4096: 20.1 us (5.8 TB/s);
//  * f8_some_kernel, to a few hundred: 64 or 128 activation rows (in the M role, so that a thread has one row and one scale) by 128 weight
//    rows, K split over clusters of up to four. Bound: HBM, then what an SM takes in from L2 (94 GB/s measured). 128 rows of
//    4096 x 14336: 16.4 us (3.7 TB/s, 0.92 PFLOP/s);
//  * f8_pair_kernel: CTA pairs, 256 activation rows by 128, 192 or 256 weight rows, persistent. Bound: what the SMs take in from L2 (32 KB per pair
//    tile and block and SM: without its MMAs the kernel takes 0.9 of its time) and the power limit. 8192 rows of 28672 x 4096: 831 us
//    (2.3 PFLOP/s), 930 us at the 1.4 GHz that 950 W leave in a long run.
// Every wait is bounded (2^22 polls): one that gives up sets the device status word and a flag that makes the other roles leave; copies
// and MMAs in flight are waited for, TMEM is released on every path.
#include <cstdlib>
#include <new>

#include "dense.cuh"
#include "state_columns.cuh"
#include "tcgen05.cuh"

// A matrix [n, k] of codes, `ld` bytes from row to row, and its scales [ceil(n / 128), ceil(k / 128)]
struct fb200_f8matrix {
  fb200_device* dev = nullptr;
  uint64_t n = 0, k = 0;
  size_t ld = 0;
  uint8_t* codes = nullptr;
  float* scales = nullptr;
  bool owned = false;
  CUtensorMap map128, map64, map48;  // boxes of 128, 64 and 48 rows
};

namespace {

constexpr int F8_BLOCK = 128, F8_A_BYTES = 128 * 128;

struct F8Out {
  void* y;
  uint32_t type;
  const float *r1, *r2, *bias;
  int m, n;
  int vec;   // four columns of y (and of the residuals) are aligned
  int pack;  // 16-bit y without residual or bias, eight columns aligned: rounded before they are turned
};

constexpr int TURN_BYTES = 32 * 128;  // a warp's 32 rows x 128 bytes on their way out, 16-byte piece p of row r at place p ^ (r % 8)

// Two outputs in 16 bits
__device__ __forceinline__ uint32_t f8_pair(const F8Out& o, float2 v) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return o.type == FB200_BF16 ? *reinterpret_cast<const uint32_t*>(&b) : *reinterpret_cast<const uint32_t*>(&h);
}
// One output, and four neighbouring ones (o.vec), rounded; `at` counts elements
__device__ __forceinline__ void f8_put(const F8Out& o, float v, size_t at) {
  if (o.type == FB200_F32) reinterpret_cast<float*>(o.y)[at] = v;
  else reinterpret_cast<uint16_t*>(o.y)[at] = (uint16_t)f8_pair(o, make_float2(v, 0.f));
}
__device__ __forceinline__ void f8_put4(const F8Out& o, const float4& v, size_t at) {
  if (o.type == FB200_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(o.y) + at) = v;
  else *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(o.y) + at) = make_uint2(f8_pair(o, make_float2(v.x, v.y)), f8_pair(o, make_float2(v.z, v.w)));
}
__device__ __forceinline__ float4 f8_add(const float4& a, const float4& b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
// Columns n .. n + 3 of a vector of N or of a row of a matrix of N columns, zeros behind it
__device__ __forceinline__ float4 f8_four(const float* p, int n, int N, bool vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (vec) {
    if (n < N) v = *reinterpret_cast<const float4*>(p + n);
  } else {
    if (n < N) v.x = p[n];
    if (n + 1 < N) v.y = p[n + 1];
    if (n + 2 < N) v.z = p[n + 2];
    if (n + 3 < N) v.w = p[n + 3];
  }
  return v;
}

// Asks L2 for a warp's part of the residuals, 32 rows from m0 and COLS columns from n0 on: it is added when the tile is done
template <int COLS>
__device__ __forceinline__ void f8_ask_residuals(const F8Out& o, int m0, int n0) {
  const int m = m0 + (int)(threadIdx.x & 31);
  if (m >= o.m) return;
#pragma unroll
  for (int c = 0; c < COLS; c += 32) {
    if (n0 + c >= o.n) break;
    const size_t at = (size_t)m * o.n + n0 + c;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(o.r1 + at));
    if (o.r2) asm volatile("prefetch.global.L2 [%0];" ::"l"(o.r2 + at));
  }
}

// Turned rows of 32 f32 columns to y, `rows` of them from m0 on; the lane's column n is on the matrix. Residuals: eight rows at a time, all
// loads, then all stores (y may be a residual, so that the compiler moves no load before a store): 4000 rows of 5001 x 700 to f32 took
// 291 us a row at a time and take 83, without residuals 42. Batches cost the rows without residuals time (16 bits: 52 us instead of 44).
template <bool RES>
__device__ __forceinline__ void f8_rows_out(const F8Out& o, const uint8_t* turn, int rows, int m0, int n) {
  const int lane = threadIdx.x & 31;
  const size_t first = (size_t)m0 * o.n + n;
  if (!RES) {
    const float bias = o.bias ? o.bias[n] : 0.f;
    const int size = o.type == FB200_F32 ? 4 : 2;
    const uintptr_t from = reinterpret_cast<uintptr_t>(turn) + 4 * lane;
    uint8_t* to = reinterpret_cast<uint8_t*>(o.y) + first * size;
#pragma unroll 8
    for (int r = 0; r < rows; ++r, to += (size_t)o.n * size) {
      const float v = *reinterpret_cast<const float*>((from ^ ((r & 7) << 4)) + r * 128) + bias;
      if (size == 4) *reinterpret_cast<float*>(to) = v;
      else *reinterpret_cast<uint16_t*>(to) = (uint16_t)f8_pair(o, make_float2(v, 0.f));
    }
    return;
  }
  const float *p1 = o.r1 + first, *p2 = o.r2 + first;
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += 8) {
    const bool all = r0 + 8 <= rows;
    float v[8], e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const float*>(turn + (r0 + i) * 128 + (((lane >> 2) ^ i) << 4) + 4 * (lane & 3));
#pragma unroll
    for (int i = 0; i < 8; ++i, p1 += o.n) e[i] = all || r0 + i < rows ? *p1 : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += e[i];
    if (o.r2) {
#pragma unroll
      for (int i = 0; i < 8; ++i, p2 += o.n) e[i] = all || r0 + i < rows ? *p2 : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] += e[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (all || r0 + i < rows) f8_put(o, v[i], first + (size_t)(r0 + i) * o.n);
  }
}

// A warp's 32 rows from m0 on, COLS columns from n0 on, a row per thread, to y: turned in shared memory, so that a row's columns leave
// together.
template <int COLS, bool RES>
__device__ __forceinline__ void f8_store_rows(const F8Out& o, const float2 (&acc)[COLS / 2], uint8_t* turn, int m0, int n0) {
  const int lane = threadIdx.x & 31, rows = min(32, o.m - m0), n_end = o.n - n0;
  uint4* mine = reinterpret_cast<uint4*>(turn + lane * 128);
  if (!RES && o.pack) {
    uint16_t* to = reinterpret_cast<uint16_t*>(o.y) + (size_t)m0 * o.n + n0 + 8 * (lane & 7);
#pragma unroll
    for (int c = 0; c < (COLS + 63) / 64; ++c) {
      if (64 * c >= n_end) break;
      const int pieces = COLS - 64 * c < 64 ? (COLS - 64 * c) / 8 : 8;
      __syncwarp();
#pragma unroll
      for (int p = 0; p < pieces; ++p) {
        const float2* v = acc + 32 * c + 4 * p;
        mine[p ^ (lane & 7)] = make_uint4(f8_pair(o, v[0]), f8_pair(o, v[1]), f8_pair(o, v[2]), f8_pair(o, v[3]));
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 4 * i + (lane >> 3);
        const uint4 v = *reinterpret_cast<const uint4*>(turn + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
        if (r < rows && 64 * c + 8 * (lane & 7) < n_end && (pieces == 8 || (lane & 7) < pieces)) *reinterpret_cast<uint4*>(to + (size_t)r * o.n + 64 * c) = v;
      }
    }
    return;
  }
  // o.vec: a lane has four columns of every fourth row. The residuals of four rows are in flight together, all loads ahead of the stores (y
  // may be a residual, so that the compiler moves none): 8192 rows of 4096 x 4096 to f32 with one take 171 us, 4000 rows of 5000 x 700 take
  // 57, one row at a time 125. Eight rows at a time spilled registers: 197 and 75 us.
  const int n4 = n0 + 4 * (lane & 7);
  const size_t at4 = (size_t)(m0 + (lane >> 3)) * o.n + n4;
#pragma unroll
  for (int c = 0; c < COLS / 32; ++c) {
    if (32 * c >= n_end) break;
    __syncwarp();
#pragma unroll
    for (int p = 0; p < 8; ++p) {
      const float2* v = acc + 16 * c + 2 * p;
      mine[p ^ (lane & 7)] = make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
    }
    __syncwarp();
    if (o.vec) {  // whole fours: N is a multiple of four then
      if (n4 + 32 * c < o.n) {
        const float4 bias = o.bias ? f8_four(o.bias, n4 + 32 * c, o.n, false) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int h = 0; h < 8; h += 4) {
          const float *p1 = o.r1 + at4 + (size_t)(4 * h) * o.n + 32 * c, *p2 = o.r2 + at4 + (size_t)(4 * h) * o.n + 32 * c;
          const int left = rows - 4 * h - (lane >> 3);
          float4 v[4], e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (RES && 4 * i < left) e[i] = *reinterpret_cast<const float4*>(p1 + (size_t)(4 * i) * o.n);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = 4 * (h + i) + (lane >> 3);
            v[i] = f8_add(*reinterpret_cast<const float4*>(turn + r * 128 + (((lane & 7) ^ (r & 7)) << 4)), bias);
            if (RES && 4 * i < left) v[i] = f8_add(v[i], e[i]);
          }
          if (RES && o.r2) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (4 * i < left) e[i] = *reinterpret_cast<const float4*>(p2 + (size_t)(4 * i) * o.n);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (4 * i < left) v[i] = f8_add(v[i], e[i]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (4 * i < left) f8_put4(o, v[i], at4 + (size_t)(4 * (h + i)) * o.n + 32 * c);
        }
      }
    } else if (32 * c + lane < n_end) {
      f8_rows_out<RES>(o, turn, rows, m0, n0 + 32 * c + lane);
    }
  }
}

// ---- few activation rows ------------------------------------------------------------------------------------------------

template <int BM>
struct Few {
  static constexpr int EPI_WARPS = 4, THREADS = (EPI_WARPS + 2) * 32;
  static constexpr int STAGE = F8_A_BYTES + BM * 128, STAGES = BM == 16 ? 5 : 4, BUFS = 4, TMEM = BUFS * BM;
  static constexpr int AHEAD = 16;  // blocks of K whose scales are fetched together
  static constexpr int SCALE_ROW = BM + 4, SCALE_BYTES = 2 * AHEAD * SCALE_ROW * 4;
  static constexpr int PART = BM * 128 * 4;  // the partial sums that come in from the cluster
  static constexpr int SMEM = STAGES * STAGE + PART + SCALE_BYTES + 256 + 1024;  // two CTAs to an SM
  // instruction descriptor: f32 accumulator, e4m3 A and B, both K-major, N = BM, M = 128
  static constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(BM >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
};

struct SplitArgs {
  const float *sx, *sw;
  F8Out out;
  int kblocks, m_tiles, split;
  int* status;
};

// Stores into the shared memory of a CTA of the cluster, counted in bytes on a barrier there
__device__ __forceinline__ void st_cluster4(uint32_t addr, float2 a, float2 b, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(addr), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "r"(bar) : "memory");
}
__device__ __forceinline__ void st_cluster2(uint32_t addr, float2 a, uint32_t bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];"
               ::"r"(addr), "f"(a.x), "f"(a.y), "r"(bar) : "memory");
}

template <int BM>
__global__ void __launch_bounds__(Few<BM>::THREADS, 2)
f8_few_kernel(const SplitArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
  using F = Few<BM>;
  extern __shared__ uint8_t sm_raw[];
  // the same offset in every CTA of the cluster: their dynamic shared memory starts at the same address
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~(uintptr_t)1023);
  float* part = reinterpret_cast<float*>(sm + F::STAGES * F::STAGE);
  float* scales = reinterpret_cast<float*>(sm + F::STAGES * F::STAGE + F::PART);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + F::STAGES * F::STAGE + F::PART + F::SCALE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * F::STAGES + 2 * F::BUFS + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t full = smem_u32(bars), stage_free = full + 8 * F::STAGES, acc_full = stage_free + 8 * F::STAGES, acc_free = acc_full + 8 * F::BUFS,
                 drained = acc_free + 8 * F::BUFS, joined = drained + 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), tile = (int)blockIdx.x / a.split;
  // activation tiles fastest: the CTAs that run together share their weight rows in L2
  const int nt = tile / a.m_tiles, mt = tile - nt * a.m_tiles, m0 = mt * BM;
  const int kb0 = (int)((long long)a.kblocks * rank / a.split), nkb = (int)((long long)a.kblocks * (rank + 1) / a.split) - kb0;
  const int pre = min(F::STAGES, nkb);

  // The copy requester sets the barriers up and asks for the first weights, which depend on no kernel in front, while tensor memory is
  // allocated (1650 cycles to that point, and the weights' latency after it, when it was done before)
  if (tid == F::EPI_WARPS * 32) {
    *dead = 0;
    for (int i = 0; i < F::STAGES; ++i) { mbar_init(full + 8 * i, 1); mbar_init(stage_free + 8 * i, 1); }
    for (int i = 0; i < F::BUFS; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_free + 8 * i, F::EPI_WARPS); }
    mbar_init(drained, 1);
    mbar_init(joined, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    mbar_expect_tx(joined, a.split > 1 ? F::PART : 0);
    for (int i = 0; i < pre; ++i) {
      mbar_expect_tx(full + 8 * i, F::STAGE);
      x_tma_box2(smem_u32(sm + i * F::STAGE), &wmap, (kb0 + i) * F8_BLOCK, nt * 128, full + 8 * i);
    }
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(F::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents_small();  // behind the allocation: a dependent must not take columns that this grid still waits for
  // The cluster meets twice: everybody has started, so that partial sums may be sent, and (behind the sending) everybody has sent, so that
  // nobody leaves while something may still come. Relaxed arrivals: the barriers' set-up is fenced above, and what is sent is counted by its
  // receiver (a release took 1000 cycles each time).
  if (a.split > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  if (warp < F::EPI_WARPS) {
    // ---- epilogue: warp w reads TMEM lanes 32 w .. = weight rows
    constexpr int ET = F::EPI_WARPS * 32, MINE = F::AHEAD * BM / ET;
    float2 acc[BM / 2];
#pragma unroll
    for (int i = 0; i < BM / 2; ++i) acc[i] = make_float2(0.f, 0.f);
    float ahead[MINE];
    // scales of AHEAD blocks: thread t holds block t % AHEAD of activation rows t / AHEAD, ..
    auto fetch = [&](int first) {
      const int kb = kb0 + first + (tid % F::AHEAD);
      const bool in = first + (tid % F::AHEAD) < nkb;
      const float w = in ? a.sw[(size_t)nt * a.kblocks + kb] : 0.f;
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        const int m = m0 + tid / F::AHEAD + i * (ET / F::AHEAD);
        ahead[i] = in && m < a.out.m ? a.sx[(size_t)m * a.kblocks + kb] * w : 0.f;
      }
    };
    pdl_wait();
    fetch(0);
    // this thread's outputs and what is added to them, asked for ahead of the blocks: `per` rows from m1 on
    const int n = nt * 128 + tid, per = BM / a.split, m1 = m0 + rank * per;
    const bool on = n < a.out.n;
    const float bias = a.out.bias && on ? a.out.bias[n] : 0.f;
    float e1[BM], e2[BM];
#pragma unroll
    for (int j = 0; j < BM; ++j) {
      const bool in = on && j < per && m1 + j < a.out.m;
      e1[j] = in && a.out.r1 ? a.out.r1[(size_t)(m1 + j) * a.out.n + n] : 0.f;
      e2[j] = in && a.out.r2 ? a.out.r2[(size_t)(m1 + j) * a.out.n + n] : 0.f;
    }
    int buf = 0;
    uint32_t parity = 0;
    for (int i = 0; i < nkb; ++i) {
      const int at = i % F::AHEAD;
      const float* half = scales + ((i / F::AHEAD) & 1) * F::AHEAD * F::SCALE_ROW;
      if (at == 0) {
        // the other half was last read before everybody came to this barrier's predecessor
#pragma unroll
        for (int j = 0; j < MINE; ++j) const_cast<float*>(half)[(tid % F::AHEAD) * F::SCALE_ROW + tid / F::AHEAD + j * (ET / F::AHEAD)] = ahead[j];
        asm volatile("bar.sync 1, %0;" ::"n"(ET) : "memory");
        if (i + F::AHEAD < nkb) fetch(i + F::AHEAD);
      }
      if (!f_wait(acc_full + 8 * buf, parity, dead, a.status)) {
        // the barriers of the scales to come are met all the same
        for (int j = (i / F::AHEAD + 1) * F::AHEAD; j < nkb; j += F::AHEAD) asm volatile("bar.sync 1, %0;" ::"n"(ET) : "memory");
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t tl = tmem + ((uint32_t)(32 * warp) << 16) + (uint32_t)(buf * BM);
      const float4* sc = reinterpret_cast<const float4*>(half + at * F::SCALE_ROW);
      uint32_t v[BM / 16][16];
#pragma unroll
      for (int j = 0; j < BM / 16; ++j) x_ld16(tl + 16 * j, v[j]);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      w_arrive(acc_free + 8 * buf);
#pragma unroll
      for (int j = 0; j < BM / 4; ++j) {
        const float4 f = sc[j];
        const uint32_t* p = &v[j / 4][4 * (j % 4)];
        acc[2 * j] = fma2(make_float2(__uint_as_float(p[0]), __uint_as_float(p[1])), make_float2(f.x, f.y), acc[2 * j]);
        acc[2 * j + 1] = fma2(make_float2(__uint_as_float(p[2]), __uint_as_float(p[3])), make_float2(f.z, f.w), acc[2 * j + 1]);
      }
      if (++buf == F::BUFS) { buf = 0; parity ^= 1u; }
    }
    if (a.split == 1) {
#pragma unroll
      for (int j = 0; j < BM; ++j)
        if (on && m1 + j < a.out.m) f8_put(a.out, (j & 1 ? acc[j / 2].y : acc[j / 2].x) + bias + e1[j] + e2[j], (size_t)(m1 + j) * a.out.n + n);
    } else {
      // The sums of the cluster's ranges of K: rank q gets activation rows BM q / split .. of all, [rank][weight row][activation row], and
      // adds them in the order of the ranks. (Fetched by their owner between two meetings of the cluster they took 1.5 us longer.)
      const uint32_t mine = smem_u32(part) + (uint32_t)((rank * 128 + tid) * per) * 4;
      __syncwarp();
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (per >= 4) {
#pragma unroll
        for (int j = 0; j < BM; j += 4) {
          const int to = j / per;
          st_cluster4(cluster_addr(mine + (uint32_t)(j - to * per) * 4, to), acc[j / 2], acc[j / 2 + 1], cluster_addr(joined, to));
        }
      } else {
#pragma unroll
        for (int j = 0; j < BM; j += 2) st_cluster2(cluster_addr(mine, j / 2), acc[j / 2], cluster_addr(joined, j / 2));
      }
      __syncwarp();
      asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
      if (f_wait(joined, 0, dead, a.status) && on) {
#pragma unroll
        for (int j = 0; j < BM / 2; ++j) {
          if (j >= per || m1 + j >= a.out.m) break;
          const float* from = part + tid * per + j;
          float v = 0.f;
          for (int q = 0; q < a.split; ++q) v += from[q * 128 * per];
          f8_put(a.out, v + bias + e1[j] + e2[j], (size_t)(m1 + j) * a.out.n + n);
        }
      }
      __syncwarp();
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (*dead) x_drain(joined, 0);
    }
  } else if (warp == F::EPI_WARPS) {
    // ---- copy requester, from the first activation rows on
    if (lane == 0) {
      pdl_wait();
      int i = 0;
      for (; i < pre; ++i) x_tma_box2(smem_u32(sm + i * F::STAGE + F8_A_BYTES), &xmap, (kb0 + i) * F8_BLOCK, m0, full + 8 * i);
      for (; i < nkb; ++i) {
        const int s = i % F::STAGES;
        if (!x_wait(stage_free + 8 * s, (uint32_t)((i / F::STAGES - 1) & 1), dead, a.status)) break;
        const uint32_t dst = smem_u32(sm + s * F::STAGE), bar = full + 8 * s;
        mbar_expect_tx(bar, F::STAGE);
        x_tma_box2(dst, &wmap, (kb0 + i) * F8_BLOCK, nt * 128, bar);
        x_tma_box2(dst + F8_A_BYTES, &xmap, (kb0 + i) * F8_BLOCK, m0, bar);
      }
      if (*dead)
        for (int j = max(0, i - F::STAGES); j < i; ++j) x_drain(full + 8 * (j % F::STAGES), (uint32_t)((j / F::STAGES) & 1));
    }
  } else {
    // ---- MMA issuer
    pdl_wait();  // the limit of its waits does not count the kernel in front
    const uint64_t adesc0 = x_desc_rows(smem_u32(sm)), bdesc0 = x_desc_rows(smem_u32(sm) + F8_A_BYTES);
    int st = 0, buf = 0;
    uint32_t parity = 0, round = 0;
    for (int i = 0; i < nkb; ++i) {
      if (!f_wait(full + 8 * st, parity, dead, a.status)) break;
      if (round && !f_wait(acc_free + 8 * buf, (round - 1) & 1, dead, a.status)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t at = (uint64_t)((st * F::STAGE) >> 4);
      w_mma4_f8<2, 2>(tmem + (uint32_t)(buf * BM), adesc0 + at, bdesc0 + at, F::IDESC, 0u);
      w_commit(acc_full + 8 * buf);
      w_commit(stage_free + 8 * st);
      if (++st == F::STAGES) { st = 0; parity ^= 1u; }
      if (++buf == F::BUFS) { buf = 0; ++round; }
    }
    w_commit(drained);
    x_drain(drained, 0);
  }
  if (warp >= F::EPI_WARPS && a.split > 1) {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(F::TMEM) : "memory");
}

// ---- some activation rows -----------------------------------------------------------------------------------------------

// XR = 64 or 128 activation rows (in the M role, 128 lanes: lanes behind 64 rows multiply what lies behind them in shared memory and are not
// read) by 128 weight rows per CTA
template <int XR>
struct Some {
  static constexpr int EPI_WARPS = 8, THREADS = (EPI_WARPS + 3) * 32;
  static constexpr int STAGE = XR * 128 + 128 * 128, STAGES = XR == 64 ? 8 : 6, BUFS = 4, TMEM = 512;
  static constexpr int SMEM = STAGES * STAGE + 256 + 1024;
  // instruction descriptor: f32 accumulator, e4m3 A and B, both K-major, N = 128, M = 128
  static constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  static_assert(STAGES % 2 == 0, "a stage belongs to one issuer");
  static_assert(STAGES * STAGE >= XR * 512, "the sums take the operands' place");
};

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Rows XR rank / SPLIT .. of the sums that the CTAs of the cluster have laid down, added in the order of the ranks, a warp to a row at a
// time; all loads of a warp are in flight together, the residuals' ahead of the meeting of the cluster. Tells the cluster when it has read.
template <int XR, int SPLIT, bool RES>
__device__ __forceinline__ void f8_join(const F8Out& o, const uint8_t* sm, int rank, int warp, int m0, int n0) {
  constexpr int PER = XR / SPLIT, ROWS = PER / 8;
  const int lane = threadIdx.x & 31, first = rank * PER + warp, n = n0 + 4 * lane;
  float4 v[ROWS][SPLIT], e1[RES ? ROWS : 1], e2[RES ? ROWS : 1];
  const float4 none = make_float4(0.f, 0.f, 0.f, 0.f), bias = o.bias ? f8_four(o.bias, n, o.n, false) : none;
#pragma unroll
  for (int i = 0; i < (RES ? ROWS : 0); ++i) {
    const size_t row = (size_t)(m0 + first + 8 * i) * o.n;
    const bool in = m0 + first + 8 * i < o.m;
    e1[i] = in ? f8_four(o.r1 + row, n, o.n, o.vec) : none;
    e2[i] = in && o.r2 ? f8_four(o.r2 + row, n, o.n, o.vec) : none;
  }
  __syncwarp();
  cluster_sync();
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = first + 8 * i;
    const uint32_t from = smem_u32(sm + r * 512 + ((lane ^ (r & 7)) << 4));
    if (m0 + r < o.m)
#pragma unroll
      for (int q = 0; q < SPLIT; ++q) v[i][q] = ld_cluster4(cluster_addr(from, (uint32_t)q));
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
#pragma unroll
    for (int q = 1; q < SPLIT; ++q) v[i][0] = f8_add(v[i][0], v[i][q]);
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int m = m0 + first + 8 * i;
    if (m >= o.m) break;
    const size_t at = (size_t)m * o.n + n;
    float4 y = f8_add(v[i][0], bias);
    if (RES) y = f8_add(f8_add(y, e1[RES ? i : 0]), e2[RES ? i : 0]);
    if (o.vec) {
      if (n < o.n) f8_put4(o, y, at);
    } else {
      const float e[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (n + j < o.n) f8_put(o, e[j], at + j);
    }
  }
}

template <int XR, bool RES>
__global__ void __launch_bounds__(Some<XR>::THREADS, 1)
f8_some_kernel(const SplitArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
  using F = Some<XR>;
  extern __shared__ uint8_t sm_raw[];
  // the same offset in every CTA of the cluster: their dynamic shared memory starts at the same address
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + F::STAGES * F::STAGE);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * F::STAGES + 2 * F::BUFS + 1);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const uint32_t full = smem_u32(bars), stage_free = full + 8 * F::STAGES, acc_full = stage_free + 8 * F::STAGES, acc_free = acc_full + 8 * F::BUFS,
                 drained = acc_free + 8 * F::BUFS;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), tile = (int)blockIdx.x / a.split;
  // activation tiles fastest: the CTAs that run together share their weight rows in L2
  const int nt = tile / a.m_tiles, mt = tile - nt * a.m_tiles, m0 = mt * XR, n0 = nt * 128;
  const int kb0 = (int)((long long)a.kblocks * rank / a.split), nkb = (int)((long long)a.kblocks * (rank + 1) / a.split) - kb0;
  const int pre = min(F::STAGES, nkb);

  if (tid == F::EPI_WARPS * 32) {  // as in f8_few_kernel
    *dead = 0;
    for (int i = 0; i < F::STAGES; ++i) { mbar_init(full + 8 * i, 1); mbar_init(stage_free + 8 * i, 1); }
    for (int i = 0; i < F::BUFS; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_free + 8 * i, XR / 32 * 2); }
    mbar_init(drained, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    for (int i = 0; i < pre; ++i) {
      mbar_expect_tx(full + 8 * i, F::STAGE);
      x_tma_box2(smem_u32(sm + i * F::STAGE + XR * 128), &wmap, (kb0 + i) * F8_BLOCK, n0, full + 8 * i);
    }
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(F::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents_small();

  const int quad = warp & 3, side = warp >> 2;
  const bool reads = warp < F::EPI_WARPS && quad < XR / 32;
  float2 acc[32];
  if (reads) {
    // ---- epilogue: warp w reads TMEM lanes 32 (w % 4) .. = activation rows, one half of the weight rows
#pragma unroll
    for (int i = 0; i < 32; ++i) acc[i] = make_float2(0.f, 0.f);
    pdl_wait();
    if (RES && a.split == 1) f8_ask_residuals<64>(a.out, m0 + 32 * quad, n0 + 64 * side);
    const float* sx = a.sx + (size_t)min(m0 + 32 * quad + lane, a.out.m - 1) * a.kblocks + kb0;
    const float* sw = a.sw + (size_t)nt * a.kblocks + kb0;
    float fx = nkb ? sx[0] : 0.f, fw = nkb ? sw[0] : 0.f;
    int buf = 0;
    uint32_t parity = 0;
#pragma unroll 1
    for (int i = 0; i < nkb; ++i) {
      if (!f_wait(acc_full + 8 * buf, parity, dead, a.status)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t tl = tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)(buf * 128 + side * 64);
      uint32_t v[4][16];
#pragma unroll
      for (int j = 0; j < 4; ++j) x_ld16(tl + 16 * j, v[j]);
      const float2 f = make_float2(fx * fw, fx * fw);
      fx = sx[min(i + 1, nkb - 1)];  // in flight until the next block
      fw = sw[min(i + 1, nkb - 1)];
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      w_arrive(acc_free + 8 * buf);
#pragma unroll
      for (int j = 0; j < 32; ++j) acc[j] = fma2(make_float2(__uint_as_float(v[j / 8][2 * j % 16]), __uint_as_float(v[j / 8][2 * j % 16 + 1])), f, acc[j]);
      if (++buf == F::BUFS) { buf = 0; parity ^= 1u; }
    }
  } else if (warp == F::EPI_WARPS) {
    // ---- copy requester, from the first activation rows on
    if (lane == 0) {
      pdl_wait();
      int i = 0;
      for (; i < pre; ++i) x_tma_box2(smem_u32(sm + i * F::STAGE), &xmap, (kb0 + i) * F8_BLOCK, m0, full + 8 * i);
      for (; i < nkb; ++i) {
        const int s = i % F::STAGES;
        if (!x_wait(stage_free + 8 * s, (uint32_t)((i / F::STAGES - 1) & 1), dead, a.status)) break;
        const uint32_t dst = smem_u32(sm + s * F::STAGE), bar = full + 8 * s;
        mbar_expect_tx(bar, F::STAGE);
        x_tma_box2(dst + XR * 128, &wmap, (kb0 + i) * F8_BLOCK, n0, bar);
        x_tma_box2(dst, &xmap, (kb0 + i) * F8_BLOCK, m0, bar);
      }
      if (*dead)
        for (int j = max(0, i - F::STAGES); j < i; ++j) x_drain(full + 8 * (j % F::STAGES), (uint32_t)((j / F::STAGES) & 1));
    }
  } else if (warp > F::EPI_WARPS) {
    // ---- two MMA issuers, every other block each
    pdl_wait();
    const uint64_t adesc0 = x_desc_rows(smem_u32(sm)), bdesc0 = x_desc_rows(smem_u32(sm) + XR * 128);
    const int which = warp - F::EPI_WARPS - 1;
    int st = which;
    uint32_t parity = 0;
    for (int i = which; i < nkb; i += 2) {
      const int buf = i % F::BUFS;
      if (!f_wait(full + 8 * st, parity, dead, a.status)) break;
      if (i >= F::BUFS && !f_wait(acc_free + 8 * buf, (uint32_t)(i / F::BUFS - 1) & 1u, dead, a.status)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint64_t at = (uint64_t)((st * F::STAGE) >> 4);
      w_mma4_f8<2, 2>(tmem + (uint32_t)(buf * 128), adesc0 + at, bdesc0 + at, F::IDESC, 0u);
      w_commit(acc_full + 8 * buf);
      w_commit(stage_free + 8 * st);
      if ((st += 2) >= F::STAGES) { st -= F::STAGES; parity ^= 1u; }
    }
    w_commit(drained);
    x_drain(drained, 0);
  }
  __syncthreads();  // nobody here multiplies from the operands any more: they make room for the sums
  pdl_wait();       // for the warps that have not been in a role that waits

  if (a.split == 1) {
    if (reads) f8_store_rows<64, RES>(a.out, acc, sm + warp * TURN_BYTES, m0 + 32 * quad, n0 + 64 * side);
  } else {
    // The sums of the cluster's ranges of K: everybody lays down its own, 512 bytes a row, 16-byte piece p of row r at place p ^ (r % 8);
    // rank q fetches rows XR q / split .. of all and adds them in the order of the ranks, a warp to a row.
    if (reads) {
      const int r = 32 * quad + lane;
#pragma unroll
      for (int p = 0; p < 16; ++p)
        *reinterpret_cast<float4*>(sm + r * 512 + (((16 * side + p) ^ (r & 7)) << 4)) = make_float4(acc[2 * p].x, acc[2 * p].y, acc[2 * p + 1].x, acc[2 * p + 1].y);
    }
    if (warp < F::EPI_WARPS) {
      if (a.split == 2) f8_join<XR, 2, RES>(a.out, sm, rank, warp, m0, n0);
      else f8_join<XR, 4, RES>(a.out, sm, rank, warp, m0, n0);
    } else {
      __syncwarp();
      cluster_sync();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // the others may still read
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(F::TMEM) : "memory");
}

// ---- many activation rows -----------------------------------------------------------------------------------------------

// Two warpgroups of epilogue warps and one of the copy requester and the issuer, which hands its registers over: 384 x 168 at launch are
// 256 x 224 + 128 x 56. A thread holds 128 sums and 64 values on their way.
constexpr int PAIR_EPI_WARPS = 8, PAIR_THREADS = (PAIR_EPI_WARPS + 4) * 32, PAIR_MAX_STAGES = 8;
template <int NW>
struct Pair {
  static constexpr int STAGE = F8_A_BYTES + NW / 2 * 128, STAGES = NW == 128 ? 8 : 6, TMEM = 512;
  // four accumulators of WIDE columns, 128 columns apart: PARTS of a block of K, BUFS blocks
  static constexpr int PARTS = NW > 128 ? 2 : 1, BUFS = 4 / PARTS, WIDE = NW / PARTS;
  static constexpr int SMEM = STAGES * STAGE + PAIR_EPI_WARPS * TURN_BYTES + 256 + 1024;
  static_assert(PARTS == 2 || STAGES % 2 == 0, "a stage belongs to one issuer");
  // instruction descriptor: f32 accumulator, e4m3 A and B, both K-major, N = WIDE, M = 256 over the pair
  static constexpr uint32_t IDESC = (1u << 4) | ((uint32_t)(WIDE >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
};

struct PairArgs {
  const float *sx, *sw;
  F8Out out;
  int kblocks, m_tiles, n_tiles, m_group;
  int* status;
};

template <int NW, bool RES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
f8_pair_kernel(const PairArgs a, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
  using P = Pair<NW>;
  extern __shared__ uint8_t sm_raw[];
  // the same offset in both CTAs: their dynamic shared memory starts at the same address
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(sm_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* turn = sm + P::STAGES * P::STAGE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sm + P::STAGES * P::STAGE + PAIR_EPI_WARPS * TURN_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * PAIR_MAX_STAGES + 9);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), pair = (int)blockIdx.x >> 1, npairs = (int)gridDim.x >> 1;
  const uint32_t full = smem_u32(bars), stage_free = full + 8 * PAIR_MAX_STAGES, acc_full = stage_free + 8 * PAIR_MAX_STAGES,
                 acc_free = acc_full + 32, drained = acc_free + 32;
  const int items = a.m_tiles * a.n_tiles;

  // The copy requester sets the barriers up and asks for the first weights, which depend on no kernel in front, as soon as both CTAs' are
  // there; tensor memory is allocated meanwhile
  if (tid == PAIR_EPI_WARPS * 32) {
    *dead = 0;
    for (int i = 0; i < P::STAGES; ++i) { mbar_init(full + 8 * i, 1); mbar_init(stage_free + 8 * i, P::PARTS); }
    for (int i = 0; i < 4; ++i) { mbar_init(acc_full + 8 * i, 1); mbar_init(acc_free + 8 * i, 2 * PAIR_EPI_WARPS / P::PARTS); }
    mbar_init(drained, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // the barriers' set-up is fenced
  if (warp == 0) pair_tmem_alloc(smem_u32(tmem_slot), P::TMEM);
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");

  // Tiles in groups of m_group activation tiles, activation tiles fastest within a group: the pairs that run together share their
  // weight rows in L2, and a group's activation rows stay there while the weights go by.
  auto split = [&](int item, int& mt, int& nt) {
    const int g = item / (a.m_group * a.n_tiles), first = g * a.m_group, height = min(a.m_group, a.m_tiles - first);
    const int at = item - first * a.n_tiles;
    nt = at / height;
    mt = first + at - nt * height;
  };
  const int pre = min(P::STAGES, a.kblocks);
  // a CTA holds one half of the weight rows of every part
  auto weights = [&](int s, int kb, int nt) {
#pragma unroll
    for (int p = 0; p < P::PARTS; ++p)
      pair_tma_box2(smem_u32(sm + s * P::STAGE) + F8_A_BYTES + p * (P::WIDE / 2 * 128), &wmap, kb * F8_BLOCK, nt * NW + P::WIDE * p + rank * (P::WIDE / 2),
                    cluster_addr(full + 8 * s, 0));
  };
  if (tid == PAIR_EPI_WARPS * 32) {
    int mt, nt;
    split(pair, mt, nt);
    for (int s = 0; s < pre; ++s) {
      if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * P::STAGE);
      weights(s, s, nt);
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents_small();  // behind the allocation: a dependent must not take columns that this grid still waits for

  if (warp < PAIR_EPI_WARPS) {
    // ---- epilogue: warp w reads TMEM lanes 32 (w % 4) .. of this CTA's 128 activation rows, one half of the weight rows
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    constexpr int HALF = NW / 2;
    const int quad = warp & 3, side = warp >> 2;
    // with two parts the sides have accumulators of their own
    const uint32_t part = P::PARTS == 2 ? side : 0, freed = cluster_addr(acc_free, 0);
    uint32_t k = 0;  // blocks of K so far, over all tiles
    int m_first = 0, n_first = 0;
    const float *sx = nullptr, *sw = nullptr;
    float fx = 0.f, fw = 0.f;  // scales of the next block
    // 96 columns may be of two scales, columns 32 `turns` .. of the second
    constexpr bool TWO = HALF % 64 != 0;
    const float* sw2 = nullptr;
    float fw2 = 0.f;
    int turns = 0;
    auto begin = [&](int item) {
      int mt, nt;
      split(item, mt, nt);
      m_first = mt * 256 + rank * 128 + quad * 32;
      n_first = nt * NW + side * HALF;
      sx = a.sx + (size_t)min(m_first + lane, a.out.m - 1) * a.kblocks;
      sw = a.sw + (size_t)min(n_first / F8_BLOCK, (a.out.n - 1) / F8_BLOCK) * a.kblocks;
      fx = sx[0];
      fw = sw[0];
      if (TWO) {
        turns = (F8_BLOCK - n_first % F8_BLOCK) / 32;
        sw2 = a.sw + (size_t)min((n_first + HALF - 1) / F8_BLOCK, (a.out.n - 1) / F8_BLOCK) * a.kblocks;
        fw2 = sw2[0];
      }
    };
    pdl_wait();
    begin(pair);
    for (int item = pair; item < items; item += npairs) {
      bool alive = true;
      if (RES) f8_ask_residuals<HALF>(a.out, m_first, n_first);
      float2 acc[HALF / 2];
#pragma unroll
      for (int i = 0; i < HALF / 2; ++i) acc[i] = make_float2(0.f, 0.f);
#pragma unroll 1
      for (int kb = 0; kb < a.kblocks; ++kb, ++k) {
        const uint32_t buf = k % P::BUFS * P::PARTS + part;
        if (!(alive = f_wait(acc_full + 8 * buf, k / P::BUFS & 1, dead, a.status))) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t tl = tmem + ((uint32_t)(32 * quad) << 16) + buf * 128 + (P::PARTS == 2 ? 0 : side * HALF);
        const float2 f = make_float2(fx * fw, fx * fw), f2 = make_float2(fx * fw2, fx * fw2);
        fx = sx[min(kb + 1, a.kblocks - 1)];  // in flight until the next block
        fw = sw[min(kb + 1, a.kblocks - 1)];
        if (TWO) fw2 = sw2[min(kb + 1, a.kblocks - 1)];
        uint32_t v[4][16];
        x_ld16(tl, v[0]);
        x_ld16(tl + 16, v[1]);
#pragma unroll
        for (int c = 0; c < HALF / 32; ++c) {
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
          if (c + 1 < HALF / 32) {
            x_ld16(tl + 32 * (c + 1), v[2 * (c + 1) & 3]);
            x_ld16(tl + 32 * (c + 1) + 16, v[(2 * (c + 1) & 3) + 1]);
          } else {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            w_cluster_arrive(freed + 8 * buf);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const uint32_t* p = &v[(2 * c & 3) + i / 8][2 * i % 16];
            acc[16 * c + i] = fma2(make_float2(__uint_as_float(p[0]), __uint_as_float(p[1])), TWO && c >= turns ? f2 : f, acc[16 * c + i]);
          }
        }
      }
      if (!alive) break;
      const int m_done = m_first, n_done = n_first;
      if (item + npairs < items) begin(item + npairs);  // its first scales arrive meanwhile
      f8_store_rows<HALF, RES>(a.out, acc, turn + warp * TURN_BYTES, m_done, n_done);
    }
  } else if (warp == PAIR_EPI_WARPS) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // ---- copy requester: a stage is one block of K, 128 activation rows and NW / 2 weight rows per CTA; the copies of both CTAs are
    // counted on the even CTA's barrier
    if (lane == 0) {
      pdl_wait();
      int k = 0;
      bool alive = true;
      for (int item = pair; item < items && alive; item += npairs) {
        int mt, nt;
        split(item, mt, nt);
        for (int kb = 0; kb < a.kblocks; ++kb, ++k) {
          const int s = k % P::STAGES, round = k / P::STAGES;
          if (round > 0 && !(alive = x_wait(stage_free + 8 * s, (uint32_t)((round - 1) & 1), dead, a.status))) break;
          if (k >= pre) {
            if (rank == 0) mbar_expect_tx(full + 8 * s, 2 * P::STAGE);
            weights(s, kb, nt);
          }
          pair_tma_box2(smem_u32(sm + s * P::STAGE), &xmap, kb * F8_BLOCK, mt * 256 + rank * 128, cluster_addr(full + 8 * s, 0));
        }
      }
      if (*dead) {
        // the even CTA waits for the copies that its barriers count; the odd one has no barrier of its own that counts
        // them and lets the limit of a wait run out instead, which takes far longer than a copy
        if (rank) x_drain(full, 0);
        else
          for (int i = max(0, k - P::STAGES); i < k; ++i) x_drain(full + 8 * (i % P::STAGES), (uint32_t)((i / P::STAGES) & 1));
      }
    }
  } else if (warp <= PAIR_EPI_WARPS + 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    // ---- two MMA issuers (even CTA), an accumulator of WIDE weight rows and a block of K at a time: of the two parts of a block one each,
    // or every other block. (One warp needs 460 cycles for an accumulator's waits, MMAs and commits, nearly twice what the MMAs take. One
    // accumulator of all NW columns, every other block each: the same time with 256, 2 % more with 192.)
    const uint32_t which = warp - PAIR_EPI_WARPS - 1, part = P::PARTS == 2 ? which : 0, step = 2 / P::PARTS;
    const uint32_t blocks = (uint32_t)((items - pair + npairs - 1) / npairs) * (uint32_t)a.kblocks;
    if (rank == 0) {
      pdl_wait();
      const uint64_t adesc0 = x_desc_rows(smem_u32(sm)), bdesc0 = x_desc_rows(smem_u32(sm) + F8_A_BYTES) + part * (P::WIDE / 2 * 128 >> 4);
      uint32_t s = P::PARTS == 2 ? 0 : which, parity = 0;
      for (uint32_t k = s; k < blocks; k += step) {
        const uint32_t buf = k % P::BUFS * P::PARTS + part;
        if (!f_wait(full + 8 * s, parity, dead, a.status)) break;
        if (k >= P::BUFS && !f_wait(acc_free + 8 * buf, (k / P::BUFS - 1) & 1, dead, a.status)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint64_t at = (uint64_t)((s * P::STAGE) >> 4);
        pair_mma4_f8<2>(tmem + buf * 128, adesc0 + at, bdesc0 + at, P::IDESC, 0u);
        pair_commit(acc_full + 8 * buf);
        pair_commit(stage_free + 8 * s);
        if ((s += step) >= P::STAGES) { s -= P::STAGES; parity ^= 1u; }
      }
      pair_commit(drained);
      x_drain(drained, 0);  // the odd CTA learns of it at the last meeting
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 0) pair_tmem_free(tmem, P::TMEM);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

struct F8Job {
  const uint8_t* x;
  size_t ld;
  const float* sx;
  const fb200_f8matrix* w;
  F8Out out;
  int kblocks;
};

template <typename K>
int allow_smem(fb200_device* dev, K kern, int bytes, bool (&configured)[64]) {
  if (configured[dev->ordinal & 63]) return FB200_OK;
  FB_CUDA(dev, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  configured[dev->ordinal & 63] = true;
  return FB200_OK;
}

// The kernels of single CTAs: clusters of `split` CTAs per tile of `rows` activation rows and 128 weight rows
template <typename K>
int launch_split(fb200_device* dev, const F8Job& j, K kern, int rows, int threads, int smem, int split, bool (&configured)[64]) {
  int rc = allow_smem(dev, kern, smem, configured);
  if (rc) return rc;
  CUtensorMap xmap;
  if (!fb200_make_map_2d_bytes(&xmap, j.x, j.w->k, (uint64_t)j.out.m, j.ld, (uint32_t)rows))
    return fb200_fail(dev, FB200_ERR_CUDA, "f8_mat_mul: tensor map refused (x %d rows every %zu bytes)", j.out.m, j.ld);
  const SplitArgs a = {j.sx, j.w->scales, j.out, j.kblocks, (j.out.m + rows - 1) / rows, split, dev->status};
  const long long ctas = (long long)a.m_tiles * ((j.out.n + 127) / 128) * split;
  if (ctas > 0x7FFFFFFF) return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "f8_mat_mul: %d x %d outputs are too many", j.out.m, j.out.n);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = dev->stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dev->pdl ? 2 : 1;
  FB_CUDA(dev, cudaLaunchKernelEx(&cfg, kern, a, j.w->map128, xmap));
  dev->launches++;
  return FB200_OK;
}
template <int BM>
int launch_few(fb200_device* dev, const F8Job& j, int split) {
  static bool configured[64] = {false};
  return launch_split(dev, j, f8_few_kernel<BM>, BM, Few<BM>::THREADS, Few<BM>::SMEM, split, configured);
}
template <int XR, bool RES>
int launch_some_as(fb200_device* dev, const F8Job& j, int split) {
  static bool configured[64] = {false};
  return launch_split(dev, j, f8_some_kernel<XR, RES>, XR, Some<XR>::THREADS, Some<XR>::SMEM, split, configured);
}
// Kernels without residuals have no room set aside for them: with it 8192 rows of 28672 x 4096 took 870 us instead of 830
template <int XR>
int launch_some(fb200_device* dev, const F8Job& j, int split) {
  return j.out.r1 ? launch_some_as<XR, true>(dev, j, split) : launch_some_as<XR, false>(dev, j, split);
}

template <int NW, bool RES>
int launch_pair_as(fb200_device* dev, const F8Job& j) {
  using P = Pair<NW>;
  static bool configured[64] = {false};
  int rc = allow_smem(dev, f8_pair_kernel<NW, RES>, P::SMEM, configured);
  if (rc) return rc;
  CUtensorMap xmap;
  if (!fb200_make_map_2d_bytes(&xmap, j.x, j.w->k, (uint64_t)j.out.m, j.ld, 128))
    return fb200_fail(dev, FB200_ERR_CUDA, "f8_mat_mul: tensor map refused (x %d rows every %zu bytes)", j.out.m, j.ld);
  PairArgs a = {j.sx, j.w->scales, j.out, j.kblocks, (j.out.m + 255) / 256, (j.out.n + NW - 1) / NW, 1, dev->status};
  const long long items = (long long)a.m_tiles * a.n_tiles;
  if (items > 0x3FFFFFFF) return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "f8_mat_mul: %d x %d outputs are too many", j.out.m, j.out.n);
  // the activation rows of a group take at most 32 MB of L2
  const long long fit = (32ll << 20) / (256ll * F8_BLOCK * j.kblocks);
  a.m_group = fit < 1 ? 1 : fit > a.m_tiles ? a.m_tiles : (int)fit;
  const int pairs = items < dev->sm_count / 2 ? (int)items : dev->sm_count / 2;
  return fb200_launch(dev, f8_pair_kernel<NW, RES>, dim3((unsigned)(2 * pairs)), dim3(PAIR_THREADS), (size_t)P::SMEM, true, a,
                      NW == 192 ? j.w->map48 : j.w->map64, xmap);
}
template <int NW>
int launch_pair(fb200_device* dev, const F8Job& j) {
  return j.out.r1 ? launch_pair_as<NW, true>(dev, j) : launch_pair_as<NW, false>(dev, j);
}

// The kernel, by the number of rows and a small cost model in microseconds (fitted to the times below, which hold for products one after
// the other over weights that come from HBM):
//  * up to 16 and up to 32 rows: the kernel for few rows, K split as far as the CTAs run at once and have four blocks each. One row,
//    4096 x 14336: 32 us unsplit, 20, 13.7 and 12.0 split by 2, 4 and 8; 28672 x 4096: 20.1 unsplit, 25.6 by 2 (two rounds). 12 rows of
//    4096 x 14336: 12.3, with the kernel for some rows 14.3;
//  * above, single CTAs with 64 or 128 rows: a round takes 0.28 or 0.31 a block and 3 more, a split 2 more. By 8 it was slower (16 clusters of
//    8 do not run at once: 64 rows of 4096 x 4096 8.6 us by 4, 17.8 by 8);
//  * against pairs: a round takes 0.27 (128 weight rows), 0.39 (192) or 0.42 (256) a block and 1.5 more, 3.5 around them. 512 rows of
//    4096 x 4096: 13.6 us on single CTAs, 14.3 on pairs; 1024 of 6144 x 4096: 38.2 on single CTAs, 35.3, 31.5 and 34.0 on pairs of 128, 192
//    and 256 (three, two and two rounds); 4096 of 6144 x 4096, where 256 take a round less: 125.6, 105.7 and 99.8.
int f8_product(fb200_device* dev, const F8Job& j) {
  const int m = j.out.m, n_tiles = (j.out.n + 127) / 128;
  int rows = m <= 16 ? 16 : 32, split = 1, pair = 0;
  if (m <= 32) {
    while (split < 8 && n_tiles * split * 2 <= dev->sm_count * 2 && j.kblocks >= split * 4) split *= 2;
  } else {
    double best = 1e30;
    for (int r = 64; r <= 128; r *= 2)
      for (int c = 1; c <= 4 && (c == 1 || j.kblocks >= c * 2); c *= 2) {
        const long long tiles = (long long)n_tiles * ((m + r - 1) / r);
        const int room = c == 4 ? dev->sm_count * 33 / 148 : dev->sm_count / c;  // clusters that run at once
        const double cost = (double)((tiles + room - 1) / room) * ((j.kblocks + c - 1) / c * (r == 64 ? 0.28 : 0.31) + 3.0) + (c > 1 ? 2.0 : 0.0);
        if (cost < best) best = cost, rows = r, split = c;
      }
    for (int nw = 128; nw <= 256; nw += 64) {
      const long long items = (long long)((j.out.n + nw - 1) / nw) * ((m + 255) / 256);
      const int room = dev->sm_count / 2;
      const double cost = (double)((items + room - 1) / room) * (j.kblocks * (nw == 128 ? 0.27 : nw == 192 ? 0.39 : 0.42) + 1.5) + 3.5;
      if (cost < best) best = cost, pair = nw;
    }
  }
  // FB200_F8_TILE (tests, tuning; read per call): "ROWS,SPLIT" activation rows (16, 32, 64, 128) and ranges of K (8 with 16 or 32 rows
  // only) of the kernels on single CTAs, "pair,NW" pairs with 128, 192 or 256 weight rows; what there is not leaves the choice to the rule
  if (const char* cfg = getenv("FB200_F8_TILE")) {
    int frows, fsplit;
    if (sscanf(cfg, "pair,%d", &frows) == 1) {
      if (frows == 128 || frows == 192 || frows == 256) pair = frows;
    } else if (sscanf(cfg, "%d,%d", &frows, &fsplit) == 2 && (frows == 16 || frows == 32 || frows == 64 || frows == 128) &&
               (fsplit == 1 || fsplit == 2 || fsplit == 4 || (fsplit == 8 && frows <= 32))) {
      rows = frows, split = fsplit, pair = 0;
    }
  }
  if (pair) return pair == 128 ? launch_pair<128>(dev, j) : pair == 192 ? launch_pair<192>(dev, j) : launch_pair<256>(dev, j);
  switch (rows) {
    case 16: return launch_few<16>(dev, j, split);
    case 32: return launch_few<32>(dev, j, split);
    case 64: return launch_some<64>(dev, j, split);
    default: return launch_some<128>(dev, j, split);
  }
}

int check_shape(fb200_device* dev, const char* op, const uint64_t* shape, int rank) {
  if (rank != 2 || !shape) return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "%s: needs a rank-2 shape, got rank %d", op, rank);
  if (!shape[0] || !shape[1] || shape[0] > (1ull << 27) || shape[1] > (1ull << 27))
    return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "%s: shape [%llu, %llu]", op, (unsigned long long)shape[0], (unsigned long long)shape[1]);
  return FB200_OK;
}

int make_maps(fb200_device* dev, fb200_f8matrix* w) {
  if (fb200_make_map_2d_bytes(&w->map128, w->codes, w->k, w->n, w->ld, 128) && fb200_make_map_2d_bytes(&w->map64, w->codes, w->k, w->n, w->ld, 64) &&
      fb200_make_map_2d_bytes(&w->map48, w->codes, w->k, w->n, w->ld, 48))
    return FB200_OK;
  return fb200_fail(dev, FB200_ERR_CUDA, "F8Matrix: tensor map refused (%llu x %llu)", (unsigned long long)w->n, (unsigned long long)w->k);
}

}  // namespace

extern "C" {

int fb200_f8matrix_from_raw_bytes(fb200_device* dev, const uint64_t* shape, int rank, const void* codes_host, size_t nbytes, const float* scales_host,
                                  size_t nscales, fb200_f8matrix** out) {
  int rc = fb200_bind(dev);
  if (rc) return rc;
  if (!out) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "out is null");
  *out = nullptr;
  if ((rc = check_shape(dev, "F8Matrix", shape, rank))) return rc;
  const uint64_t n = shape[0], k = shape[1], blocks = ((n + 127) / 128) * ((k + 127) / 128);
  if (!codes_host || !scales_host) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "F8Matrix: null argument");
  if (nbytes != n * k || nscales != blocks)
    return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "F8Matrix: shape [%llu, %llu] needs %llu codes and %llu scales, got %zu and %zu", (unsigned long long)n,
                      (unsigned long long)k, (unsigned long long)(n * k), (unsigned long long)blocks, nbytes, nscales);
  fb200_f8matrix* w = new (std::nothrow) fb200_f8matrix();
  if (!w) return fb200_fail(dev, FB200_ERR_CAPACITY, "F8Matrix: no host memory");
  w->dev = dev; w->n = n; w->k = k; w->ld = (k + 15) / 16 * 16; w->owned = true;
  cudaError_t e = cudaMalloc(&w->codes, n * w->ld);
  if (e == cudaSuccess) e = cudaMalloc(&w->scales, blocks * sizeof(float));
  if (e == cudaSuccess) e = cudaMemcpy2DAsync(w->codes, w->ld, codes_host, k, k, n, cudaMemcpyHostToDevice, dev->stream);
  if (e == cudaSuccess) e = cudaMemcpyAsync(w->scales, scales_host, blocks * sizeof(float), cudaMemcpyHostToDevice, dev->stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(dev->stream);
  rc = e == cudaSuccess ? make_maps(dev, w) : fb200_fail(dev, FB200_ERR_CUDA, "F8Matrix upload: %s", cudaGetErrorString(e));
  if (e != cudaSuccess) cudaGetLastError();  // reported here, not by the check of a later launch
  if (rc) {
    cudaFree(w->codes);
    cudaFree(w->scales);
    delete w;
    return rc;
  }
  *out = w;
  return FB200_OK;
}

int fb200_f8matrix_from_device(fb200_device* dev, const uint64_t* shape, int rank, const uint8_t* codes_dev, size_t ld, const float* scales_dev,
                               fb200_f8matrix** out) {
  int rc = fb200_bind(dev);
  if (rc) return rc;
  if (!out) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "out is null");
  *out = nullptr;
  if ((rc = check_shape(dev, "F8Matrix", shape, rank))) return rc;
  if (!codes_dev || !scales_dev) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "F8Matrix: null argument");
  if (ld < shape[1] || ld % 16 || (uintptr_t)codes_dev % 16 || (uintptr_t)scales_dev % 4)
    return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "F8Matrix: rows of %llu codes every %zu bytes (a multiple of 16, from a multiple of 16 on)",
                      (unsigned long long)shape[1], ld);
  fb200_f8matrix* w = new (std::nothrow) fb200_f8matrix();
  if (!w) return fb200_fail(dev, FB200_ERR_CAPACITY, "F8Matrix: no host memory");
  w->dev = dev; w->n = shape[0]; w->k = shape[1]; w->ld = ld;
  w->codes = const_cast<uint8_t*>(codes_dev); w->scales = const_cast<float*>(scales_dev);
  // products fetch the codes without waiting for the kernel in front of them: what writes them has to be done
  const cudaError_t e = cudaStreamSynchronize(dev->stream);
  rc = e == cudaSuccess ? make_maps(dev, w) : fb200_fail(dev, FB200_ERR_CUDA, "F8Matrix: %s", cudaGetErrorString(e));
  if (e != cudaSuccess) cudaGetLastError();
  if (rc) {
    delete w;
    return rc;
  }
  *out = w;
  return FB200_OK;
}

int fb200_f8matrix_free(fb200_f8matrix* w) {
  if (!w) return FB200_OK;
  const int rc = fb200_bind(w->dev);
  if (rc) return rc;
  if (w->owned) {
    cudaStreamSynchronize(w->dev->stream);
    cudaFree(w->codes);
    cudaFree(w->scales);
  }
  delete w;
  return FB200_OK;
}

int fb200_f8matrix_shape(const fb200_f8matrix* w, uint64_t* n_out, uint64_t* k_out) {
  if (!w) return FB200_ERR_INVALID_ARGUMENT;
  if (n_out) *n_out = w->n;
  if (k_out) *k_out = w->k;
  return FB200_OK;
}

int fb200_f8_mat_mul(fb200_device* dev, const uint8_t* codes_dev, size_t ld, const float* scales_dev, size_t m, const fb200_f8matrix* w, uint32_t y_type,
                     void* y_dev, const fb200_epilogue* ep) {
  const int rc = fb200_bind(dev);
  if (rc) return rc;
  if (!w || !codes_dev || !scales_dev || !y_dev) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "f8_mat_mul: null argument");
  if (w->dev != dev) return fb200_fail(dev, FB200_ERR_DEVICE_MISMATCH, "f8_mat_mul: weight lives on another device handle");
  if (y_type != FB200_F32 && y_type != FB200_F16 && y_type != FB200_BF16)
    return fb200_fail(dev, FB200_ERR_UNSUPPORTED_DTYPE, "f8_mat_mul: outputs of type %u (F32, F16 or BF16)", y_type);
  const int epi = ep ? ep->kind : FB200_EPI_NONE;
  if (epi < 0 || epi > 3) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "f8_mat_mul: epilogue kind %d", epi);
  if (epi == FB200_EPI_SWIGLU)
    return fb200_fail(dev, FB200_ERR_UNSUPPORTED_DTYPE, "f8_mat_mul: no SwiGLU epilogue (fb200_silu_mul_f8 takes the product's rows)");
  if (epi != FB200_EPI_NONE && !ep->r1_dev) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "f8_mat_mul: residual / bias epilogue without r1");
  if (epi == FB200_EPI_BIAS && ep->r2_dev) return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "f8_mat_mul: the bias epilogue takes r1 only");
  if (m > (1ull << 27)) return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "f8_mat_mul: %zu rows are too many", m);
  if (ld < w->k || ld % 16 || (uintptr_t)codes_dev % 16 || (uintptr_t)scales_dev % 4 || (uintptr_t)y_dev % (y_type == FB200_F32 ? 4 : 2))
    return fb200_fail(dev, FB200_ERR_INVALID_SHAPE, "f8_mat_mul: rows of %llu codes every %zu bytes (a multiple of 16, from a multiple of 16 on)",
                      (unsigned long long)w->k, ld);
  if (epi != FB200_EPI_NONE && ((uintptr_t)ep->r1_dev % 4 || (uintptr_t)ep->r2_dev % 4))
    return fb200_fail(dev, FB200_ERR_INVALID_ARGUMENT, "f8_mat_mul: r1 or r2 is not aligned");
  if (m == 0) return FB200_OK;
  F8Job j = {codes_dev, ld, scales_dev, w, {y_dev, y_type, nullptr, nullptr, nullptr, (int)m, (int)w->n, 0, 0}, (int)((w->k + 127) / 128)};
  if (epi == FB200_EPI_BIAS) j.out.bias = ep->r1_dev;
  if (epi == FB200_EPI_RESIDUAL) { j.out.r1 = ep->r1_dev; j.out.r2 = ep->r2_dev; }
  const uintptr_t four = y_type == FB200_F32 ? 16 : 8;
  j.out.vec = w->n % 4 == 0 && (uintptr_t)y_dev % four == 0 && (uintptr_t)j.out.r1 % 16 == 0 && (uintptr_t)j.out.r2 % 16 == 0;
  j.out.pack = y_type != FB200_F32 && epi == FB200_EPI_NONE && w->n % 8 == 0 && (uintptr_t)y_dev % 16 == 0;
  fb200_op_trace scope(dev, m <= 32 ? "f8_mat_mul (1..32 rows)" : "f8_mat_mul (> 32 rows)",
                       (double)w->n * (double)w->k + (double)m * ((double)w->k + (y_type == FB200_F32 ? 4.0 : 2.0) * (double)w->n));
  return f8_product(dev, j);
}

}  // extern "C"
