// A projection shared by many requests, beside each request's own low-rank
// adapter:
//
//   y[m] = W x[m] + s_i B_i (A_i x[m]) (+ bias),   i = ids[m], none for ids[m] < 0
//
// x (M, K), W (N, K), A (n, rank, K), B (n, N, rank), y (M, N); fp32 sums, one
// rounding at the end. 2 M N K + 2 M rank (K + N) flop over each operand once:
// a few rows are bound by reading W, many rows by the product with it.
//
// Two launches: the first computes h[m] = s_i A_i x[m] (rank values a row), the
// second the product with W, to whose fp32 accumulator it adds B_i h[m]:
//   * few rows (bf16): lora_rows_kernel, W as the 128-row operand of tcgen05
//     MMAs and the rows of x as its narrow one, K split over a cluster (a row or
//     two: h in the same launch);
//   * many rows (bf16): gemm_tc.cu's tiles with the adapters as further K
//     blocks (h as the sum of two bf16 parts, rows of other adapters masked off);
//   * fp32: lora_gemv_kernel (few rows) and lora_sgemm_kernel, on the CUDA cores;
//   * bf16 layouts that TMA does not take: lora_simt_kernel.
// Order of the launches: a kernel of the first kind waits for all earlier work
// before it lets its successor start, and writes h and the slot lists alone.
// The second may therefore read x and W, and write y, before its own wait for
// the first: only the adapters' part comes after it, so the first launch runs
// beside the product.
#include <math_constants.h>

#include "common.cuh"
#include "kernels.h"

namespace ck {

namespace {

struct LoraParams {
  ck_lora_args a;
  float* h;  // [M][rank]
};

// tensor-core path: h as the GEMM's operand and the adapters of every 128-row tile
struct TileParams {
  ck_lora_args a;
  uint8_t* h;         // [tiles][blocks of 64 ranks][parts][128 rows] (kernels.h)
  int32_t max_slots;  // per tile
  int32_t tiles;
  int32_t* cnt;       // [tiles]
  uint4* slots;       // [tiles][max_slots][2]
};

__device__ __forceinline__ float tofl(float v) { return v; }
__device__ __forceinline__ float tofl(__nv_bfloat16 v) { return bf2f(v); }
template <typename T>
__device__ __forceinline__ T fromf(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 fromf<__nv_bfloat16>(float v) { return f2bf(v); }

// 16 bytes as floats (4 fp32 or 8 bf16)
template <typename T>
__device__ __forceinline__ void load16(const T* p, float* f) {
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
  if constexpr (sizeof(T) == 2) {
    unpack8(v, f);
  } else {
    f[0] = __uint_as_float(v.x);
    f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z);
    f[3] = __uint_as_float(v.w);
  }
}

// Adapter of row m, -1 for none; one outside the table is recorded and counts as none.
__device__ __forceinline__ int adapter_of(const ck_lora_args& a, int64_t m, bool report) {
  const int id = __ldg(a.ids + m);
  if (id < a.n_adapters) return id < 0 ? -1 : id;
  if (report) set_status(CK_ERR_INDEX, (int)m, id);
  return -1;
}

// h: a warp per row and JB ranks, its lanes over K; the JB sums are reduced
// together (a lane gives half of its sums away at each step). Bound by latency: x
// and A come from L2 (48 rows, K 4096, rank 16: about 5 us, most of them beside the
// product).
template <typename T, int JB, bool VEC>
__global__ void __launch_bounds__(256) lora_shrink_kernel(const LoraParams p, int jblocks, int early) {
  grid_dep_wait();
  if (early) grid_dep_launch();
  const ck_lora_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= a.M * jblocks) return;
  const int64_t m = item / jblocks;
  const int j0 = (int)(item - m * jblocks) * JB;
  const int id = adapter_of(a, m, j0 == 0 && lane == 0);
  float acc[JB];
#pragma unroll
  for (int j = 0; j < JB; ++j) acc[j] = 0.f;
  if (id >= 0) {
    const T* x = reinterpret_cast<const T*>(a.x) + m * a.ldx;
    const T* A = reinterpret_cast<const T*>(a.a) + ((int64_t)id * a.rank + j0) * a.K;
    if constexpr (VEC) {
      constexpr int E = 16 / sizeof(T);
#pragma unroll 4
      for (int64_t k = lane * E; k < a.K; k += 32 * E) {
        float xv[E];
        load16(x + k, xv);
#pragma unroll
        for (int j = 0; j < JB; ++j) {
          if (j0 + j < a.rank) {
            float av[E];
            load16(A + j * a.K + k, av);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[j] = fmaf(xv[e], av[e], acc[j]);
          }
        }
      }
    } else {
      for (int64_t k = lane; k < a.K; k += 32) {
        const float xv = tofl(x[k]);
#pragma unroll
        for (int j = 0; j < JB; ++j)
          if (j0 + j < a.rank) acc[j] = fmaf(xv, tofl(A[j * a.K + k]), acc[j]);
      }
    }
  }
  if constexpr (JB == 8) {
#pragma unroll
    for (int w = 4, bit = 16; w > 0; w >>= 1, bit >>= 1) {
      const bool up = (lane & bit) != 0;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < w) {
          const float give = up ? acc[j] : acc[j + w];
          const float keep = up ? acc[j + w] : acc[j];
          acc[j] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
        }
    }
    float s = acc[0];
    s += __shfl_xor_sync(0xffffffffu, s, 2);
    s += __shfl_xor_sync(0xffffffffu, s, 1);
    const int j = j0 + (lane >> 2);
    if ((lane & 3) == 0 && j < a.rank)
      p.h[m * a.rank + j] = id < 0 ? 0.f : s * (a.scaling != nullptr ? __ldg(a.scaling + id) : 1.f);
  } else {
    const float s = warp_sum(acc[0]);
    if (lane == 0)
      p.h[m * a.rank + j0] = id < 0 ? 0.f : s * (a.scaling != nullptr ? __ldg(a.scaling + id) : 1.f);
  }
}

// ── fp32 ─────────────────────────────────────────────────────────────────────
//
// On the CUDA cores: TF32 tensor-core products would not match fp32.

__device__ __forceinline__ float adapter_part(const LoraParams& p, int id, int64_t m, int64_t n) {
  const float* b = reinterpret_cast<const float*>(p.a.b) + ((int64_t)id * p.a.N + n) * p.a.rank;
  const float* h = p.h + m * p.a.rank;
  float d = 0.f;
  for (int j = 0; j < p.a.rank; ++j) d = fmaf(h[j], __ldg(b + j), d);
  return d;
}

// Up to MR rows of x at a time: a warp a row of W, read once for them; bound by W
// (2 x 4096 x 4096 36 us a call, captured, 67 MB at 1.9 TB/s; 1 x 512 x 1536 4.1 us).
template <int MR, bool VEC>
__global__ void __launch_bounds__(256) lora_gemv_kernel(const LoraParams p) {
  grid_dep_wait();
  grid_dep_launch();
  const ck_lora_args& a = p.a;
  const int lane = threadIdx.x & 31;
  const int64_t n = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (n >= a.N) return;
  const int64_t m0 = (int64_t)blockIdx.y * MR;
  const float* w = reinterpret_cast<const float*>(a.w) + n * a.ldw;
  const float* x = reinterpret_cast<const float*>(a.x) + m0 * a.ldx;
  const int rows = (int)min((int64_t)MR, a.M - m0);
  float acc[MR];
#pragma unroll
  for (int r = 0; r < MR; ++r) acc[r] = 0.f;
  if constexpr (VEC) {
#pragma unroll 4
    for (int64_t k = 4 * lane; k < a.K; k += 128) {
      float wv[4];
      load16(w + k, wv);
#pragma unroll
      for (int r = 0; r < MR; ++r) {
        if (r < rows) {
          float xv[4];
          load16(x + r * a.ldx + k, xv);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[r] = fmaf(wv[e], xv[e], acc[r]);
        }
      }
    }
  } else {
    for (int64_t k = lane; k < a.K; k += 32) {
      const float wv = __ldg(w + k);
#pragma unroll
      for (int r = 0; r < MR; ++r)
        if (r < rows) acc[r] = fmaf(wv, __ldg(x + r * a.ldx + k), acc[r]);
    }
  }
  float mine = 0.f;  // lane r: row r's sum
#pragma unroll
  for (int r = 0; r < MR; ++r) {
    const float s = warp_sum(acc[r]);
    if (lane == r) mine = s;
  }
  if (lane < rows) {
    const int64_t m = m0 + lane;
    const int id = adapter_of(a, m, false);
    if (id >= 0) mine += adapter_part(p, id, m, n);
    if (a.bias != nullptr) mine += __ldg(reinterpret_cast<const float*>(a.bias) + n);
    reinterpret_cast<float*>(a.y)[m * a.ldy + n] = mine;
  }
}

// Tiles of 4 MT WM x 32 WN: a thread MT x 4 elements, rows lm + 4 i and columns
// ln + 8 j of its warp's 4 MT x 32. Both operands come in by asynchronous
// copies (16 bytes each, or 4 where rows are not 16-byte aligned), slices of 32
// along K, three slices ahead; rows padded to 36 floats, so that the 16-byte
// reads of 4 and 8 rows meet in no bank. The adapters are further slices: 32
// ranks of h against 32 ranks of B_i for each adapter i of the tile's rows, added to the
// rows that name it alone (chosen, not multiplied by zero: an infinity of one
// adapter stays with its rows). A slice is summed by itself, even and odd k in
// the two halves of paired FMAs, and added to the total: K / 32 + 16 roundings
// in a row instead of K. Where the tiles leave SMs idle, the SK CTAs of a cluster
// share one: each takes a part of K and every SK-th adapter, and finishes TM / SK
// rows from the partial tiles in distributed shared memory, in rank order. Bound
// by the FMA pipe: 1266 x 4096 x 4096 1207 us, 35 TF/s; 301 x 256 x 768 12.7 us a call
// (captured).
template <int MT, int WM, int WN, int SK, bool VEC>
__global__ void __launch_bounds__(32 * WM * WN, 3)
    lora_sgemm_kernel(const LoraParams p, int n_tiles) {
  constexpr int TM = 4 * MT * WM, TN = 32 * WN, TK = 32, LD = TK + 4, NS = 4;
  constexpr int THREADS = 32 * WM * WN;
  static_assert(TM <= THREADS, "a thread lists one row's adapter");
  extern __shared__ __align__(16) float sm[];  // [NS][TM + TN][LD]
  __shared__ int s_id[TM], s_list[TM];
  __shared__ int s_first[THREADS / 32];
  grid_dep_wait();
  grid_dep_launch();
  const ck_lora_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lm = lane >> 3, ln = lane & 7;
  const int wm = warp / WN, wn = warp % WN;
  const int rank = SK > 1 ? (int)cl_rank() : 0;
  const int64_t m0 = (int64_t)(blockIdx.x / SK / n_tiles) * TM;
  const int64_t n0 = (int64_t)(blockIdx.x / SK % n_tiles) * TN;
  const float* x = reinterpret_cast<const float*>(a.x);
  const float* w = reinterpret_cast<const float*>(a.w);
  const float* B = reinterpret_cast<const float*>(a.b);
  // this CTA's slices of K: [k_first, k_first + slices)
  const int all = (int)((a.K + TK - 1) / TK);
  const int k_first = (int)((int64_t)all * rank / SK);
  const int slices = (int)((int64_t)all * (rank + 1) / SK) - k_first;
  const int64_t k_begin = (int64_t)k_first * TK;
  const int rank_slices = (a.rank + TK - 1) / TK;
  int total = slices;  // and those of the adapters, once they are listed

  // columns [c, c + TK) of TM rows of `left` and TN rows of `right` into the
  // ring slot of slice s
  auto fetch = [&](int s, const float* left, int64_t ld_l, const float* right, int64_t ld_r,
                   int64_t c0, int64_t width, bool vec) {
    const uint32_t dst = smem_u32(sm + (s % NS) * (TM + TN) * LD);
    auto copy = [&](int r, int c, int n) {
      const int64_t k = c0 + c;
      const bool in = k < width && (r < TM ? m0 + r < a.M : n0 + r - TM < a.N);
      const float* src = r < TM ? left + (in ? r * ld_l + k : 0) : right + (in ? (r - TM) * ld_r + k : 0);
      const uint32_t to = dst + (r * LD + c) * 4;
      if (n == 4)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(in ? 16 : 0) : "memory");
      else
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(src), "r"(in ? 4 : 0) : "memory");
    };
    if (vec) {  // (width a multiple of 4)
#pragma unroll
      for (int i = tid; i < (TM + TN) * (TK / 4); i += THREADS) copy(i / (TK / 4), i % (TK / 4) * 4, 4);
    } else {
      for (int i = tid; i < (TM + TN) * TK; i += THREADS) copy(i / TK, i % TK, 1);
    }
  };
  // slices of K: this thread's pieces of them, whose addresses advance by a slice
  constexpr int PIECES = (TM + TN) * (TK / 4) / THREADS;
  static_assert((TM + TN) * (TK / 4) % THREADS == 0, "whole pieces per thread");
  const float* src[VEC ? PIECES : 1];
  uint32_t there = 0u;
  if constexpr (VEC) {
#pragma unroll
    for (int q = 0; q < PIECES; ++q) {
      const int i = tid + q * THREADS, r = i / (TK / 4), c = i % (TK / 4) * 4;
      const int64_t row = r < TM ? m0 + r : n0 + r - TM;
      const bool in = row < (r < TM ? a.M : a.N);
      src[q] = (r < TM ? x + (in ? row : 0) * a.ldx : w + (in ? row : 0) * a.ldw) + k_begin + c;
      there |= (uint32_t)in << q;
    }
  }
  auto fetch_slice = [&](int s) {
    if (s < slices) {
      if constexpr (VEC) {
        const uint32_t dst = smem_u32(sm + (s % NS) * (TM + TN) * LD);
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
          const int i = tid + q * THREADS, r = i / (TK / 4), c = i % (TK / 4) * 4;
          const bool in = ((there >> q) & 1u) && (s + 1 < slices || k_begin + s * (int64_t)TK + c < a.K);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + (r * LD + c) * 4),
                       "l"(in ? src[q] : x), "r"(in ? 16 : 0)
                       : "memory");
          src[q] += TK;
        }
      } else {
        fetch(s, x + m0 * a.ldx, a.ldx, w + n0 * a.ldw, a.ldw, k_begin + (int64_t)s * TK, a.K,
              false);
      }
    } else if (s < total) {
      const int item = rank + SK * ((s - slices) / rank_slices);
      const int c0 = (s - slices) % rank_slices * TK;
      fetch(s, p.h + m0 * a.rank, a.rank, B + ((int64_t)s_list[item] * a.N + n0) * a.rank, a.rank, c0,
            a.rank, a.rank % 4 == 0 && (reinterpret_cast<uintptr_t>(B) & 15u) == 0);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the first slices are on their way before the adapters are listed, unless K
  // ends within them
  if (slices >= NS - 1)
    for (int s = 0; s < NS - 1; ++s) fetch_slice(s);
  // the tile's adapters, in the order of their first row
  if (tid < TM) s_id[tid] = m0 + tid < a.M ? adapter_of(a, m0 + tid, false) : -1;
  __syncthreads();
  {
    const int id = tid < TM ? s_id[tid] : -1;
    const uint32_t peers = __match_any_sync(0xffffffffu, id);
    bool first = id >= 0 && (peers & ((1u << lane) - 1u)) == 0u;
    for (int j = 0; j < min(warp * 32, TM); ++j) first = first && s_id[j] != id;
    const uint32_t fm = __ballot_sync(0xffffffffu, first);
    if (lane == 0) s_first[warp] = __popc(fm);
    __syncthreads();
    int before = __popc(fm & ((1u << lane) - 1u)), count = 0;
#pragma unroll
    for (int v = 0; v < THREADS / 32; ++v) {
      if (v < warp) before += s_first[v];
      count += s_first[v];
    }
    if (first) s_list[before] = id;
    __syncthreads();
    total = slices + (count > rank ? (count - rank + SK - 1) / SK : 0) * rank_slices;
  }
  if (slices < NS - 1)
    for (int s = 0; s < NS - 1; ++s) fetch_slice(s);
  int my_id[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) my_id[i] = s_id[wm * 4 * MT + lm + 4 * i];

  float acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  for (int s = 0; s < total; ++s) {
    asm volatile("cp.async.wait_group %0;" ::"n"(NS - 2) : "memory");
    __syncthreads();  // the slice is there, and everyone has left the one before
    fetch_slice(s + NS - 1);
    const float* A = sm + (s % NS) * (TM + TN) * LD + (wm * 4 * MT + lm) * LD;
    const float* W = sm + (s % NS) * (TM + TN) * LD + (TM + wn * 32 + ln) * LD;
    unsigned long long part[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) part[i][j] = 0ull;
#pragma unroll
    for (int k = 0; k < TK; k += 4) {
      ulonglong2 wv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) wv[j] = *reinterpret_cast<const ulonglong2*>(W + 8 * j * LD + k);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const ulonglong2 av = *reinterpret_cast<const ulonglong2*>(A + 4 * i * LD + k);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          part[i][j] = ffma2(av.x, wv[j].x, part[i][j]);
          part[i][j] = ffma2(av.y, wv[j].y, part[i][j]);
        }
      }
    }
    const int only = s < slices ? -2 : s_list[rank + SK * ((s - slices) / rank_slices)];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float lo, hi;
        f2up(part[i][j], lo, hi);
        if (only == -2 || my_id[i] == only) acc[i][j] += lo + hi;
      }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  const float* bias = reinterpret_cast<const float*>(a.bias);
  float* y = reinterpret_cast<float*>(a.y);
  if constexpr (SK > 1) {
    __syncthreads();  // the ring is drained: the partial tile takes its place
    float* part = sm;  // [TM][TN]
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        part[(wm * 4 * MT + lm + 4 * i) * TN + wn * 32 + ln + 8 * j] = acc[i][j];
    cl_sync();
    constexpr int ROWS = TM / SK;
    static_assert(TM % SK == 0, "whole rows per CTA");
    for (int i = tid; i < ROWS * TN; i += THREADS) {
      const int r = rank * ROWS + i / TN, c = i % TN;
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < SK; ++k) {
        float f;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(f)
                     : "r"(cl_map(part + r * TN + c, k))
                     : "memory");
        v += f;
      }
      if (m0 + r < a.M && n0 + c < a.N)
        y[(m0 + r) * a.ldy + n0 + c] = v + (bias != nullptr ? __ldg(bias + n0 + c) : 0.f);
    }
    cl_sync();  // no CTA leaves while another reads its partials
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + wn * 32 + ln + 8 * j;
      if (n >= a.N) continue;
      const float bj = bias != nullptr ? __ldg(bias + n) : 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + wm * 4 * MT + lm + 4 * i;
        if (m < a.M) y[m * a.ldy + n] = acc[i][j] + bj;
      }
    }
  }
}

// bf16 whose strides break TMA's 16-byte rules: 64 x 64 tiles, 4 x 4 a thread,
// the next K slice in registers while this one is multiplied. Not made for speed:
// 2000 x 510 x 1536 229 us, where 2000 x 512 x 1536 takes 12 by the tiles (captured).
__global__ void __launch_bounds__(256) lora_simt_kernel(const LoraParams p, int n_tiles) {
  using T = __nv_bfloat16;
  constexpr int TM = 64, TN = 64, TK = 16;
  __shared__ __align__(16) float As[TK][TM + 4];
  __shared__ __align__(16) float Ws[TK][TN + 4];
  __shared__ int s_id[TM];
  grid_dep_wait();
  grid_dep_launch();
  const ck_lora_args& a = p.a;
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int64_t m0 = (int64_t)(blockIdx.x / n_tiles) * TM;
  const int64_t n0 = (int64_t)(blockIdx.x % n_tiles) * TN;
  if (tid < TM) s_id[tid] = m0 + tid < a.M ? adapter_of(a, m0 + tid, false) : -1;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* w = reinterpret_cast<const T*>(a.w);
  const int lr = tid / 4, lk = (tid % 4) * 4;  // this thread's 4 elements of a slice
  float xr[4], wr[4];
  auto fetch = [&](int64_t k0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t k = k0 + lk + i;
      xr[i] = (m0 + lr < a.M && k < a.K) ? tofl(x[(m0 + lr) * a.ldx + k]) : 0.f;
      wr[i] = (n0 + lr < a.N && k < a.K) ? tofl(w[(n0 + lr) * a.ldw + k]) : 0.f;
    }
  };
  float acc[4][4] = {};
  fetch(0);
  for (int64_t k0 = 0; k0 < a.K; k0 += TK) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      As[lk + i][lr] = xr[i];
      Ws[lk + i][lr] = wr[i];
    }
    __syncthreads();
    if (k0 + TK < a.K) fetch(k0 + TK);
#pragma unroll
    for (int kk = 0; kk < TK; ++kk) {
      const float4 av = *reinterpret_cast<const float4*>(&As[kk][4 * ty]);
      const float4 bv = *reinterpret_cast<const float4*>(&Ws[kk][4 * tx]);
      const float af[4] = {av.x, av.y, av.z, av.w}, bf[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(af[i], bf[j], acc[i][j]);
    }
  }
  const T* B = reinterpret_cast<const T*>(a.b);
  const T* bias = reinterpret_cast<const T*>(a.bias);
  T* y = reinterpret_cast<T*>(a.y);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t m = m0 + 4 * ty + i;
    if (m >= a.M) continue;
    const int id = s_id[4 * ty + i];
    const float* h = p.h + m * a.rank;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + 4 * tx + j;
      if (n >= a.N) continue;
      float v = acc[i][j];
      if (id >= 0) {
        const T* br = B + ((int64_t)id * a.N + n) * a.rank;
        float d = 0.f;
        for (int r = 0; r < a.rank; ++r) d = fmaf(h[r], tofl(br[r]), d);
        v += d;
      }
      if (bias != nullptr) v += tofl(bias[n]);
      y[m * a.ldy + n] = fromf<T>(v);
    }
  }
}

// ── many rows: h and the tiles' adapters ─────────────────────────────────────
//
// A cluster of SK CTAs per 128-row tile of x and SL adapters. It lists the
// tile's adapters in the order of their first row (with, for each, the rows that
// are not its own) and computes D[128 x SL RP] = x_tile A^T for its SL of them,
// one MMA's columns: both operands by TMA into a ring of 64-wide K blocks whose
// depth is what the adapters' number leaves, each CTA an SK-th of K. A row then takes the columns of its own
// adapter; the ranks' partials meet in distributed shared memory, each CTA
// finishing RP / SK columns: sum in rank order, times s_i, as two bf16 parts, each
// written as the GEMM's operand lies in shared memory. (The first alone leaves 2^-8
// |B||h|, as large as the result's own rounding; captured, us, with and without the
// second: 8192 x 512 x 1536 in runs 22.0 / 21.6, 12001 x 768 x 2304 49.0 / 47.9, 64
// adapters by rows 80.7 / 78.8.) Bound by x, read once a cluster; clusters whose SL the
// tile has no adapters for leave after the list. h of rows without an adapter stays
// unwritten: no block of the GEMM uses it. 8192 x 512, 8 adapters of rank 16: 10.2 us
// from cold caches, of which the chain ids, list, first operands, partials, sum is
// all; its bytes would take 1.5.
// N words (1, 2 or 4), aligned as one
template <int N>
__device__ __forceinline__ void store_words(void* to, const uint32_t* w) {
  if constexpr (N == 4) *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(to) = w[0];
}

template <int RP, int SK>
struct TilesCfg {
  static constexpr int SL = 256 / RP;  // one MMA's columns
  static constexpr int X_BYTES = 128 * 128;
  static constexpr int A_BYTES = RP * 128;
  static constexpr int RING = 96 * 1024;  // two CTAs an SM
  static constexpr int STAGES = RING / (X_BYTES + A_BYTES);  // (fewer with more adapters)
  static constexpr int SMEM = 1024 + RING + 256;
  static constexpr uint32_t COLS = 256;
  static_assert(RP * 128 * 4 <= RING, "the partials lie over the drained ring");
};

template <int RP, int SK>
__global__ void __launch_bounds__(128) lora_tiles_kernel(const __grid_constant__ CUtensorMap tmX,
                                                         const __grid_constant__ CUtensorMap tmA,
                                                         const TileParams p) {
  using C = TilesCfg<RP, SK>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int s_id[128], s_list[128];
  __shared__ uint32_t s_first[4];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* part = reinterpret_cast<float*>(smem);  // [RP][128], once the ring is drained
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::RING);
  uint64_t* empty = full + C::STAGES;
  uint64_t* done = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const ck_lora_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = SK > 1 ? (int)cl_rank() : 0;
  const int tile = (int)(blockIdx.x / SK) % p.tiles;
  const int slot0 = (int)(blockIdx.x / SK) / p.tiles * C::SL;  // this cluster's first adapter of the tile
  const int kb_all = (int)((a.K + 63) / 64);
  const int kb_per = (kb_all + SK - 1) / SK;
  const int kb0 = min(kb_all, rank * kb_per), kb1 = min(kb_all, kb0 + kb_per);

  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmA);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_wait();
  grid_dep_launch();

  // the tile's adapters
  const int64_t m = (int64_t)tile * 128 + tid;
  const bool lists = rank == 0 && slot0 == 0;  // the CTA that writes the tile's list
  const int id = m < a.M ? adapter_of(a, m, lists) : -1;
  s_id[tid] = id;
  __syncthreads();
  const uint32_t lt = (1u << lane) - 1u;
  const uint32_t peers = __match_any_sync(0xffffffffu, id);  // (every lane, with an adapter or without)
  bool first = id >= 0 && (peers & lt) == 0u;
  for (int j = 0; j < warp * 32; ++j) first = first && s_id[j] != id;
  const uint32_t fm = __ballot_sync(0xffffffffu, first);
  if (lane == 0) s_first[warp] = fm;
  __syncthreads();
  int before = __popc(fm & lt), total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < warp) before += __popc(s_first[w]);
    total += __popc(s_first[w]);
  }
  if (first) s_list[before] = id;
  __syncthreads();
  int slot = -1;  // this row's place in the list
  for (int i = 0; i < total; ++i) {
    const bool mine = id == s_list[i];
    const uint32_t mask = __ballot_sync(0xffffffffu, mine);
    if (mine) slot = i;
    if (lists) {
      uint4* dst = p.slots + 2 * ((int64_t)tile * p.max_slots + i);
      if (lane == 0) reinterpret_cast<uint32_t*>(dst + 1)[warp] = ~mask;
      if (tid == 0) dst[0] = make_uint4((uint32_t)s_list[i], 0u, 0u, 0u);
    }
  }
  if (lists && tid == 0) p.cnt[tile] = total;
  const float scale = id >= 0 && a.scaling != nullptr ? __ldg(a.scaling + id) : 1.f;

  // a pass per RP ranks (one, up to 64); none without adapters from slot0 on
  const int n_slots = min(C::SL, total - slot0);
  const int passes = n_slots > 0 ? (a.rank + RP - 1) / RP : 0;
  // a stage: 64 columns of x, then of the adapters' A one after the other
  const int stage_bytes = C::X_BYTES + max(n_slots, 1) * C::A_BYTES;
  const int stages = min(C::STAGES, C::RING / stage_bytes);
  int stage = 0, issued = 0;  // of the producing and of the multiplying thread
  uint32_t phase = 0;
  for (int pass = 0; pass < passes; ++pass) {
    const int j0 = pass * RP;
    if (warp == 0 && lane == 0) {
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, 30)) break;
        mbar_arrive_expect_tx(&full[stage], (uint32_t)stage_bytes);
        uint8_t* to = smem + stage * stage_bytes;
        tma_load_2d(to, &tmX, &full[stage], kb * 64, tile * 128);
        for (int i = 0; i < n_slots; ++i)  // (rows past the rank are columns that nobody takes)
          tma_load_2d(to + C::X_BYTES + i * C::A_BYTES, &tmA, &full[stage], kb * 64,
                      s_list[slot0 + i] * a.rank + j0);
        ++issued;
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (*abort_flag != 0)  // a wait ran out: no copy may land after this CTA's exit
        for (int s = 0; s < stages && s < issued; ++s) {
          const int last = issued - 1 - ((issued - 1 - s) % stages);
          mbar_wait(&full[s], (uint32_t)((last / stages) & 1), nullptr, 33);
        }
    } else if (warp == 1 && lane == 0) {
      const uint32_t idesc = idesc_bf16(128, (uint32_t)(n_slots * RP), 0u);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, 31)) break;
        tc_fence_after();
        const uint32_t xa = smem_u32(smem + stage * stage_bytes), aa = xa + C::X_BYTES;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          tc_mma_ss(tmem, sw128_desc(xa + k * 32, 16, 1024), sw128_desc(aa + k * 32, 16, 1024),
                    idesc, (kb != kb0 || k != 0) ? 1u : 0u);
        tc_commit(&empty[stage]);
        if (++stage == stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      tc_commit(done);
      mbar_wait(done, (uint32_t)(pass & 1), nullptr, 32);
    }
    __syncthreads();
    tc_fence_after();
    const int mine = slot - slot0;  // 0 .. n_slots - 1: this row's columns are here
    const bool take = mine >= 0 && mine < n_slots;
    for (int i = 0; i < n_slots; ++i) {
      if (!__any_sync(0xffffffffu, mine == i)) continue;
#pragma unroll
      for (int c = 0; c < RP; c += 16) {
        uint32_t v[16];
        tmem_ld16w(tmem + ((uint32_t)(warp * 32) << 16) + i * RP + c, v);
        tc_wait_ld();
        if (mine == i) {
#pragma unroll
          for (int e = 0; e < 16; ++e)
            part[(c + e) * 128 + tid] = kb1 > kb0 ? __uint_as_float(v[e]) : 0.f;
        }
        __syncwarp();
      }
    }
    tc_fence_before();
    if (SK > 1) cl_sync(); else __syncthreads();
    if (take && *abort_flag == 0) {
      constexpr int PER = RP / SK;
      const int c0 = rank * PER;
      uint32_t src[SK];
#pragma unroll
      for (int r = 0; r < SK; ++r) src[r] = SK > 1 ? cl_map(part + tid, r) : smem_u32(part + tid);
      constexpr int W = PER < 8 ? PER : 8;  // columns a store (16 bytes where there are 8)
      constexpr int ROW = 2 * RP;
      auto swizzled = [](int at) { return at ^ (((at >> 7) & (ROW / 16 - 1)) << 4); };
      uint8_t* to = p.h + ((int64_t)tile * ((a.rank + 63) / 64) + pass) * 2 * 128 * ROW;
#pragma unroll
      for (int c = 0; c < PER; c += W) {
        uint32_t high[W / 2], low[W / 2];
#pragma unroll
        for (int e = 0; e < W; e += 2) {
          float v[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int r = 0; r < SK; ++r) {
              float f;
              asm volatile("ld.shared::cluster.f32 %0, [%1];"
                           : "=f"(f)
                           : "r"(src[r] + (c0 + c + e + i) * 512)
                           : "memory");
              v[i] += f;
            }
            v[i] = j0 + c0 + c + e + i < a.rank ? v[i] * scale : 0.f;
          }
          two_bf16x2(v[0], v[1], high[e / 2], low[e / 2]);
          if (fabsf(v[0]) == CUDART_INF_F) low[e / 2] = (low[e / 2] & 0xffff0000u) | (high[e / 2] & 0xffffu);
          if (fabsf(v[1]) == CUDART_INF_F) low[e / 2] = (low[e / 2] & 0xffffu) | (high[e / 2] & 0xffff0000u);
        }
        const int at = tid * ROW + (c0 + c) * 2;
        store_words<W / 2>(to + swizzled(at), high);
        store_words<W / 2>(to + 128 * ROW + swizzled(at), low);
      }
    }
    // the partials (for the next pass's copies) and the accumulators are free again
    fence_proxy_async_smem();
    if (SK > 1) cl_sync(); else __syncthreads();
    tc_fence_after();
  }
  if (warp == 1) tmem_dealloc(tmem, C::COLS);
}

// Row copies with a change of stride: B rows padded to 16-byte rows (rank not
// a multiple of 8; 2000 x 512 x 1536 of rank 12 16 us against 12 of rank 16), and y
// out of the padded staging rows (N or ldy not one; 24 us at N 1535).
__global__ void __launch_bounds__(256) lora_copy_kernel(const __nv_bfloat16* src, int64_t ld_src,
                                                        __nv_bfloat16* dst, int64_t ld_dst,
                                                        int64_t rows, int64_t cols) {
  grid_dep_wait();
  grid_dep_launch();
  const int64_t total = rows * cols;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / cols, c = i - r * cols;
    dst[r * ld_dst + c] = src[r * ld_src + c];
  }
}

// ── few rows ─────────────────────────────────────────────────────────────────
//
// W is read once and bounds the call, so it is the operand that streams: a CTA
// takes 128 rows of W and NTOK rows of x, D[128 x NTOK] = W_tile x^T in TMEM,
// both operands by TMA into a ring of 64-wide K blocks. The SK CTAs of a
// cluster share a tile, each an SK-th of K, so that a small W still fills the
// SMs; they exchange their fp32 partials through distributed shared memory,
// each finishing NTOK / SK of the rows: sum over the ranks in order, adapter
// and bias added, one rounding, a warp storing 32 neighbouring columns. 48 rows,
// K = N = 4096: 18 us a call (captured), W at 1.9 TB/s.
//
// ONE: no first launch. Each CTA computes its K part of every row's h = A_i x in
// the two warps that have nothing else to do, and the parts meet as the others
// do. Every tile of W does that again, so only a few values are left to it.

template <int NTOK, int SK>
struct RowsCfg {
  static constexpr int W_BYTES = 128 * 128;
  static constexpr int X_BYTES = NTOK * 128;
  static constexpr int STAGE = W_BYTES + X_BYTES;
  static constexpr int STAGES = 96 * 1024 / STAGE;  // two CTAs an SM
  static constexpr int PART = 128 * NTOK * 4;  // partials, over the ring once it is drained
  static constexpr int RING = STAGES * STAGE > PART ? STAGES * STAGE : PART;
  static constexpr int SMEM = 1024 + RING + 256 + NTOK * 4;
  static constexpr uint32_t COLS = NTOK < 32 ? 32 : NTOK;
};

// Values of h (M rank) that lora_rows_kernel computes itself: as many as its two
// warps hold at once. One launch against two, us a call: 1 x 512 x 1536, rank 16, eager
// 13.1 / 17.6, captured 4.65 / 4.83; captured 1 x 4096 x 4096, rank 32, 10.5 / 10.1; with 64
// values 4 x 512 x 1536, rank 16, 5.7 / 5.2.
constexpr int kOneH = 32;

template <int NTOK, int SK, bool ONE>
__global__ void __launch_bounds__(128) lora_rows_kernel(const __grid_constant__ CUtensorMap tmW,
                                                        const __grid_constant__ CUtensorMap tmX,
                                                        const LoraParams p, int n_tiles) {
  using C = RowsCfg<NTOK, SK>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  uint8_t* sW = smem;
  uint8_t* sX = smem + C::STAGES * C::W_BYTES;
  float* part = reinterpret_cast<float*>(smem);  // [NTOK][128]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::RING);
  uint64_t* empty = full + C::STAGES;
  uint64_t* done = empty + C::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* s_id = reinterpret_cast<int*>(smem + C::RING + 256);  // [NTOK] adapters of the rows
  __shared__ float s_part[ONE ? kOneH : 1];  // h of this CTA's part of K
  __shared__ __align__(16) float s_h[ONE ? kOneH : 1];  // h of the rows that it finishes
  const ck_lora_args& a = p.a;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = SK > 1 ? (int)cl_rank() : 0;
  const int unit = blockIdx.x / SK;
  const int n0 = (unit % n_tiles) * 128;
  const int64_t m0 = (int64_t)(unit / n_tiles) * NTOK;
  const int kb_all = (int)((a.K + 63) / 64);
  const int kb_per = (kb_all + SK - 1) / SK;
  const int kb0 = min(kb_all, rank * kb_per), kb1 = min(kb_all, kb0 + kb_per);

  if (tid == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tmW);
    prefetch_tmap(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (ONE) {
    grid_dep_wait();
    grid_dep_launch();
  }

  constexpr int PER = (NTOK + SK - 1) / SK;  // rows of x that this CTA finishes
  const int c0 = rank * PER;
  const int rows = max(0, min(min(PER, NTOK - c0), (int)min((int64_t)NTOK, a.M - m0) - c0));
  bool ok = true;
  if (warp >= 2) {
    // the idle warps fetch the adapters' rows that the epilogue will read
    for (int c = tid - 64; c < rows; c += 64) s_id[c] = adapter_of(a, m0 + c0 + c, ONE && n0 == 0);
    asm volatile("bar.sync 1, 64;" ::: "memory");
    const int64_t line = (int64_t)min((int64_t)128, a.N - n0) * a.rank * 2;  // bytes of B_i's 128 rows
    for (int c = 0; c < rows; ++c)
      if (s_id[c] >= 0) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(a.b) +
                             ((int64_t)s_id[c] * a.N + n0) * a.rank * 2;
        for (int64_t o = (tid - 64) * 128; o < line; o += 64 * 128)
          asm volatile("prefetch.global.L2 [%0];" ::"l"(src + o));
      }
    if constexpr (ONE) {
      // 8 lanes for VB values of h, 16 bytes of a K block each
      constexpr int VB = kOneH / 8;
      const int values = (int)a.M * a.rank, sub = lane & 7;
      const __nv_bfloat16 *x[VB], *A[VB];
      float d[VB];
      bool in[VB];
#pragma unroll
      for (int i = 0; i < VB; ++i) {
        const int v = (tid - 64) / 8 + 8 * i;
        const int r = min(v, values - 1) / a.rank, j = min(v, values - 1) - r * a.rank;
        const int id = v < values ? adapter_of(a, r, false) : -1;
        in[i] = id >= 0;
        x[i] = reinterpret_cast<const __nv_bfloat16*>(a.x) + r * a.ldx;
        A[i] = reinterpret_cast<const __nv_bfloat16*>(a.a) + ((int64_t)max(id, 0) * a.rank + j) * a.K;
        d[i] = 0.f;
      }
#pragma unroll 2
      for (int kb = kb0; kb < kb1; ++kb) {
        const int64_t k = kb * (int64_t)64 + sub * 8;
        float xv[VB][8], av[VB][8];
#pragma unroll
        for (int i = 0; i < VB; ++i) {
          const bool here = in[i] && k < a.K;
          const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
          unpack8(here ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : zero, xv[i]);
          unpack8(here ? __ldg(reinterpret_cast<const uint4*>(A[i] + k)) : zero, av[i]);
        }
#pragma unroll
        for (int i = 0; i < VB; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e) d[i] = fmaf(xv[i][e], av[i][e], d[i]);
      }
#pragma unroll
      for (int i = 0; i < VB; ++i) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) d[i] += __shfl_xor_sync(0xffffffffu, d[i], o);
        const int v = (tid - 64) / 8 + 8 * i;
        if (sub == 0 && v < values) s_part[v] = d[i];
      }
    }
  }
  if (warp == 0 && lane == 0) {
    int issued = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++issued) {
      const int s = issued % C::STAGES;
      if (!mbar_wait(&empty[s], ((issued / C::STAGES) & 1) ^ 1, abort_flag, 20)) break;
      mbar_arrive_expect_tx(&full[s], C::STAGE);
      tma_load_2d(sW + s * C::W_BYTES, &tmW, &full[s], kb * 64, n0);
      tma_load_2d(sX + s * C::X_BYTES, &tmX, &full[s], kb * 64, (int)m0);
    }
    // every copy lands before this CTA can exit or reuse the ring
    for (int s = 0; s < C::STAGES && s < issued; ++s) {
      const int last = issued - 1 - ((issued - 1 - s) % C::STAGES);
      mbar_wait(&full[s], (uint32_t)((last / C::STAGES) & 1), nullptr, 21);
    }
  } else if (warp == 1 && lane == 0) {
    constexpr uint32_t idesc = idesc_bf16(128, NTOK, 0u);
    int i = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++i) {
      const int s = i % C::STAGES;
      if (!mbar_wait(&full[s], (uint32_t)((i / C::STAGES) & 1), abort_flag, 22)) break;
      tc_fence_after();
      const uint32_t wa = smem_u32(sW + s * C::W_BYTES), xa = smem_u32(sX + s * C::X_BYTES);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        tc_mma_ss(tmem, sw128_desc(wa + k * 32, 16, 1024), sw128_desc(xa + k * 32, 16, 1024), idesc,
                  (i | k) != 0 ? 1u : 0u);
      tc_commit(&empty[s]);
    }
    tc_commit(done);
    mbar_wait(done, 0, nullptr, 23);
  }
  __syncthreads();  // (the two threads above come back once the ring is drained)
  tc_fence_after();
  ok = *abort_flag == 0;

  // partials: lane n of the accumulator, column by column
  {
    const uint32_t base = tmem + ((uint32_t)(warp * 32) << 16);
#pragma unroll
    for (int c = 0; c < NTOK; c += 16) {
      uint32_t v[16];
      if (kb1 > kb0) {
        tmem_ld16w(base + c, v);
        tc_wait_ld();
      }
#pragma unroll
      for (int i = 0; i < 16; ++i)
        part[(c + i) * 128 + tid] = kb1 > kb0 ? __uint_as_float(v[i]) : 0.f;
    }
  }
  tc_fence_before();
  if (!ONE) {
    grid_dep_wait();  // h is there
    grid_dep_launch();
  }
  if (SK > 1) cl_sync(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::COLS);
  }
  if constexpr (ONE) {
    for (int i = tid; i < rows * a.rank; i += 128) {
      const int id = s_id[i / a.rank];
      float v = 0.f;
#pragma unroll
      for (int r = 0; r < SK; ++r) {
        float f;
        asm volatile("ld.shared::cluster.f32 %0, [%1];"
                     : "=f"(f)
                     : "r"((SK > 1 ? cl_map(s_part, r) : smem_u32(s_part)) + (c0 * a.rank + i) * 4)
                     : "memory");
        v += f;
      }
      s_h[i] = id >= 0 && a.scaling != nullptr ? v * __ldg(a.scaling + id) : v;
    }
    __syncthreads();
  }
  const float* h_rows = ONE ? s_h : p.h + (m0 + c0) * a.rank;  // of the rows that it finishes
  const int n = n0 + tid;
  if (ok && n < a.N) {
    constexpr int UB = PER < 4 ? PER : 4;  // rows in flight
    uint32_t src[SK];
#pragma unroll
    for (int r = 0; r < SK; ++r) src[r] = SK > 1 ? cl_map(part + tid, r) : smem_u32(part + tid);
    const float bias = a.bias != nullptr ? bf2f(reinterpret_cast<const __nv_bfloat16*>(a.bias)[n]) : 0.f;
    const __nv_bfloat16* B = reinterpret_cast<const __nv_bfloat16*>(a.b);
    const bool vec = a.rank % 8 == 0;  // (b is 16-byte aligned)
    for (int c = 0; c < rows; c += UB) {
      float v[UB];
#pragma unroll
      for (int u = 0; u < UB; ++u) {
        v[u] = bias;
#pragma unroll
        for (int r = 0; r < SK; ++r) {
          float f = 0.f;
          if (c + u < rows)
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(f)
                         : "r"(src[r] + (c0 + c + u) * 512)
                         : "memory");
          v[u] += f;
        }
      }
      for (int j = 0; j < a.rank; j += 8) {
        uint4 w[UB];
        float4 h0[UB], h1[UB];
#pragma unroll
        for (int u = 0; u < UB; ++u) {
          const int id = c + u < rows ? s_id[c + u] : -1;
          w[u] = make_uint4(0u, 0u, 0u, 0u);
          h0[u] = h1[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (id < 0) continue;
          const __nv_bfloat16* br = B + ((int64_t)id * a.N + n) * a.rank + j;
          const float* h = h_rows + (c + u) * a.rank + j;
          if (vec) {
            w[u] = __ldg(reinterpret_cast<const uint4*>(br));
            h0[u] = *reinterpret_cast<const float4*>(h);
            h1[u] = *reinterpret_cast<const float4*>(h + 4);
          } else {
            uint32_t e[8];
            float g[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              e[i] = j + i < a.rank ? (uint32_t)__bfloat16_as_ushort(br[i]) : 0u;
              g[i] = j + i < a.rank ? h[i] : 0.f;
            }
            w[u] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
            h0[u] = make_float4(g[0], g[1], g[2], g[3]);
            h1[u] = make_float4(g[4], g[5], g[6], g[7]);
          }
        }
#pragma unroll
        for (int u = 0; u < UB; ++u) {
          if (c + u >= rows || s_id[c + u] < 0) continue;
          float f[8];
          unpack8(w[u], f);
          v[u] = fmaf(f[0], h0[u].x, v[u]);
          v[u] = fmaf(f[1], h0[u].y, v[u]);
          v[u] = fmaf(f[2], h0[u].z, v[u]);
          v[u] = fmaf(f[3], h0[u].w, v[u]);
          v[u] = fmaf(f[4], h1[u].x, v[u]);
          v[u] = fmaf(f[5], h1[u].y, v[u]);
          v[u] = fmaf(f[6], h1[u].z, v[u]);
          v[u] = fmaf(f[7], h1[u].w, v[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < UB; ++u)
        if (c + u < rows)
          reinterpret_cast<__nv_bfloat16*>(a.y)[(m0 + c0 + c + u) * a.ldy + n] = f2bf(v[u]);
    }
  }
  if (SK > 1) cl_sync();  // no CTA leaves while another reads its partials
}

enum Path { PATH_ROWS, PATH_TILES, PATH_F32, PATH_SIMT };

struct LoraPlan {
  LoraParams p;
  Path path;
  bool one;                       // PATH_ROWS: one launch, no workspace
  int max_slots, tiles;           // PATH_TILES
  int64_t ld_b, ld_stage;         // packed B / staged y row strides, 0: used in place
  size_t off_h, off_cnt, off_slots, off_b, off_y;
  size_t bytes;
};

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

// Whether lora_rows_kernel runs: its epilogue reads h and B_i once a row, where
// the tiles multiply B_i once for all rows that name it but take a block for each
// adapter of a tile. Measured (captured, us, rows against tiles; adapters all
// different, then in runs of 64 rows): 4 x 512 x 1536, rank 32, 6.0 against 9.2; 32 x
// 768 x 2304, rank 64, 13.2 against 27.2, in runs 13.5 against 9.1; 64 x 768 x 2304, rank
// 32, 13.8 against 29.6, in runs 13.7 against 8.6, rank 64, 25.8 against 46.7, in runs 23.9
// against 9.5. More rows than one operand of 64, only while all of them are few CTAs:
// 128 x 512 x 1536 (24 tiles of W by rows), rank 8, 16 adapters, 8.9 against 15.6; 256 x
// 4096 x 1024 (32), rank 32, 25.0 against 40.9; 192 x 512 x 1536 (36), 8 adapters of rank
// 16, 18.9 against 11.2. 512 x 512 x 512, rank 32, 20.2 against 33.0, in runs 20.8 against
// 10.6: more than 8192 values of h are left to the tiles.
bool by_rows(const ck_lora_args& a) {
  if (a.M <= 32) return true;
  if (a.rank > 32) return false;
  return a.M <= 64 || ((a.M + 63) / 64 * ((a.N + 127) / 128) <= 32 && a.M * a.rank <= 8192);
}

int make_plan(const ck_lora_args& a, LoraPlan& pl) {
  if (a.dtype != CK_F32 && a.dtype != CK_BF16) return CK_ERR_UNSUPPORTED;
  if (a.M < 0 || a.N < 0 || a.K <= 0 || a.rank < 1 || a.n_adapters < 0) return CK_ERR_INVALID_ARG;
  // (indexes inside a tile that reaches past the end stay below 2^31)
  if (a.M > (int64_t)1 << 28 || a.N > INT32_MAX - 256 || a.K > INT32_MAX - 256 || a.rank > 256)
    return CK_ERR_UNSUPPORTED;
  if (((a.M + 31) / 32) * ((a.N + 63) / 64) > INT32_MAX || (a.M * a.rank + 7) / 8 > INT32_MAX)
    return CK_ERR_UNSUPPORTED;
  pl.p.a = a;
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  const bool tma = a.dtype == CK_BF16 && a.K % 8 == 0 && a.ldx % 8 == 0 && a.ldw % 8 == 0 &&
                   aligned16(a.x) && aligned16(a.w) && aligned16(a.a) && aligned16(a.b) &&
                   (int64_t)a.n_adapters * a.N <= INT32_MAX - 256 &&
                   (int64_t)a.n_adapters * a.rank <= INT32_MAX - 256;
  pl.path = a.dtype == CK_F32 ? PATH_F32 : !tma ? PATH_SIMT : by_rows(a) ? PATH_ROWS : PATH_TILES;
  pl.one = pl.path == PATH_ROWS && a.M <= 16 && a.M * a.rank <= kOneH;
  if (pl.path != PATH_TILES) {
    pl.bytes = pl.one ? 0 : up((size_t)a.M * a.rank * 4);
    return CK_OK;
  }
  pl.tiles = (int)((a.M + 127) / 128);
  pl.max_slots = a.n_adapters < 1 ? 1 : (a.n_adapters < 128 ? a.n_adapters : 128);
  pl.ld_b = a.rank % 8 == 0 ? 0 : (a.rank + 7) / 8 * 8;
  pl.ld_stage = a.ldy % 8 == 0 && aligned16(a.y) ? 0 : (a.N + 7) / 8 * 8;
  pl.off_h = 0;
  // h: a tile's 128 rows of 16, 32 or 64 columns a block, twice
  pl.off_cnt = (size_t)pl.tiles * ((a.rank + 63) / 64) * 2 * 128 * (a.rank <= 16 ? 32 : a.rank <= 32 ? 64 : 128);
  pl.off_slots = pl.off_cnt + up((size_t)pl.tiles * 4);
  pl.off_b = pl.off_slots + up((size_t)pl.tiles * pl.max_slots * 32);
  pl.off_y = pl.off_b + up((size_t)a.n_adapters * a.N * pl.ld_b * 2);
  pl.bytes = pl.off_y + up((size_t)a.M * pl.ld_stage * 2);
  return CK_OK;
}

// early: its successor may start beside it. That pays where the successor streams
// W with a CTA or two an SM (captured, 48 rows x 4096 x 4096: 17.8 against 21.0 us); the
// fp32 tiles would crowd on the SMs that this kernel leaves free (301 x 256 x 768
// 15.8 against 12.7 us, 128 x 4096 x 4096 214 against 156).
template <typename T>
int shrink(const LoraParams& p, int early, cudaStream_t st) {
  const ck_lora_args& a = p.a;
  constexpr int E = 16 / sizeof(T);
  const bool vec = a.K % E == 0 && a.ldx % E == 0 && aligned16(a.x) && aligned16(a.a);
  // one rank a warp while that leaves SMs without work, else 8
  const bool wide = a.M * a.rank >= 8 * 16 * (int64_t)(num_sms() > 0 ? num_sms() : 148);
  const int jb = wide ? 8 : 1;
  const int jblocks = (a.rank + jb - 1) / jb;
  const dim3 grid((unsigned)((a.M * jblocks + 7) / 8));
  if (wide)
    return vec ? launch_pdl(lora_shrink_kernel<T, 8, true>, grid, dim3(256), 0, st, p, jblocks, early)
               : launch_pdl(lora_shrink_kernel<T, 8, false>, grid, dim3(256), 0, st, p, jblocks, early);
  return vec ? launch_pdl(lora_shrink_kernel<T, 1, true>, grid, dim3(256), 0, st, p, jblocks, early)
             : launch_pdl(lora_shrink_kernel<T, 1, false>, grid, dim3(256), 0, st, p, jblocks, early);
}

// Tiles of 32 x 64 (128 x 64 took 87 us where they take 65 at 1024 x 512 x 1536, and
// 1234 against 1189 at 1266 x 4096 x 4096).
template <int SK, bool VEC>
int launch_sgemm(const LoraParams& p, cudaStream_t st) {
  constexpr int MT = 4, WM = 2, WN = 2, TM = 4 * MT * WM, TN = 32 * WN;
  constexpr int smem = 4 * (TM + TN) * 36 * 4;
  auto kern = lora_sgemm_kernel<MT, WM, WN, SK, VEC>;
  if (!smem_attr_ready(reinterpret_cast<const void*>(kern), smem)) return record_cuda_error();
  const int n_tiles = (int)((p.a.N + TN - 1) / TN);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SK;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((p.a.M + TM - 1) / TM * n_tiles * SK));
  cfg.blockDim = dim3(32 * WM * WN);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return launch_cfg(cfg, kern, p, n_tiles);
}

template <bool VEC>
int run_f32(const LoraParams& p, cudaStream_t st) {
  const ck_lora_args& a = p.a;
  const unsigned gx = (unsigned)((a.N + 7) / 8);
  if (a.M == 1) return launch_pdl(lora_gemv_kernel<1, VEC>, dim3(gx), dim3(256), 0, st, p);
  // W once for 8 rows, against tiles whose K is split (us): 8 x 4096 x 4096 44 / 49, 16 67
  // / 51; 8 x 512 x 1536 7.2 / 9.5, 24 12.1 / 9.6; 24 x 2048 x 512 12.7 / 13.5, 24 x 256 x
  // 256 5.5 / 9.2.
  if (a.M <= 8 || (a.M <= 24 && a.N <= 1024))
    return launch_pdl(lora_gemv_kernel<8, VEC>, dim3(gx, (unsigned)((a.M + 7) / 8)), dim3(256), 0, st, p);
  // K split while the SMs (three CTAs each) have room and a CTA keeps two slices:
  // 32 x 4096 x 4096 51 us against 114 unsplit, 64 x 512 x 1536 12.4 against 21.4
  const int64_t tiles = (a.M + 31) / 32 * ((a.N + 63) / 64), slices = (a.K + 31) / 32;
  const int sms = num_sms() > 0 ? num_sms() : 148;
  int sk = 1;
  while (sk < 8 && 2 * tiles * sk <= 3 * sms && slices >= 4 * sk) sk *= 2;
  if (sk == 8) return launch_sgemm<8, VEC>(p, st);
  if (sk == 4) return launch_sgemm<4, VEC>(p, st);
  if (sk == 2) return launch_sgemm<2, VEC>(p, st);
  return launch_sgemm<1, VEC>(p, st);
}

template <int NTOK, int SK, bool ONE>
int launch_rows(const LoraParams& p, cudaStream_t st) {
  using C = RowsCfg<NTOK, SK>;
  const ck_lora_args& a = p.a;
  CUtensorMap tw, tx;
  if (!make_tmap_2d(&tw, a.w, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.K, a.N, a.ldw, 64, 128, 128) ||
      !make_tmap_2d(&tx, a.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.K, a.M, a.ldx, 64, NTOK, 128))
    return CK_ERR_INVALID_ARG;
  auto kern = lora_rows_kernel<NTOK, SK, ONE>;
  if (!smem_attr_ready(reinterpret_cast<const void*>(kern), C::SMEM)) return record_cuda_error();
  const int n_tiles = (int)((a.N + 127) / 128);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SK;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_tiles * ((a.M + NTOK - 1) / NTOK) * SK));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = (size_t)C::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return launch_cfg(cfg, kern, tw, tx, p, n_tiles);
}

template <int NTOK, bool ONE = false>
int launch_rows_k(const LoraParams& p, cudaStream_t st) {
  // K split until the tiles give every SM a CTA (or a CTA one K block)
  const int64_t units = (p.a.N + 127) / 128 * ((p.a.M + NTOK - 1) / NTOK);
  const int64_t kb = (p.a.K + 63) / 64;
  const int sms = num_sms() > 0 ? num_sms() : 148;
  int sk = 1;
  while (sk < 8 && units * sk < sms && kb >= 2 * sk) sk *= 2;
  if (sk == 8) return launch_rows<NTOK, 8, ONE>(p, st);
  if (sk == 4) return launch_rows<NTOK, 4, ONE>(p, st);
  if (sk == 2) return launch_rows<NTOK, 2, ONE>(p, st);
  return launch_rows<NTOK, 1, ONE>(p, st);
}

template <int RP, int SK>
int launch_tiles(const TileParams& t, int tiles, cudaStream_t st) {
  using C = TilesCfg<RP, SK>;
  const ck_lora_args& a = t.a;
  CUtensorMap tx, ta;
  // (without adapters no tile lists one, and no block reads this map)
  const bool any = a.n_adapters > 0;
  if (!make_tmap_2d(&tx, a.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.K, a.M, a.ldx, 64, 128, 128) ||
      !make_tmap_2d(&ta, any ? a.a : a.x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.K,
                    any ? (uint64_t)a.n_adapters * a.rank : (uint64_t)a.M, any ? a.K : a.ldx, 64, RP,
                    128))
    return CK_ERR_INVALID_ARG;
  auto kern = lora_tiles_kernel<RP, SK>;
  if (!smem_attr_ready(reinterpret_cast<const void*>(kern), C::SMEM)) return record_cuda_error();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SK;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  const int groups = (t.max_slots + C::SL - 1) / C::SL;
  cfg.gridDim = dim3((unsigned)((int64_t)tiles * groups * SK));
  cfg.blockDim = dim3(128);
  cfg.dynamicSmemBytes = (size_t)C::SMEM;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return launch_cfg(cfg, kern, tx, ta, t);
}

template <int RP>
int launch_tiles_k(const TileParams& t, int tiles, cudaStream_t st) {
  // K split while the SMs have room and every CTA keeps two K blocks
  const int64_t kb = (t.a.K + 63) / 64;
  const int sms = num_sms() > 0 ? num_sms() : 148;
  int sk = 1;
  while (sk < 8 && 2 * (int64_t)tiles * sk <= sms && kb >= 4 * sk) sk *= 2;
  if (sk == 8) return launch_tiles<RP, 8>(t, tiles, st);
  if (sk == 4) return launch_tiles<RP, 4>(t, tiles, st);
  if (sk == 2) return launch_tiles<RP, 2>(t, tiles, st);
  return launch_tiles<RP, 1>(t, tiles, st);
}

int copy_strided(const void* src, int64_t ld_src, void* dst, int64_t ld_dst, int64_t rows,
                 int64_t cols, cudaStream_t st) {
  int64_t blocks = (rows * cols + 1023) / 1024;
  const int64_t most = 16 * (int64_t)num_sms();
  if (blocks > most) blocks = most;
  return launch_pdl(lora_copy_kernel, dim3((unsigned)blocks), dim3(256), 0, st,
                    reinterpret_cast<const __nv_bfloat16*>(src), ld_src,
                    reinterpret_cast<__nv_bfloat16*>(dst), ld_dst, rows, cols);
}

int run_tiles(const LoraPlan& pl, uint8_t* ws, cudaStream_t st) {
  const ck_lora_args& a = pl.p.a;
  int rc;
  const void* b = a.b;
  if (pl.ld_b > 0 && a.n_adapters > 0) {
    b = ws + pl.off_b;
    rc = copy_strided(a.b, a.rank, ws + pl.off_b, pl.ld_b, a.n_adapters * a.N, a.rank, st);
    if (rc != CK_OK) return rc;
  }
  TileParams t;
  t.a = a;
  t.h = ws + pl.off_h;
  t.max_slots = pl.max_slots;
  t.tiles = pl.tiles;
  t.cnt = reinterpret_cast<int32_t*>(ws + pl.off_cnt);
  t.slots = reinterpret_cast<uint4*>(ws + pl.off_slots);
  rc = a.rank <= 16 ? launch_tiles_k<16>(t, pl.tiles, st)
       : a.rank <= 32 ? launch_tiles_k<32>(t, pl.tiles, st)
                      : launch_tiles_k<64>(t, pl.tiles, st);
  if (rc != CK_OK) return rc;
  GemmFusion fz;
  fz.lora_h = t.h;
  // without any adapter no slot is listed and no block reads b
  fz.lora_b = a.n_adapters > 0 ? b : a.w;
  fz.lora_n = a.n_adapters > 0 ? a.n_adapters : 1;
  fz.lora_b_ld = pl.ld_b > 0 ? pl.ld_b : a.rank;
  fz.lora_rank = a.rank;
  fz.lora_max = pl.max_slots;
  fz.lora_cnt = t.cnt;
  fz.lora_slots = t.slots;
  void* y = pl.ld_stage > 0 ? ws + pl.off_y : a.y;
  const int64_t ldy = pl.ld_stage > 0 ? pl.ld_stage : a.ldy;
  rc = gemm_tc(a.x, a.M, a.K, a.ldx, a.w, CK_BF16, CK_W_NK, a.N, a.ldw, nullptr,
               a.bias != nullptr ? CK_EPI_BIAS : CK_EPI_STORE, a.bias, 0, 0, y, ldy, st, &fz);
  if (rc != CK_OK || pl.ld_stage == 0) return rc;
  return copy_strided(y, ldy, a.y, a.ldy, a.M, a.N, st);
}

}  // namespace

int lora_linear(const ck_lora_args& a, void* ws, size_t ws_bytes, cudaStream_t st) {
  LoraPlan pl;
  int rc = make_plan(a, pl);
  if (rc != CK_OK) return rc;
  if (a.M == 0 || a.N == 0) return CK_OK;
  if (!a.x || !a.w || !a.y || !a.ids || (a.n_adapters > 0 && (!a.a || !a.b)))
    return CK_ERR_INVALID_ARG;
  if (pl.bytes > 0 && (ws == nullptr || ws_bytes < pl.bytes || !aligned16(ws))) return CK_ERR_WORKSPACE;
  if (pl.path == PATH_TILES) return run_tiles(pl, reinterpret_cast<uint8_t*>(ws), st);
  pl.p.h = reinterpret_cast<float*>(ws);
  if (pl.path == PATH_ROWS) {
    if (pl.one) return launch_rows_k<16, true>(pl.p, st);
    rc = shrink<__nv_bfloat16>(pl.p, 1, st);
    if (rc != CK_OK) return rc;
    if (a.M <= 16) return launch_rows_k<16>(pl.p, st);
    if (a.M <= 32) return launch_rows_k<32>(pl.p, st);
    return launch_rows_k<64>(pl.p, st);
  }
  if (pl.path == PATH_F32) {
    rc = shrink<float>(pl.p, 0, st);
    if (rc != CK_OK) return rc;
    const bool vec = a.K % 4 == 0 && a.ldx % 4 == 0 && a.ldw % 4 == 0 && aligned16(a.x) && aligned16(a.w);
    return vec ? run_f32<true>(pl.p, st) : run_f32<false>(pl.p, st);
  }
  rc = shrink<__nv_bfloat16>(pl.p, 0, st);
  if (rc != CK_OK) return rc;
  const int n_tiles = (int)((a.N + 63) / 64);
  const dim3 grid((unsigned)(((a.M + 63) / 64) * n_tiles));
  return launch_pdl(lora_simt_kernel, grid, dim3(256), 0, st, pl.p, n_tiles);
}

}  // namespace ck

extern "C" size_t ck_lora_workspace_bytes(const ck_lora_args* args) {
  ck::LoraPlan pl;
  return args != nullptr && ck::make_plan(*args, pl) == CK_OK ? pl.bytes : 0;
}

extern "C" int ck_lora_linear(const ck_lora_args* args, void* workspace, size_t workspace_bytes,
                              void* stream) {
  if (args == nullptr) return CK_ERR_INVALID_ARG;
  return ck::lora_linear(*args, workspace, workspace_bytes, reinterpret_cast<cudaStream_t>(stream));
}
