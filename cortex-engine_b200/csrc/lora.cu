// A projection shared by many requests, beside each request's own low-rank
// adapter:
//
//   y[m] = W x[m] + s_i B_i (A_i x[m]) (+ bias),   i = ids[m], none for ids[m] < 0
//
// x (M, K), W (N, K), A (n, rank, K), B (n, N, rank), y (M, N); fp32 sums, one
// rounding at the end. 2 M N K + 2 M rank (K + N) flop over each operand once:
// a few rows are bound by reading W, many rows by the product with it.
//
// shrink_kernel computes h[m] = s_i A_i x[m] (fp32, rank values a row); the
// product with W then adds B_i h[m] to its accumulator before it rounds.
#include "common.cuh"
#include "kernels.h"

namespace ck {

namespace {

struct LoraParams {
  ck_lora_args a;
  float* h;  // [M][rank]
};

__device__ __forceinline__ float tofl(float v) { return v; }
__device__ __forceinline__ float tofl(__nv_bfloat16 v) { return bf2f(v); }
template <typename T>
__device__ __forceinline__ T fromf(float v);
template <>
__device__ __forceinline__ float fromf<float>(float v) { return v; }
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
// together (a lane gives half of its sums away at each step).
template <typename T, int JB, bool VEC>
__global__ void __launch_bounds__(256) lora_shrink_kernel(const LoraParams p, int jblocks) {
  grid_dep_wait();
  grid_dep_launch();
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

// The product with W on the CUDA cores, for fp32 (which TF32 tensor-core
// products would not match) and for bf16 whose strides break the 16-byte
// rules: 64 x 64 tiles, 4 x 4 a thread, the next K slice in registers while
// this one is multiplied.
template <typename T>
__global__ void __launch_bounds__(256) lora_simt_kernel(const LoraParams p, int n_tiles) {
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

struct LoraPlan {
  LoraParams p;
  size_t bytes;
};

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

int make_plan(const ck_lora_args& a, LoraPlan& pl) {
  if (a.dtype != CK_F32 && a.dtype != CK_BF16) return CK_ERR_UNSUPPORTED;
  if (a.M < 0 || a.N < 0 || a.K <= 0 || a.rank < 1 || a.n_adapters < 0) return CK_ERR_INVALID_ARG;
  if (a.M > INT32_MAX || a.N > INT32_MAX || a.K > INT32_MAX) return CK_ERR_UNSUPPORTED;
  if (a.rank > 256) return CK_ERR_UNSUPPORTED;
  if (((a.M + 63) / 64) * ((a.N + 63) / 64) > INT32_MAX || (a.M * a.rank + 7) / 8 > INT32_MAX)
    return CK_ERR_UNSUPPORTED;
  pl.p.a = a;
  pl.bytes = (size_t)a.M * a.rank * 4;
  return CK_OK;
}

template <typename T>
int shrink(const LoraParams& p, cudaStream_t st) {
  const ck_lora_args& a = p.a;
  constexpr int E = 16 / sizeof(T);
  const bool vec = a.K % E == 0 && a.ldx % E == 0 && aligned16(a.x) && aligned16(a.a);
  // one rank a warp while that leaves SMs without work, else 8
  const bool wide = a.M * a.rank >= 8 * 16 * (int64_t)(num_sms() > 0 ? num_sms() : 148);
  const int jb = wide ? 8 : 1;
  const int jblocks = (a.rank + jb - 1) / jb;
  const dim3 grid((unsigned)((a.M * jblocks + 7) / 8));
  if (wide)
    return vec ? launch_pdl(lora_shrink_kernel<T, 8, true>, grid, dim3(256), 0, st, p, jblocks)
               : launch_pdl(lora_shrink_kernel<T, 8, false>, grid, dim3(256), 0, st, p, jblocks);
  return vec ? launch_pdl(lora_shrink_kernel<T, 1, true>, grid, dim3(256), 0, st, p, jblocks)
             : launch_pdl(lora_shrink_kernel<T, 1, false>, grid, dim3(256), 0, st, p, jblocks);
}

}  // namespace

int lora_linear(const ck_lora_args& a, void* ws, size_t ws_bytes, cudaStream_t st) {
  LoraPlan pl;
  int rc = make_plan(a, pl);
  if (rc != CK_OK) return rc;
  if (a.M == 0 || a.N == 0) return CK_OK;
  if (!a.x || !a.w || !a.y || !a.ids || (a.n_adapters > 0 && (!a.a || !a.b)))
    return CK_ERR_INVALID_ARG;
  if (ws == nullptr || ws_bytes < pl.bytes || !aligned16(ws)) return CK_ERR_WORKSPACE;
  pl.p.h = reinterpret_cast<float*>(ws);
  const bool bf = a.dtype == CK_BF16;
  rc = bf ? shrink<__nv_bfloat16>(pl.p, st) : shrink<float>(pl.p, st);
  if (rc != CK_OK) return rc;
  const int n_tiles = (int)((a.N + 63) / 64);
  const dim3 grid((unsigned)(((a.M + 63) / 64) * n_tiles));
  return bf ? launch_pdl(lora_simt_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, pl.p, n_tiles)
            : launch_pdl(lora_simt_kernel<float>, grid, dim3(256), 0, st, pl.p, n_tiles);
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
