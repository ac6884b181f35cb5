// Attention of one new token per sequence over a paged K|V pool.
//
//   o[b, h] = sum_{j < n_b} p_hj v_j,   p_h = softmax_j(scale q[b, h] . k_j)
//   w_out[b, j] = w_in[b, j] + sum_h p_hj          (optional: what eviction reads)
//
// A pool row holds one position: K of every K|V head, then V of every head
// (kv_proj's layout, the rows of StreamingKVCache). Position j of sequence b is
// row j % page_size of page page_table[b, j / page_size].
//
// The call reads every live row once and does 2 G flop per byte (bf16, G query
// heads to a K|V head), so HBM bounds it. The length is cut into chunks so
// that a few long sequences still fill the card: paged_*_kernel computes one
// (sequence, chunk, head unit) and leaves the running maximum m, the sum l and
// the unnormalised output; join_kernel puts the chunks together. With one
// chunk and no weights the first kernel writes the output and nothing else
// runs. The weights need the final m and l of every head, so the first kernel
// leaves the scores (4 B per head and position) for join_kernel, which sums
// each position's probabilities over the heads in head order: no atomics, one
// result for one input.
//
// All statistics are fp32 in the log2 domain (s log2(e), exp2).
#include <math_constants.h>

#include "common.cuh"
#include "kernels.h"

namespace ck {

namespace {

constexpr int kSub = 512;         // positions whose row offsets are staged at a time
constexpr int kMaxChunks = 1024;  // chunks per sequence (join_kernel's shared arrays)

struct PagedParams {
  ck_paged_attention_args a;
  int32_t G;         // query heads per K|V head
  int32_t units;     // head units per sequence (Hkv * groups of at most GT heads)
  int32_t chunk;     // positions per chunk
  int32_t n_chunks;  // chunks of the longest possible sequence
  int64_t cap;       // page_table_width * page_size
  float qk_scale;    // scale * log2(e)
  float2* part_ml;   // [B * H][n_chunks] (m, l); NULL: write the output here
  float* part_o;     // [B * H][n_chunks][Dh]
  float* scores;     // [B * H][cap] or NULL
};

// Live positions of sequence b; a length outside [0, cap] is recorded and clamped.
__device__ __forceinline__ int64_t live_rows(const PagedParams& p, int b, bool report) {
  int64_t n = p.a.lengths[b];
  if (n < 0 || n > p.cap) {
    if (report) set_status(CK_ERR_INDEX, b, (int)n);
    n = n < 0 ? 0 : p.cap;
  }
  return n;
}

// Element offsets of rows [j0, j0 + cnt) of sequence b into shared memory; -1
// for a page outside the pool (recorded; its rows count as absent).
__device__ __forceinline__ void stage_rows(const PagedParams& p, int b, int64_t j0, int cnt,
                                           int64_t* rows) {
  for (int i = threadIdx.x; i < cnt; i += blockDim.x) {
    const uint32_t j = (uint32_t)(j0 + i);
    const uint32_t slot = j / (uint32_t)p.a.page_size;
    const int32_t page = __ldg(p.a.page_table + (int64_t)b * p.a.page_table_ld + slot);
    int64_t off = -1;
    if (page >= 0 && page < p.a.num_pages)
      off = (int64_t)page * p.a.page_ld + (int64_t)(j - slot * (uint32_t)p.a.page_size) * p.a.row_ld;
    else
      set_status(CK_ERR_INDEX, b, page);
    rows[i] = off;
  }
}

template <typename T>
__device__ __forceinline__ void store_out(T* p, float v);
template <>
__device__ __forceinline__ void store_out<float>(float* p, float v) { *p = v; }
template <>
__device__ __forceinline__ void store_out<__nv_bfloat16>(__nv_bfloat16* p, float v) { *p = f2bf(v); }

// The (m, l, o) of NW warps over heads [h0, h0 + nh) put together and written:
// the output itself (one chunk) or this chunk's partials. sm_ml [NW][HT],
// sm_o [NW][HT][Dh]. A row without any key (l = 0) gives 0.
template <typename T, int NW>
__device__ __forceinline__ void finish_unit(const PagedParams& p, int b, int c, int h0, int nh,
                                            int HT, const float2* sm_ml, const float* sm_o) {
  const int Dh = p.a.Dh;
  for (int i = threadIdx.x; i < nh * Dh; i += blockDim.x) {
    const int h = i / Dh, d = i - h * Dh;
    float m = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, sm_ml[w * HT + h].x);
    const float ref = m == -CUDART_INF_F ? 0.f : m;
    float l = 0.f, o = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 ml = sm_ml[w * HT + h];
      const float f = exp2f(ml.x - ref);
      l += ml.y * f;
      o += sm_o[(w * HT + h) * Dh + d] * f;
    }
    if (p.part_ml == nullptr) {
      store_out<T>(reinterpret_cast<T*>(p.a.o) + (int64_t)b * p.a.o_ld_b +
                       (int64_t)(h0 + h) * p.a.o_ld_h + d,
                   l == 0.f ? 0.f : o / l);
    } else {
      const int64_t part = ((int64_t)b * p.a.H + h0 + h) * p.n_chunks + c;
      p.part_o[part * Dh + d] = o;
      if (d == 0) p.part_ml[part] = make_float2(m, l);
    }
  }
}

// ── bf16, head dims 32 / 64 / 128: matrix instructions fed from registers ────
//
// A warp takes 16 positions at a time as the M side of mma.m16n8k16, with the
// G <= 8 * NT query heads of the K|V head as the N side:
//   S^T[16 x 8] = K[16 x Dh] Q^T,  O^T[Dh x 8] += V^T[Dh x 16] P^T[16 x 8].
// The sums over Dh and over positions may be taken in any order as long as
// both operands agree, so every lane loads whole 16-byte pieces of K and V
// rows straight from HBM into the registers the instruction wants: no shared
// memory, no barrier in the loop. V's operand pairs neighbouring positions:
// two rows' words are interleaved by byte permutes. P goes from S^T's
// accumulator layout to the B operand by an 8 x 8 transpose (movmatrix),
// rounded to bf16 for the instruction; l sums the fp32 values.
// The next iteration's K loads are issued once S is done with the registers,
// the next V loads once O is, so each warp keeps its loads in flight through
// the arithmetic without a second set of registers.

__device__ __forceinline__ void mma16816(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint4 ldg_stream(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

__device__ __forceinline__ uint2 ldg_stream8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

template <int DH, int NT, int NW>
__global__ void __launch_bounds__(NW * 32) paged_tc_kernel(const PagedParams p) {
  constexpr int UT = DH == 128 ? 1 : 2;  // 16-position tiles per iteration
  constexpr int KC = DH / 32;            // 16-byte pieces of a K row per lane
  constexpr int MT = DH / 16;            // 16-wide pieces of Dh in O^T
  constexpr int VW = DH >= 64 ? 4 : 2;   // words of a V piece
  constexpr int VP = DH >= 64 ? DH / 64 : 1;  // V pieces per row per lane
  constexpr int HT = 8 * NT;
  constexpr int STEP = 16 * UT;
  extern __shared__ __align__(16) uint8_t smem[];
  int64_t* s_row = reinterpret_cast<int64_t*>(smem);  // [kSub]

  grid_dep_wait();
  grid_dep_launch();
  const int unit = blockIdx.x % p.units;
  const int bc = blockIdx.x / p.units;
  const int c = bc % p.n_chunks;
  const int b = bc / p.n_chunks;
  const int groups = p.units / p.a.Hkv;
  const int hk = unit / groups;
  const int g0 = (unit - hk * groups) * HT;  // first query head of the group
  const int nh = min(HT, p.G - g0);
  const int h0 = hk * p.G + g0;
  const int64_t n = live_rows(p, b, c == 0 && unit == 0 && threadIdx.x == 0);
  const int64_t c_begin = (int64_t)c * p.chunk;
  const int64_t c_end = min(n, c_begin + p.chunk);
  if (c_begin >= n && p.part_ml != nullptr) return;  // (one chunk: writes the zeros)

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const __nv_bfloat16* kbase =
      reinterpret_cast<const __nv_bfloat16*>(p.a.pool) + (int64_t)hk * DH + 8 * t;
  const __nv_bfloat16* vbase = reinterpret_cast<const __nv_bfloat16*>(p.a.pool) +
                               (int64_t)(p.a.Hkv + hk) * DH + 2 * VW * g;

  // query operand: lane (g, t) holds head g's pieces t, t + 4, ...
  uint4 q[NT][KC];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + g;
#pragma unroll
    for (int i = 0; i < KC; ++i)
      q[nt][i] = h < nh ? __ldg(reinterpret_cast<const uint4*>(
                              reinterpret_cast<const __nv_bfloat16*>(p.a.q) +
                              (int64_t)b * p.a.q_ld_b + (int64_t)(h0 + h) * p.a.q_ld_h + 8 * t +
                              32 * i))
                        : make_uint4(0u, 0u, 0u, 0u);
  }

  float o[NT][MT][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt][0] = m[nt][1] = -CUDART_INF_F;
    l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
  }

  for (int64_t sub = c_begin; sub < c_end; sub += kSub) {
    const int cnt = (int)min((int64_t)kSub, c_end - sub);
    if (sub != c_begin) __syncthreads();
    stage_rows(p, b, sub, cnt, s_row);
    __syncthreads();

    uint4 kr[UT][2][KC];
    uint32_t vr[UT][4][VP][VW];
    auto load_k = [&](int j0) {
#pragma unroll
      for (int u = 0; u < UT; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int j = j0 + 16 * u + 8 * r + g;
          const int64_t off = j < cnt ? s_row[j] : -1;
#pragma unroll
          for (int i = 0; i < KC; ++i)
            kr[u][r][i] = off >= 0 ? ldg_stream(kbase + off + 32 * i) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    auto load_v = [&](int j0) {
#pragma unroll
      for (int u = 0; u < UT; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = j0 + 16 * u + 2 * t + (r & 1) + 8 * (r >> 1);
          const int64_t off = j < cnt ? s_row[j] : -1;
#pragma unroll
          for (int i = 0; i < VP; ++i) {
            if constexpr (VW == 4) {
              const uint4 v = off >= 0 ? ldg_stream(vbase + off + 64 * i) : make_uint4(0u, 0u, 0u, 0u);
              vr[u][r][i][0] = v.x;
              vr[u][r][i][1] = v.y;
              vr[u][r][i][2] = v.z;
              vr[u][r][i][3] = v.w;
            } else {
              const uint2 v = off >= 0 ? ldg_stream8(vbase + off) : make_uint2(0u, 0u);
              vr[u][r][i][0] = v.x;
              vr[u][r][i][1] = v.y;
            }
          }
        }
    };
    int j0 = warp * STEP;
    if (j0 < cnt) {
      load_k(j0);
      load_v(j0);
    }
    for (; j0 < cnt; j0 += NW * STEP) {
      const int jn = j0 + NW * STEP;
      float s[UT][NT][4];
#pragma unroll
      for (int u = 0; u < UT; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
#pragma unroll
          for (int i = 0; i < KC; ++i) {
            mma16816(s[u][nt], kr[u][0][i].x, kr[u][1][i].x, kr[u][0][i].y, kr[u][1][i].y,
                     q[nt][i].x, q[nt][i].y);
            mma16816(s[u][nt], kr[u][0][i].z, kr[u][1][i].z, kr[u][0][i].w, kr[u][1][i].w,
                     q[nt][i].z, q[nt][i].w);
          }
        }
      // absent rows get -inf whatever the arithmetic above made of them
#pragma unroll
      for (int u = 0; u < UT; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int j = j0 + 16 * u + 8 * r + g;
          const bool live = j < cnt && s_row[j] >= 0;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float v = live ? s[u][nt][2 * r + e] * p.qk_scale : -CUDART_INF_F;
              s[u][nt][2 * r + e] = v;
              const int h = nt * 8 + 2 * t + e;
              if (p.scores != nullptr && h < nh && j < cnt)
                p.scores[((int64_t)b * p.a.H + h0 + h) * p.cap + sub + j] = v;
            }
        }
      if (jn < cnt) load_k(jn);
      // running maximum over the positions (lanes g), rescale, probabilities
      uint32_t pb[UT][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = m[nt][e];
#pragma unroll
          for (int u = 0; u < UT; ++u) mx = fmaxf(mx, fmaxf(s[u][nt][e], s[u][nt][2 + e]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float ref = mx == -CUDART_INF_F ? 0.f : mx;
          f[e] = exp2f(m[nt][e] - ref);
          m[nt][e] = mx;
          l[nt][e] *= f[e];
#pragma unroll
          for (int u = 0; u < UT; ++u) {
            s[u][nt][e] = exp2f(s[u][nt][e] - ref);
            s[u][nt][2 + e] = exp2f(s[u][nt][2 + e] - ref);
            l[nt][e] += s[u][nt][e] + s[u][nt][2 + e];
          }
        }
#pragma unroll
        for (int u = 0; u < UT; ++u) {
          pb[u][nt][0] = transpose8x8(cvt_bf16x2(s[u][nt][0], s[u][nt][1]));
          pb[u][nt][1] = transpose8x8(cvt_bf16x2(s[u][nt][2], s[u][nt][3]));
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[nt][i][e] *= f[e & 1];
      }
#pragma unroll
      for (int u = 0; u < UT; ++u)
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int pc = i / VW, w = i - pc * VW;
          const uint32_t a0 = prmt(vr[u][0][pc][w], vr[u][1][pc][w], 0x5410u);
          const uint32_t a1 = prmt(vr[u][0][pc][w], vr[u][1][pc][w], 0x7632u);
          const uint32_t a2 = prmt(vr[u][2][pc][w], vr[u][3][pc][w], 0x5410u);
          const uint32_t a3 = prmt(vr[u][2][pc][w], vr[u][3][pc][w], 0x7632u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][i], a0, a1, a2, a3, pb[u][nt][0], pb[u][nt][1]);
        }
      if (jn < cnt) load_v(jn);
    }
  }

  // lane (g, t): O^T of heads 2t, 2t + 1 at Dh indices 2 VW (g + 8 pc) + 2 w (+ 1)
  float2* sm_ml = reinterpret_cast<float2*>(smem + kSub * 8);       // [NW][HT]
  float* sm_o = reinterpret_cast<float*>(sm_ml + NW * HT);          // [NW][HT][DH]
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float ls = l[nt][e];
      ls += __shfl_xor_sync(0xffffffffu, ls, 4);
      ls += __shfl_xor_sync(0xffffffffu, ls, 8);
      ls += __shfl_xor_sync(0xffffffffu, ls, 16);
      const int h = nt * 8 + 2 * t + e;
      if (g == 0) sm_ml[warp * HT + h] = make_float2(m[nt][e], ls);
      float* dst = sm_o + (warp * HT + h) * DH;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int pc = i / VW, w = i - pc * VW;
        const int d = 2 * VW * (g + 8 * pc) + 2 * w;
        *reinterpret_cast<float2*>(dst + d) = make_float2(o[nt][i][e], o[nt][i][2 + e]);
      }
    }
  __syncthreads();
  finish_unit<__nv_bfloat16, NW>(p, b, c, h0, nh, HT, sm_ml, sm_o);
}

// ── fp32, and bf16 layouts the matrix kernel does not take ───────────────────
//
// A warp takes 8 rows at a time, a row's Dh elements spread over its lanes
// (VEC contiguous ones per lane, NV times). The 8 dot products are reduced
// together: at each of the first three butterfly steps a lane gives half of
// its sums away and keeps the other half, so 9 shuffles serve 8 rows instead
// of 40, and lane L ends with the score of row L / 4. The exponentials are then
// one per lane for all 8 rows.

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  if constexpr (sizeof(T) == 4 && VEC == 4) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else if constexpr (sizeof(T) == 4 && VEC == 2) {
    const float2 v = __ldg(reinterpret_cast<const float2*>(p));
    f[0] = v.x; f[1] = v.y;
  } else if constexpr (sizeof(T) == 2 && VEC == 4) {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
    f[0] = bf16_lo(v.x); f[1] = bf16_hi(v.x);
    f[2] = bf16_lo(v.y); f[3] = bf16_hi(v.y);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = (float)p[i];
  }
}

template <typename T, int VEC, int NV, int GT, int NW>
__global__ void __launch_bounds__(NW * 32) paged_simt_kernel(const PagedParams p) {
  constexpr int E = VEC * NV;
  extern __shared__ __align__(16) uint8_t smem[];
  int64_t* s_row = reinterpret_cast<int64_t*>(smem);  // [kSub]

  grid_dep_wait();
  grid_dep_launch();
  const int Dh = p.a.Dh;
  const int unit = blockIdx.x % p.units;
  const int bc = blockIdx.x / p.units;
  const int c = bc % p.n_chunks;
  const int b = bc / p.n_chunks;
  const int groups = p.units / p.a.Hkv;
  const int hk = unit / groups;
  const int g0 = (unit - hk * groups) * GT;
  const int nh = min(GT, p.G - g0);
  const int h0 = hk * p.G + g0;
  const int64_t n = live_rows(p, b, c == 0 && unit == 0 && threadIdx.x == 0);
  const int64_t c_begin = (int64_t)c * p.chunk;
  const int64_t c_end = min(n, c_begin + p.chunk);
  if (c_begin >= n && p.part_ml != nullptr) return;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* kbase = reinterpret_cast<const T*>(p.a.pool) + (int64_t)hk * Dh;
  const T* vbase = reinterpret_cast<const T*>(p.a.pool) + (int64_t)(p.a.Hkv + hk) * Dh;
  float q[GT][E], o[GT][E], m[GT], l[GT];
#pragma unroll
  for (int h = 0; h < GT; ++h) {
    m[h] = -CUDART_INF_F;
    l[h] = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int d = (i / VEC) * 32 * VEC + lane * VEC + i % VEC;
      o[h][i] = 0.f;
      q[h][i] = (h < nh && d < Dh)
                    ? (float)reinterpret_cast<const T*>(p.a.q)[(int64_t)b * p.a.q_ld_b +
                                                              (int64_t)(h0 + h) * p.a.q_ld_h + d]
                    : 0.f;
    }
  }

  for (int64_t sub = c_begin; sub < c_end; sub += kSub) {
    const int cnt = (int)min((int64_t)kSub, c_end - sub);
    if (sub != c_begin) __syncthreads();
    stage_rows(p, b, sub, cnt, s_row);
    __syncthreads();
    for (int j0 = warp * 8; j0 < cnt; j0 += NW * 8) {
      float k[8][E], v[8][E];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int64_t off = j0 + r < cnt ? s_row[j0 + r] : -1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int d = i * 32 * VEC + lane * VEC;
          if (off >= 0 && d < Dh) {  // (Dh is a multiple of VEC)
            load_vec<T, VEC>(kbase + off + d, &k[r][i * VEC]);
            load_vec<T, VEC>(vbase + off + d, &v[r][i * VEC]);
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) k[r][i * VEC + e] = v[r][i * VEC + e] = 0.f;
          }
        }
      }
      const int jr = j0 + (lane >> 2);  // the row whose score this lane ends with
      const bool live = jr < cnt && s_row[jr] >= 0;
#pragma unroll
      for (int h = 0; h < GT; ++h) {
        float a[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          a[r] = 0.f;
#pragma unroll
          for (int i = 0; i < E; ++i) a[r] = fmaf(q[h][i], k[r][i], a[r]);
        }
        // lane bits 4, 3, 2 choose row bits 2, 1, 0
#pragma unroll
        for (int w = 4, bit = 16; w > 0; w >>= 1, bit >>= 1) {
          const bool up = (lane & bit) != 0;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            if (r < w) {
              const float give = up ? a[r] : a[r + w];
              const float keep = up ? a[r + w] : a[r];
              a[r] = keep + __shfl_xor_sync(0xffffffffu, give, bit);
            }
          }
        }
        float s = a[0];
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s = live ? s * p.qk_scale : -CUDART_INF_F;
        if (p.scores != nullptr && h < nh && (lane & 3) == 0 && jr < cnt)
          p.scores[((int64_t)b * p.a.H + h0 + h) * p.cap + sub + jr] = s;
        float mx = fmaxf(m[h], s);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float ref = mx == -CUDART_INF_F ? 0.f : mx;
        const float f = exp2f(m[h] - ref);
        m[h] = mx;
        const float pr = exp2f(s - ref);
        l[h] = l[h] * f + pr;  // this lane's row (four lanes hold the same sum)
#pragma unroll
        for (int i = 0; i < E; ++i) o[h][i] *= f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
          const float w = __shfl_sync(0xffffffffu, pr, r * 4);
#pragma unroll
          for (int i = 0; i < E; ++i) o[h][i] = fmaf(w, v[r][i], o[h][i]);
        }
      }
    }
  }

  float2* sm_ml = reinterpret_cast<float2*>(smem + kSub * 8);  // [NW][GT]
  float* sm_o = reinterpret_cast<float*>(sm_ml + NW * GT);     // [NW][GT][Dh]
#pragma unroll
  for (int h = 0; h < GT; ++h) {
    float ls = l[h];
    ls += __shfl_xor_sync(0xffffffffu, ls, 4);
    ls += __shfl_xor_sync(0xffffffffu, ls, 8);
    ls += __shfl_xor_sync(0xffffffffu, ls, 16);
    if (lane == 0) sm_ml[warp * GT + h] = make_float2(m[h], ls);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int d = (i / VEC) * 32 * VEC + lane * VEC + i % VEC;
      if (d < Dh) sm_o[(warp * GT + h) * Dh + d] = o[h][i];
    }
  }
  __syncthreads();
  finish_unit<T, NW>(p, b, c, h0, nh, GT, sm_ml, sm_o);
}

// ── chunks put together; weights ─────────────────────────────────────────────
//
// Blocks [0, out_blocks) write one (b, h) output each (when there are
// partials); the rest write the weights of 256 positions of one sequence each.

constexpr int JT = 256;

template <typename T>
__global__ void __launch_bounds__(JT) join_kernel(const PagedParams p, int out_blocks,
                                                  int w_blocks) {
  __shared__ float s_f[kMaxChunks];
  __shared__ float s_red[JT];
  __shared__ float s_l;
  extern __shared__ __align__(16) float2 s_ml[];  // weights: [H] (m, 1 / l)
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x < out_blocks) {
    const int b = blockIdx.x / p.a.H, h = blockIdx.x - b * p.a.H;
    const int Dh = p.a.Dh;
    const int64_t n = live_rows(p, b, false);
    const int nc = (int)((n + p.chunk - 1) / p.chunk);
    const int64_t part = (int64_t)blockIdx.x * p.n_chunks;
    if (warp == 0) {
      float m = -CUDART_INF_F;
      for (int i = lane; i < nc; i += 32) m = fmaxf(m, p.part_ml[part + i].x);
      m = warp_max(m);
      const float ref = m == -CUDART_INF_F ? 0.f : m;
      float l = 0.f;
      for (int i = lane; i < nc; i += 32) {
        const float2 ml = p.part_ml[part + i];
        const float f = exp2f(ml.x - ref);
        s_f[i] = f;
        l += ml.y * f;
      }
      l = warp_sum(l);
      if (lane == 0) s_l = l;
    }
    __syncthreads();
    const float inv = s_l == 0.f ? 0.f : 1.f / s_l;
    // ways threads share a column of the output, each every ways-th chunk
    const int ways = JT / Dh > 0 ? JT / Dh : 1;
    const int way = tid / Dh, d = tid - way * Dh;
    float acc = 0.f;
    if (way < ways)
      for (int i = way; i < nc; i += ways) acc += s_f[i] * p.part_o[(part + i) * Dh + d];
    s_red[tid] = acc;
    __syncthreads();
    if (tid < Dh) {
      for (int w = 1; w < ways; ++w) acc += s_red[w * Dh + tid];
      store_out<T>(reinterpret_cast<T*>(p.a.o) + (int64_t)b * p.a.o_ld_b +
                       (int64_t)h * p.a.o_ld_h + tid,
                   nc == 0 || s_l == 0.f ? 0.f : acc * inv);
    }
    return;
  }
  const int wb = blockIdx.x - out_blocks;
  const int b = wb / w_blocks;
  const int64_t j = (int64_t)(wb - b * w_blocks) * JT + tid;
  const int64_t n = live_rows(p, b, false);
  const float* w_in = p.a.w_in + (int64_t)b * p.a.w_in_ld;
  float* w_out = p.a.w_out + (int64_t)b * p.a.w_out_ld;
  if ((int64_t)(wb - b * w_blocks) * JT < n) {
    // a warp per head: the chunks' (m, l) to the head's
    const int nc = (int)((n + p.chunk - 1) / p.chunk);
    for (int h = warp; h < p.a.H; h += JT / 32) {
      const int64_t part = ((int64_t)b * p.a.H + h) * p.n_chunks;
      float m = -CUDART_INF_F;
      for (int i = lane; i < nc; i += 32) m = fmaxf(m, p.part_ml[part + i].x);
      m = warp_max(m);
      const float ref = m == -CUDART_INF_F ? 0.f : m;
      float l = 0.f;
      for (int i = lane; i < nc; i += 32) {
        const float2 ml = p.part_ml[part + i];
        l += ml.y * exp2f(ml.x - ref);
      }
      l = warp_sum(l);
      if (lane == 0) s_ml[h] = make_float2(ref, l == 0.f ? 0.f : 1.f / l);
    }
    __syncthreads();
  }
  if (j >= p.a.w_width) return;
  if (j < n) {
    float w = 0.f;
    const float* sc = p.scores + (int64_t)b * p.a.H * p.cap + j;
#pragma unroll 4
    for (int h = 0; h < p.a.H; ++h) w += exp2f(sc[(int64_t)h * p.cap] - s_ml[h].x) * s_ml[h].y;
    w_out[j] = w_in[j] + w;
  } else if (w_out != w_in) {
    w_out[j] = w_in[j];
  }
}

// ── host ─────────────────────────────────────────────────────────────────────

struct Plan {
  PagedParams p;
  int path;  // 0: matrix kernel, 1: CUDA-core kernel
  int gt;    // heads per unit
  int vec, nv;
  bool partials;
  int64_t w_blocks;
  size_t off_ml, off_o, off_s, bytes;
};

constexpr int NWARP = 4;

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

int make_plan(const ck_paged_attention_args& a, Plan& pl) {
  if (a.dtype != CK_F32 && a.dtype != CK_BF16) return CK_ERR_UNSUPPORTED;
  if (a.B < 0 || a.H <= 0 || a.Hkv <= 0 || a.H % a.Hkv != 0 || a.Dh <= 0 || a.num_pages < 0 ||
      a.page_size <= 0 || a.page_table_width < 0)
    return CK_ERR_INVALID_ARG;
  if (a.Dh > 256 || a.H > 4096) return CK_ERR_UNSUPPORTED;
  if (!(a.scale == a.scale)) return CK_ERR_INVALID_ARG;
  PagedParams& p = pl.p;
  p.a = a;
  p.G = a.H / a.Hkv;
  p.cap = (int64_t)a.page_table_width * a.page_size;
  if (p.cap > INT32_MAX) return CK_ERR_INVALID_ARG;
  if (a.w_out != nullptr && (a.w_in == nullptr || a.w_width < p.cap)) return CK_ERR_INVALID_ARG;
  p.qk_scale = a.scale * 1.4426950408889634f;
  const bool vec16 = aligned16(a.pool) && aligned16(a.q) && (a.page_ld * 2) % 16 == 0 &&
                     (a.row_ld * 2) % 16 == 0 && (a.q_ld_b * 2) % 16 == 0 &&
                     (a.q_ld_h * 2) % 16 == 0;
  pl.path = (a.dtype == CK_BF16 && (a.Dh == 32 || a.Dh == 64 || a.Dh == 128) && vec16) ? 0 : 1;
  if (pl.path == 0) {
    pl.gt = p.G <= 8 ? 8 : 16;
  } else {
    pl.gt = p.G == 1 ? 1 : 4;
    const bool v4 = aligned16(a.pool) && a.page_ld % 4 == 0 && a.row_ld % 4 == 0 && a.Dh % 4 == 0;
    pl.vec = v4 && a.Dh > 32 ? (a.dtype == CK_F32 && a.Dh <= 64 ? 2 : 4) : 1;
    pl.nv = a.Dh <= 32 * pl.vec ? 1 : (pl.vec == 4 ? 2 : 8);
  }
  p.units = a.Hkv * ((p.G + pl.gt - 1) / pl.gt);
  // Chunks: enough blocks for several rounds over the SMs, at least 64
  // positions each.
  const int64_t want = 8 * (int64_t)(num_sms() > 0 ? num_sms() : 148);
  const int64_t seqs = (int64_t)(a.B > 0 ? a.B : 1) * p.units;
  int64_t chunk = (p.cap * seqs + want - 1) / want;
  chunk = (chunk + 63) / 64 * 64;
  if (chunk < 64) chunk = 64;
  if (chunk > 1024) chunk = 1024;
  if (chunk < (p.cap + kMaxChunks - 1) / kMaxChunks) chunk = (p.cap + kMaxChunks - 1) / kMaxChunks;
  p.chunk = (int32_t)chunk;
  p.n_chunks = (int32_t)((p.cap + chunk - 1) / chunk);
  if (p.n_chunks < 1) p.n_chunks = 1;
  pl.w_blocks = a.w_out != nullptr ? (a.w_width + JT - 1) / JT : 0;
  if ((int64_t)a.B * p.n_chunks * p.units > INT32_MAX ||
      (int64_t)a.B * (a.H + pl.w_blocks) > INT32_MAX)
    return CK_ERR_UNSUPPORTED;
  pl.partials = p.n_chunks > 1 || a.w_out != nullptr;
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  const size_t heads = (size_t)(a.B > 0 ? a.B : 0) * a.H;
  pl.off_ml = 0;
  pl.off_o = up(pl.partials ? heads * p.n_chunks * 8 : 0);
  pl.off_s = pl.off_o + up(pl.partials ? heads * p.n_chunks * (size_t)a.Dh * 4 : 0);
  pl.bytes = pl.off_s + up(a.w_out != nullptr ? heads * (size_t)p.cap * 4 : 0);
  return CK_OK;
}

template <int DH, int NT>
int launch_tc(const PagedParams& p, cudaStream_t st) {
  constexpr int smem = kSub * 8 + NWARP * 8 * NT * 8 + NWARP * 8 * NT * DH * 4;
  auto kern = paged_tc_kernel<DH, NT, NWARP>;
  if (!smem_attr_ready(reinterpret_cast<const void*>(kern), smem)) return record_cuda_error();
  return launch_pdl(kern, dim3((unsigned)(p.a.B * p.n_chunks * p.units)), dim3(NWARP * 32), smem, st, p);
}

template <typename T, int VEC, int NV>
int launch_simt(const PagedParams& p, int gt, cudaStream_t st) {
  const int smem = kSub * 8 + NWARP * gt * 8 + NWARP * gt * p.a.Dh * 4;
  const dim3 grid((unsigned)(p.a.B * p.n_chunks * p.units));
  if (gt == 1) return launch_pdl(paged_simt_kernel<T, VEC, NV, 1, NWARP>, grid, dim3(NWARP * 32), smem, st, p);
  return launch_pdl(paged_simt_kernel<T, VEC, NV, 4, NWARP>, grid, dim3(NWARP * 32), smem, st, p);
}

}  // namespace

size_t paged_attention_workspace_bytes(const ck_paged_attention_args& a) {
  Plan pl;
  return make_plan(a, pl) == CK_OK ? pl.bytes : 0;
}

int paged_attention(const ck_paged_attention_args& a, void* ws, size_t ws_bytes, cudaStream_t st) {
  Plan pl;
  int rc = make_plan(a, pl);
  if (rc != CK_OK) return rc;
  if (a.B == 0) return CK_OK;
  PagedParams& p = pl.p;
  if (!a.q || !a.o || !a.lengths) return CK_ERR_INVALID_ARG;
  if (p.cap > 0 && ((a.num_pages > 0 && !a.pool) || !a.page_table)) return CK_ERR_INVALID_ARG;
  if (pl.bytes > 0 && (ws == nullptr || ws_bytes < pl.bytes || !aligned16(ws)))
    return CK_ERR_WORKSPACE;
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  p.part_ml = pl.partials ? reinterpret_cast<float2*>(w + pl.off_ml) : nullptr;
  p.part_o = pl.partials ? reinterpret_cast<float*>(w + pl.off_o) : nullptr;
  p.scores = a.w_out != nullptr ? reinterpret_cast<float*>(w + pl.off_s) : nullptr;
  if (pl.path == 0) {
    const int nt = pl.gt / 8;
    if (a.Dh == 32) rc = nt == 1 ? launch_tc<32, 1>(p, st) : launch_tc<32, 2>(p, st);
    if (a.Dh == 64) rc = nt == 1 ? launch_tc<64, 1>(p, st) : launch_tc<64, 2>(p, st);
    if (a.Dh == 128) rc = nt == 1 ? launch_tc<128, 1>(p, st) : launch_tc<128, 2>(p, st);
  } else if (a.dtype == CK_BF16) {
    if (pl.vec == 4)
      rc = pl.nv == 1 ? launch_simt<__nv_bfloat16, 4, 1>(p, pl.gt, st)
                      : launch_simt<__nv_bfloat16, 4, 2>(p, pl.gt, st);
    else
      rc = pl.nv == 1 ? launch_simt<__nv_bfloat16, 1, 1>(p, pl.gt, st)
                      : launch_simt<__nv_bfloat16, 1, 8>(p, pl.gt, st);
  } else if (pl.vec == 4) {
    rc = pl.nv == 1 ? launch_simt<float, 4, 1>(p, pl.gt, st) : launch_simt<float, 4, 2>(p, pl.gt, st);
  } else if (pl.vec == 2) {
    rc = launch_simt<float, 2, 1>(p, pl.gt, st);
  } else {
    rc = pl.nv == 1 ? launch_simt<float, 1, 1>(p, pl.gt, st) : launch_simt<float, 1, 8>(p, pl.gt, st);
  }
  if (rc != CK_OK || !pl.partials) return rc;
  const int out_blocks = a.B * a.H;
  const int64_t w_blocks = pl.w_blocks;
  const int64_t blocks = out_blocks + (int64_t)a.B * w_blocks;
  const size_t smem = a.w_out != nullptr ? (size_t)a.H * 8 : 0;
  if (a.dtype == CK_BF16)
    return launch_pdl(join_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(JT), smem, st, p,
                      out_blocks, (int)w_blocks);
  return launch_pdl(join_kernel<float>, dim3((unsigned)blocks), dim3(JT), smem, st, p, out_blocks,
                    (int)w_blocks);
}

}  // namespace ck

extern "C" size_t ck_paged_attention_workspace_bytes(const ck_paged_attention_args* args) {
  return args == nullptr ? 0 : ck::paged_attention_workspace_bytes(*args);
}

extern "C" int ck_paged_attention(const ck_paged_attention_args* args, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (args == nullptr) return CK_ERR_INVALID_ARG;
  return ck::paged_attention(*args, workspace, workspace_bytes,
                             reinterpret_cast<cudaStream_t>(stream));
}
