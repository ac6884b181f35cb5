// Attention of one new token per sequence over a paged K|V pool.
//
//   o[b, h] = sum_{j < n_b} p_hj v_j,   p_h = softmax_j(scale q[b, h] . k_j)
//   w_out[b, j] = w_in[b, j] + sum_h p_hj          (optional: what eviction reads)
//
// A pool row holds one position: K of every K|V head, then V of every head
// (kv_proj's layout, the rows of StreamingKVCache). Position j of sequence b is
// row j % page_size of page page_table[b, j / page_size].
//
// The call does 2 G flop per byte (bf16, G query heads to a K|V head), so HBM bounds
// it. Every live row is read once where the G query heads make one unit (up to 16 in
// bf16, 4 in fp32), else once a unit, side by side and so mostly from L2 (16 sequences
// of 3000 to 16384 positions, fp32, 32 heads over 4 of 64: 111 us for 258 MB). The positions of all sequences make one
// list of tiles of 16 or 32, cut into equal runs however ragged the lengths are;
// a warp takes one run for one unit (the query heads of one K|V head, at most GT
// of them), the warps of one run side by side, so that the pieces of a row are
// read at about the same time. A warp streams the rows of its tiles through its
// own ring in shared memory by 16-byte asynchronous copies, ST - 1 tiles ahead
// and straight across the ends of sequences, and waits for nobody: after the
// split of the list there is no barrier. Where a run begins or ends inside a
// sequence the warp leaves the running maximum m, the sum l and the unnormalised
// output, and join_kernel puts the parts together; a sequence inside one run is
// written at once.
//
// The weights need the final m and l of every head, so the scores are left for
// join_kernel (4 B per head and position), which sums each position's
// probabilities over the heads in head order. No atomics: one result for one
// input.
//
// All statistics are fp32 in the log2 domain (s log2(e), 2^x).
//
// Measured (captured, a call): 16 sequences of 3000 to 32768 positions, 32 heads over 8 of
// 128, 840 MB, 138 us (6.1 TB/s); 32 sequences of 32 to 4096, 12 heads of 64, 86 MB, with
// weights 30 us (2.9 TB/s), without 27; 300 positions, 8 heads of 64, 4.3 us. Short rows
// are bound by their instructions too: more than 500 a tile of 8 KB, and with one query
// head to a K|V head six of the eight columns of every product and softmax are empty.
#include <math_constants.h>

#include "common.cuh"
#include "kernels.h"

namespace ck {

namespace {

constexpr int kSub = 512;          // generic kernel: positions staged at a time
constexpr int kMaxParts = 2048;    // parts of a unit (join_kernel's shared array)

struct PagedParams {
  ck_paged_attention_args a;
  int32_t G;         // query heads per K|V head
  int32_t gt;        // query heads per unit, at most
  int32_t units;     // units per sequence (Hkv * groups of at most gt heads)
  int32_t chunk;     // generic kernel: positions per block
  int32_t n_chunks;  // generic kernel: blocks of the longest possible sequence
  int64_t cap;       // page_table_width * page_size
  float qk_scale;    // scale * log2(e)
  uint32_t page_mul, page_shift;  // j / page_size = (umulhi(page_mul, j) + j) >> page_shift
  int2* seg;         // [B * units] (first part, parts); NULL: one part, written at once
  int32_t part_step; // from one part of a (sequence, unit) to its next
  int32_t runs;      // runs of the list, at most
  float2* part_ml;   // [part][gt] (m, l)
  float* part_o;     // [part][gt][Dh]
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

// j / page_size for 0 <= j < 2^31 (exact: multiplication by the rounded-up
// reciprocal, Granlund and Montgomery 1994)
__device__ __forceinline__ uint32_t page_of(const PagedParams& p, uint32_t j) {
  return (__umulhi(p.page_mul, j) + j) >> p.page_shift;
}

// Element offset of row `in_page` of a page of sequence b; -1 for a page
// outside the pool (recorded; its rows count as absent).
__device__ __forceinline__ int64_t row_offset(const PagedParams& p, int b, int32_t page,
                                              uint32_t in_page) {
  if (page >= 0 && page < p.a.num_pages)
    return (int64_t)page * p.a.page_ld + (int64_t)in_page * p.a.row_ld;
  set_status(CK_ERR_INDEX, b, page);
  return -1;
}

// 2^x; results below the smallest normal number are 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void store_out(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_out(__nv_bfloat16* p, float v) { *p = f2bf(v); }

template <typename T>
__device__ __forceinline__ T* out_row(const PagedParams& p, int b, int h) {
  return reinterpret_cast<T*>(p.a.o) + (int64_t)b * p.a.o_ld_b + (int64_t)h * p.a.o_ld_h;
}

// The (m, l, o) of NW warps over heads [h0, h0 + nh) put together and written:
// the output (part < 0), else this part. sm_ml [NW][HT], sm_o [NW][HT][Dh]. A
// row without any key (l = 0) gives 0.
template <typename T, int NW>
__device__ __forceinline__ void finish_unit(const PagedParams& p, int b, int64_t part, int h0,
                                            int nh, int HT, const float2* sm_ml,
                                            const float* sm_o) {
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
      const float f = ex2(ml.x - ref);
      l += ml.y * f;
      o += sm_o[(w * HT + h) * Dh + d] * f;
    }
    if (part < 0) {
      store_out(out_row<T>(p, b, h0 + h) + d, l == 0.f ? 0.f : o / l);
    } else {
      p.part_o[(part * p.gt + h) * Dh + d] = o;
      if (d == 0) p.part_ml[part * p.gt + h] = make_float2(m, l);
    }
  }
}

// ── tiles through a warp's ring ──────────────────────────────────────────────

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

template <bool TRANS>
__device__ __forceinline__ uint4 ldmatrix4(uint32_t addr) {
  uint4 v;
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
  return v;
}

// 16 bytes global -> shared; the second form writes zeros, and reads nothing, when !live
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(live ? 16 : 0)
               : "memory");
}

// Shape of a ring: rows of DH elements of T, TP positions to a K (or V) tile,
// ST tiles. off() is the byte offset of 16-byte piece c of row r; pieces are
// permuted within a row so that neither the copies nor the reads below meet in
// a bank. Rows of at most 128 bytes go 32 to a tile: with 16 the instructions
// of a tile, not its bytes, set the pace. Three tiles in a ring and two blocks
// an SM beat two and three (the same shared memory, fewer bytes in flight): 157
// against 196 us at 16 sequences of 3000 to 32768 positions, 8 K|V heads of 128.
template <typename T, int DH>
struct Ring {
  static constexpr int ROW = DH * (int)sizeof(T);
  static constexpr int PC = ROW / 16;
  static constexpr int TP = ROW <= 128 ? 32 : 16;
  static constexpr int TILE = TP * ROW;
  static constexpr int ST = ROW == 64 ? 4 : 3;
  static constexpr int BYTES = ST * 2 * TILE;
  __device__ static __forceinline__ uint32_t off(int r, int c) {
    if (sizeof(T) == 4) return (uint32_t)(r * ROW + ((c ^ ((r & 3) << 1)) << 4));
    if (ROW == 64) return (uint32_t)(r * ROW + ((c ^ ((r >> 1) & 3)) << 4));
    return (uint32_t)(r * ROW + ((c ^ (r & 7)) << 4));
  }
};

// The running state of up to GT query heads over the tiles of a unit.
template <typename T, int DH, int GT>
struct Heads;

// bf16: 16 positions at a time are the M side of mma.m16n8k16, the heads (8 NT) its
// N side: S^T[16 x 8] = K[16 x Dh] Q^T, O^T[Dh x 8] += V^T[Dh x 16] P^T[16 x 8].
// P goes from S^T's accumulator layout to the B operand by an 8 x 8 transpose
// (movmatrix) as the sum of two bf16 numbers of the same sign, so that an infinite value
// stays one, the second what the first lost: one
// alone leaves an error of 2^-8 sum p |v|, as large as the result's own rounding
// (captured, us, with and without the second: 8 sequences of 8000 to 32000 positions, 12
// heads of 64, 78.5 / 79.0; 32 of 32 to 4096 with weights 29.8 / 29.6; one of 1000, 8 heads
// of 64, 7.0 / 6.7; 16 of 3000 to 32768, 32 heads over 2 of 128, 60.3 / 57.5). l sums the
// fp32 values.
// Up to four heads stand in the eight columns twice, so that one product takes both
// parts, columns 0-3 the first ones, columns 4-7 the second (two products: 30.05 for the
// 29.8 above).
template <int DH, int GT>
struct Heads<__nv_bfloat16, DH, GT> {
  using R = Ring<__nv_bfloat16, DH>;
  static constexpr bool TWICE = GT == 4;
  static constexpr int NT = TWICE ? 1 : GT / 8;
  static constexpr int KS = DH / 16;
  static constexpr int Q_FLOATS = 0;
  uint32_t q[NT][KS][2];
  float o[NT][KS][4];
  float m[NT][2], l[NT][2];

  __device__ __forceinline__ void begin(const PagedParams& p, int b, int h0, int nh, float*) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // lane (g, t) holds head g's elements 2t, 2t + 1 of every 8
      const int h = TWICE ? g & 3 : nt * 8 + g;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(
          reinterpret_cast<const __nv_bfloat16*>(p.a.q) + (int64_t)b * p.a.q_ld_b +
          (int64_t)(h0 + h) * p.a.q_ld_h + 2 * t);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        q[nt][i][0] = h < nh ? __ldg(src + 8 * i) : 0u;
        q[nt][i][1] = h < nh ? __ldg(src + 8 * i + 4) : 0u;
      }
      m[nt][0] = m[nt][1] = -CUDART_INF_F;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][i][e] = 0.f;
    }
  }

  // One tile: positions j0.. of sequence b, those present in `live`; `sc` the
  // scores of the unit's first head (or NULL), of positions below n.
  __device__ __forceinline__ void tile(const PagedParams& p, uint32_t kt, uint32_t live, int j0,
                                       int n, int nh, float* sc, const float*) {
    constexpr int U = R::TP / 16;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t vt = kt + R::TILE;
    float s[U][NT][4];
    // matrices: rows 0-7 | 8-15 of piece 2i, then of piece 2i + 1
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint4 a = ldmatrix4<false>(kt + R::off(16 * u + (lane & 15), 2 * i + (lane >> 4)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816(s[u][nt], a.x, a.y, a.z, a.w, q[nt][i][0], q[nt][i][1]);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][nt][e] *= p.qk_scale;
    if (live != (R::TP == 32 ? 0xffffffffu : 0xffffu)) {
      // absent rows get -inf whatever the arithmetic above made of them
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (!((live >> (16 * u + 8 * r + g)) & 1u)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[u][nt][2 * r] = s[u][nt][2 * r + 1] = -CUDART_INF_F;
          }
    }
    if (sc != nullptr) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (nt * 8 + 2 * t + e < nh) {
            float* dst = sc + (int64_t)(nt * 8 + 2 * t + e) * p.cap + j0 + g;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (j0 + 16 * u + 8 * r + g < n) dst[16 * u + 8 * r] = s[u][nt][2 * r + e];
          }
    }
    // running maximum over the positions (lanes g), rescale, probabilities
    uint32_t ph[U][NT][2], pl[U][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = m[nt][e];
#pragma unroll
        for (int u = 0; u < U; ++u) mx[e] = fmaxf(mx[e], fmaxf(s[u][nt][e], s[u][nt][2 + e]));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 4));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 8));
        mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 16));
      }
      // (the sums stay as they are when no head has a new maximum)
      if (__any_sync(0xffffffffu, mx[0] != m[nt][0] || mx[1] != m[nt][1])) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = ex2(m[nt][e] - (mx[e] == -CUDART_INF_F ? 0.f : mx[e]));
          m[nt][e] = mx[e];
          l[nt][e] *= f;
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            o[nt][i][e] *= f;
            o[nt][i][2 + e] *= f;
          }
        }
      }
      const float ref0 = mx[0] == -CUDART_INF_F ? 0.f : mx[0];
      const float ref1 = mx[1] == -CUDART_INF_F ? 0.f : mx[1];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p0 = ex2(s[u][nt][0] - ref0), p1 = ex2(s[u][nt][1] - ref1);
        const float p2 = ex2(s[u][nt][2] - ref0), p3 = ex2(s[u][nt][3] - ref1);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        uint32_t high[2], low[2];
        two_bf16x2(p0, p1, high[0], low[0]);
        two_bf16x2(p2, p3, high[1], low[1]);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          if (TWICE) {
            ph[u][nt][r] = transpose8x8(t < 2 ? high[r] : low[r]);
          } else {
            ph[u][nt][r] = transpose8x8(high[r]);
            pl[u][nt][r] = transpose8x8(low[r]);
          }
        }
      }
    }
    // V^T tiles: matrices of positions 0-7 in pieces 2i, 2i + 1, then 8-15
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const uint4 a = ldmatrix4<true>(
            vt + R::off(16 * u + (lane & 7) + ((lane >> 4) << 3), 2 * i + ((lane >> 3) & 1)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816(o[nt][i], a.x, a.y, a.z, a.w, ph[u][nt][0], ph[u][nt][1]);
          if (!TWICE) mma16816(o[nt][i], a.x, a.y, a.z, a.w, pl[u][nt][0], pl[u][nt][1]);
        }
      }
  }

  __device__ __forceinline__ void total(int nt, int e, float& ls) const {
    ls = l[nt][e];
    ls += __shfl_xor_sync(0xffffffffu, ls, 4);
    ls += __shfl_xor_sync(0xffffffffu, ls, 8);
    ls += __shfl_xor_sync(0xffffffffu, ls, 16);
  }

  // put(h, d, value) for this lane's outputs and put_ml(h, m, l) once a head
  template <typename Put, typename PutMl>
  __device__ __forceinline__ void emit(int nh, bool normalise, Put put, PutMl put_ml) const {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float ls;
        total(nt, e, ls);
        const int h = nt * 8 + 2 * t + e;
        float sum[KS][2];  // both parts
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            sum[i][r] = o[nt][i][2 * r + e];
            if (TWICE) sum[i][r] += __shfl_xor_sync(0xffffffffu, sum[i][r], 2);
          }
        if (h < nh) {
          if (g == 0) put_ml(h, m[nt][e], ls);
          const float f = !normalise ? 1.f : (ls == 0.f ? 0.f : 1.f / ls);
#pragma unroll
          for (int i = 0; i < KS; ++i) {
            put(h, 16 * i + g, f == 0.f && normalise ? 0.f : sum[i][0] * f);
            put(h, 16 * i + g + 8, f == 0.f && normalise ? 0.f : sum[i][1] * f);
          }
        }
      }
  }
};

// fp32 on the CUDA cores: lanes 2r, 2r + 1 take the two interleaved halves of
// row r's pieces for its scores, then every lane DH / 32 columns of V for all 16
// rows. The queries of the unit lie in the warp's shared memory.
template <int DH, int GT>
struct Heads<float, DH, GT> {
  using R = Ring<float, DH>;
  static constexpr int VE = DH / 32;
  static constexpr int Q_FLOATS = GT * DH;
  float o[GT][VE];
  float m[GT], l[GT];

  __device__ __forceinline__ void begin(const PagedParams& p, int b, int h0, int nh, float* sq) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    const float* src = reinterpret_cast<const float*>(p.a.q) + (int64_t)b * p.a.q_ld_b;
    for (int i = lane; i < GT * DH; i += 32)
      sq[i] = i / DH < nh ? __ldg(src + (int64_t)(h0 + i / DH) * p.a.q_ld_h + i % DH) : 0.f;
    __syncwarp();
#pragma unroll
    for (int h = 0; h < GT; ++h) {
      m[h] = -CUDART_INF_F;
      l[h] = 0.f;
#pragma unroll
      for (int e = 0; e < VE; ++e) o[h][e] = 0.f;
    }
  }

  __device__ __forceinline__ void tile(const PagedParams& p, uint32_t kt, uint32_t live, int j0,
                                       int n, int nh, float* sc, const float* sq) {
#pragma unroll 1
    for (int u = 0; u < R::TP / 16; ++u)
      rows16(p, kt + u * 16 * R::ROW, (live >> (16 * u)) & 0xffffu, j0 + 16 * u, n, nh, sc, sq);
  }

  __device__ __forceinline__ void rows16(const PagedParams& p, uint32_t kt, uint32_t live, int j0,
                                         int n, int nh, float* sc, const float* sq) {
    const int lane = threadIdx.x & 31, r = lane >> 1, half = lane & 1;
    const uint32_t vt = kt + R::TILE;
    float s[GT];
#pragma unroll
    for (int h = 0; h < GT; ++h) s[h] = 0.f;
#pragma unroll
    for (int i = 0; i < R::PC / 2; ++i) {
      const uint4 k = lds128(kt + R::off(r, 2 * i + half));
#pragma unroll
      for (int h = 0; h < GT; ++h) {
        const float4 qv = *reinterpret_cast<const float4*>(sq + h * DH + 4 * (2 * i + half));
        s[h] = fmaf(__uint_as_float(k.x), qv.x, s[h]);
        s[h] = fmaf(__uint_as_float(k.y), qv.y, s[h]);
        s[h] = fmaf(__uint_as_float(k.z), qv.z, s[h]);
        s[h] = fmaf(__uint_as_float(k.w), qv.w, s[h]);
      }
    }
    const bool here = (live >> r) & 1u;
#pragma unroll
    for (int h = 0; h < GT; ++h) {
      s[h] += __shfl_xor_sync(0xffffffffu, s[h], 1);
      s[h] = here ? s[h] * p.qk_scale : -CUDART_INF_F;
      if (sc != nullptr && half == 0 && h < nh && j0 + r < n) sc[(int64_t)h * p.cap + j0 + r] = s[h];
      float mx = fmaxf(m[h], s[h]);
#pragma unroll
      for (int k = 2; k < 32; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
      const float ref = mx == -CUDART_INF_F ? 0.f : mx;
      const float f = ex2(m[h] - ref);
      m[h] = mx;
      s[h] = ex2(s[h] - ref);
      l[h] = l[h] * f + s[h];
#pragma unroll
      for (int e = 0; e < VE; ++e) o[h][e] *= f;
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float v[VE];
      const uint32_t at = vt + R::off(k, lane * VE / 4) + (lane * VE % 4) * 4;
      if constexpr (VE == 4) {
        const uint4 u = lds128(at);
        v[0] = __uint_as_float(u.x); v[1] = __uint_as_float(u.y);
        v[2] = __uint_as_float(u.z); v[3] = __uint_as_float(u.w);
      } else if constexpr (VE == 2) {
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(at) : "memory");
      } else {
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v[0]) : "r"(at) : "memory");
      }
#pragma unroll
      for (int h = 0; h < GT; ++h) {
        const float w = __shfl_sync(0xffffffffu, s[h], 2 * k);
#pragma unroll
        for (int e = 0; e < VE; ++e) o[h][e] = fmaf(w, v[e], o[h][e]);
      }
    }
  }

  template <typename Put, typename PutMl>
  __device__ __forceinline__ void emit(int nh, bool normalise, Put put, PutMl put_ml) const {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int h = 0; h < GT; ++h) {
      float ls = l[h];
#pragma unroll
      for (int k = 2; k < 32; k <<= 1) ls += __shfl_xor_sync(0xffffffffu, ls, k);
      if (h < nh) {
        if (lane == 0) put_ml(h, m[h], ls);
        const float f = !normalise ? 1.f : (ls == 0.f ? 0.f : 1.f / ls);
#pragma unroll
        for (int e = 0; e < VE; ++e)
          put(h, lane * VE + e, f == 0.f && normalise ? 0.f : o[h][e] * f);
      }
    }
  }
};

// A place in the list of tiles, and the unit it is read for.
struct Cursor {
  int b, unit;
  int tile, tiles;  // within the sequence
  int64_t n;        // live positions of b
  int64_t left;     // tiles to the end of the run
};

// DIRECT: a block per unit, its warps share the unit's tiles and put the result
// together in shared memory (short tables: one launch, no parts). Otherwise a
// warp per run of the list.
template <typename T, int DH, int GT, int NW, bool DIRECT>
__global__ void __launch_bounds__(NW * 32) paged_stream_kernel(const PagedParams p) {
  using R = Ring<T, DH>;
  using H = Heads<T, DH, GT>;
  constexpr int ST = R::ST, RS = R::ST + 1;
  constexpr int LANES = R::PC < 32 ? R::PC : 32;  // lanes that copy one row
  constexpr int RPI = 32 / LANES;                 // rows per copy instruction
  constexpr int TP = R::TP;
  constexpr int CPY = TP / RPI;
  constexpr uint32_t FULL = TP == 32 ? 0xffffffffu : 0xffffu;
  static_assert(R::PC <= 32, "a row is copied by one warp instruction at most");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t s_off[NW][RS][TP];  // byte offsets of a tile's rows (0: absent)
  __shared__ uint32_t s_live[NW][RS];    // which are present
  __shared__ int64_t s_sum[NW];

  grid_dep_wait();
  grid_dep_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int groups = p.units / p.a.Hkv;
  const int worker = blockIdx.x * NW + warp;
  auto tiles_of = [](int64_t n) { return (int)((n + TP - 1) / TP); };

  Cursor at;
  // warps side by side on one run: one per unit, or all of them in turns
  const int unit_step = min(p.units, (int)gridDim.x * NW);
  int64_t first = 0, span = 1, run_tiles = 0;  // this warp's run in the list, tiles per run
  int64_t count;                               // tiles of this warp
  int run = 0;
  if constexpr (DIRECT) {
    at.b = blockIdx.x / p.units;
    at.unit = blockIdx.x - at.b * p.units;
    at.n = live_rows(p, at.b, at.unit == 0 && tid == 0);
    at.tiles = tiles_of(at.n);
    at.tile = warp;
    count = at.tiles > warp ? (at.tiles - warp + NW - 1) / NW : 0;
    at.left = 0;
  } else {
    // length of the list, then the sequence in which this warp's run begins
    int64_t mine = 0;
    for (int b = tid; b < p.a.B; b += NW * 32) mine += tiles_of(live_rows(p, b, blockIdx.x == 0));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) total += s_sum[w];
    span = (total + p.runs - 1) / p.runs;
    if (span < 1) span = 1;
    run = worker / unit_step;
    first = run * span;
    run_tiles = min(span, total - first);
    at.unit = worker - run * unit_step;
    if (run_tiles <= 0 || at.unit >= p.units) return;  // (no barrier below)
    count = run_tiles * ((p.units - at.unit + unit_step - 1) / unit_step);
    int64_t before = 0;
    int b = 0;
    for (int b0 = 0; b0 < p.a.B; b0 += 32) {
      const int t = b0 + lane < p.a.B ? tiles_of(live_rows(p, b0 + lane, false)) : 0;
      int64_t sum = t;  // inclusive sums over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + sum > first);
      if (past != 0u) {
        const int k = __ffs(past) - 1;
        b = b0 + k;
        before += __shfl_sync(0xffffffffu, sum - t, k);
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
    at.b = b;
    at.n = live_rows(p, b, false);
    at.tiles = tiles_of(at.n);
    at.tile = (int)(first - before);
    at.left = run_tiles;
  }
  const Cursor start = at;
  auto advance = [&](Cursor& c) {
    if constexpr (DIRECT) {
      c.tile += NW;
    } else if (--c.left == 0) {  // the run again for this warp's next unit, if it has one
      const int unit = c.unit + unit_step;
      c = start;
      c.unit = unit;
    } else if (++c.tile == c.tiles) {
      c.tile = 0;
      do {
        ++c.b;
        c.n = c.b < p.a.B ? live_rows(p, c.b, false) : 0;
      } while (c.n == 0 && c.b < p.a.B);
      c.tiles = tiles_of(c.n);
    }
  };

  uint8_t* ring_p = smem + warp * (R::BYTES + H::Q_FLOATS * 4);
  const uint32_t ring = smem_u32(ring_p);
  float* sq = reinterpret_cast<float*>(ring_p + R::BYTES);
  int64_t(*off)[TP] = s_off[warp];
  uint32_t* live = s_live[warp];
  const int cr = lane / LANES, cc = lane % LANES;
  const uint8_t* base = reinterpret_cast<const uint8_t*>(p.a.pool) + cc * 16;
  const int64_t v_bytes = (int64_t)p.a.Hkv * DH * sizeof(T);

  // Row `lane` of a tile in two steps, so that the page table's latency runs
  // under the tile between them: its page and row, then the byte offset of its
  // K (of the unit's head), -1 when absent.
  struct Found {
    int32_t page;
    uint32_t in_page;
    int b, unit;  // b < 0: absent
  };
  auto find = [&](const Cursor& c) -> Found {
    Found f = {0, 0u, -1, c.unit};
    const int64_t j = (int64_t)c.tile * TP + lane;
    if (lane < TP && j < c.n) {
      const uint32_t slot = page_of(p, (uint32_t)j);
      f.page = __ldg(p.a.page_table + (int64_t)c.b * p.a.page_table_ld + slot);
      f.in_page = (uint32_t)j - slot * (uint32_t)p.a.page_size;
      f.b = c.b;
    }
    return f;
  };
  auto locate = [&](const Found& f) -> int64_t {
    if (f.b < 0) return -1;
    const int64_t o = row_offset(p, f.b, f.page, f.in_page);
    return o < 0 ? -1 : (o + (int64_t)(f.unit / groups) * DH) * (int64_t)sizeof(T);
  };
  auto put_row = [&](int slot, int64_t o) {
    const uint32_t here = __ballot_sync(0xffffffffu, o >= 0);
    if (lane < TP) off[slot][lane] = o >= 0 ? o : 0;
    if (lane == 0) live[slot] = here;
  };
  // tile k of this warp into ring stage `stage`, its rows in off[slot]
  auto copy_tile = [&](int64_t k, int stage, int slot) {
    if (k < count) {
      const uint32_t kd = ring + (uint32_t)stage * 2 * R::TILE;
      const int64_t* o = off[slot] + cr;
      const uint32_t here = live[slot];
      if (here == FULL) {
#pragma unroll
        for (int i = 0; i < CPY; ++i) {
          const uint8_t* src = base + o[i * RPI];
          copy16(kd + R::off(cr + i * RPI, cc), src);
          copy16(kd + R::TILE + R::off(cr + i * RPI, cc), src + v_bytes);
        }
      } else {
#pragma unroll
        for (int i = 0; i < CPY; ++i) {
          const int r = cr + i * RPI;
          const bool in = (here >> r) & 1u;
          const uint8_t* src = base + o[i * RPI];
          copy16(kd + R::off(r, cc), src, in);
          copy16(kd + R::TILE + R::off(r, cc), in ? src + v_bytes : src, in);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  Cursor ahead = at;  // the tile whose rows are located next
  {
    Found f[ST];
#pragma unroll
    for (int k = 0; k < ST; ++k) {
      f[k].b = -1;
      if (k < count) {
        f[k] = find(ahead);
        advance(ahead);
      }
    }
#pragma unroll
    for (int k = 0; k < ST; ++k) {
      put_row(k, locate(f[k]));
    }
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < ST - 1; ++k) copy_tile(k, k, k);

  H st;
  int h0 = 0, nh = 0;
  float* sc = nullptr;
  int part_first = 0;  // tile of the unit at which this warp entered it
  bool enter = true;
  // k modulo ST and RS, and those of the tiles being copied and located
  int stage = 0, stage_copy = ST - 1, slot = 0, slot_copy = ST - 1, slot_next = ST;
  auto step = [](int& i, int n) { i = i + 1 == n ? 0 : i + 1; };
  for (int64_t k = 0; k < count; ++k) {
    if (enter) {
      const int hk = at.unit / groups, g0 = (at.unit - hk * groups) * GT;
      h0 = hk * p.G + g0;
      nh = min(GT, p.G - g0);
      st.begin(p, at.b, h0, nh, sq);
      sc = p.scores != nullptr ? p.scores + ((int64_t)at.b * p.a.H + h0) * p.cap : nullptr;
      part_first = at.tile;
      enter = false;
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
    __syncwarp();  // every lane's part of the tile is there, and all have left the one before
    copy_tile(k + ST - 1, stage_copy, slot_copy);
    Found next = {0, 0u, -1, 0};
    if (k + ST < count) {
      next = find(ahead);
      advance(ahead);
    }
    st.tile(p, ring + (uint32_t)stage * 2 * R::TILE, live[slot], at.tile * TP, (int)at.n, nh, sc, sq);
    put_row(slot_next, locate(next));  // (the slot of tile k - 1)
    step(stage, ST);
    step(stage_copy, ST);
    step(slot, RS);
    step(slot_copy, RS);
    step(slot_next, RS);
    if constexpr (!DIRECT) {
      if (at.tile + 1 == at.tiles || at.left == 1) {
        const int64_t u = (int64_t)at.b * p.units + at.unit;
        const int64_t part = u + (int64_t)run * p.units;
        const bool whole = part_first == 0 && at.tile + 1 == at.tiles;
        if (part_first == 0 && lane == 0) {
          // runs that this sequence, whose first tile is here, reaches into
          const int64_t u0 = first + run_tiles - at.left - at.tile;
          p.seg[u] = make_int2((int)part, (int)((u0 + at.tiles - 1) / span - run + 1));
        }
        auto put_ml = [&](int h, float m, float l) { p.part_ml[part * GT + h] = make_float2(m, l); };
        if (whole) {
          st.emit(nh, true, [&](int h, int d, float v) { store_out(out_row<T>(p, at.b, h0 + h) + d, v); },
                  put_ml);
        } else {
          st.emit(nh, false, [&](int h, int d, float v) { p.part_o[(part * GT + h) * DH + d] = v; },
                  put_ml);
        }
        enter = true;
      }
    }
    advance(at);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if constexpr (DIRECT) {
    if (count == 0) {
      const int hk = at.unit / groups, g0 = (at.unit - hk * groups) * GT;
      h0 = hk * p.G + g0;
      nh = min(GT, p.G - g0);
      st.begin(p, at.b, h0, nh, sq);
    }
    __syncthreads();  // every warp has left its ring
    float2* sm_ml = reinterpret_cast<float2*>(smem);          // [NW][GT]
    float* sm_o = reinterpret_cast<float*>(sm_ml + NW * GT);  // [NW][GT][DH]
    st.emit(nh, false, [&](int h, int d, float v) { sm_o[(warp * GT + h) * DH + d] = v; },
            [&](int h, float m, float l) { sm_ml[warp * GT + h] = make_float2(m, l); });
    __syncthreads();
    finish_unit<T, NW>(p, at.b, -1, h0, nh, GT, sm_ml, sm_o);
  }
}

// ── layouts the ring does not take (head dims other than 32, 64, 128, rows
// that are not 16-byte aligned) ─────────────────────────────────────────────
//
// A block takes one chunk of one unit.
// A warp takes 8 rows at a time, a row's Dh elements spread over its lanes
// (VEC contiguous ones per lane, NV times). The 8 dot products are reduced
// together: at each of the first three butterfly steps a lane gives half of
// its sums away and keeps the other half, so 9 shuffles serve 8 rows instead
// of 40, and lane L ends with the score of row L / 4. The exponentials are then
// one per lane for all 8 rows. Bound by its instructions: 16 sequences of 3000 to
// 32768 positions, 32 heads over 8 of 96, 965 us, a tenth of the copy rate: rows of
// 192 bytes that are aligned could go through a ring as well.

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
  extern __shared__ __align__(128) uint8_t smem[];
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
  const int64_t part = p.seg == nullptr ? -1 : ((int64_t)b * p.units + unit) * p.n_chunks + c;
  if (c_begin >= n && part >= 0) return;
  if (c == 0 && part >= 0 && threadIdx.x == 0)
    p.seg[(int64_t)b * p.units + unit] = make_int2((int)part, (int)((n + p.chunk - 1) / p.chunk));

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
    for (int i = threadIdx.x; i < cnt; i += NW * 32) {
      const uint32_t j = (uint32_t)(sub + i), slot = page_of(p, j);
      s_row[i] = row_offset(p, b, __ldg(p.a.page_table + (int64_t)b * p.a.page_table_ld + slot),
                            j - slot * (uint32_t)p.a.page_size);
    }
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
        const float f = ex2(m[h] - ref);
        m[h] = mx;
        const float pr = ex2(s - ref);
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
  finish_unit<T, NW>(p, b, part, h0, nh, GT, sm_ml, sm_o);
}

// ── parts put together; weights ─────────────────────────────────────────────
//
// Blocks [0, out_blocks) write one (b, h) output each; the rest write the
// weights of 256 positions of one sequence each. Bound by loads that depend on one
// another, so six blocks share an SM (40 registers): 10.9 us against 14.6 with two
// (32 sequences of 32 to 4096, 12 heads).

constexpr int JT = 256;

// (b, h)'s unit and its place among the unit's heads
__device__ __forceinline__ int2 unit_of(const PagedParams& p, int h) {
  const int groups = p.units / p.a.Hkv;
  const int hk = h / p.G, g = h - hk * p.G;
  return make_int2(hk * groups + g / p.gt, g % p.gt);
}

template <typename T>
__global__ void __launch_bounds__(JT, 6) join_kernel(const PagedParams p, int out_blocks,
                                                  int w_blocks, int chunked) {
  __shared__ float s_f[kMaxParts];
  __shared__ float s_red[JT];
  __shared__ float s_l;
  extern __shared__ __align__(16) float2 s_ml[];  // weights: [H] (m, 1 / l)
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if ((int)blockIdx.x < out_blocks) {
    const int b = blockIdx.x / p.a.H, h = blockIdx.x - b * p.a.H;
    const int Dh = p.a.Dh;
    T* out = out_row<T>(p, b, h);
    if (live_rows(p, b, false) == 0) {
      if (tid < Dh) store_out(out + tid, 0.f);
      return;
    }
    const int2 u = unit_of(p, h);
    const int2 seg = p.seg[(int64_t)b * p.units + u.x];
    if (seg.y == 1 && !chunked) return;  // written at once
    const int64_t step = (int64_t)p.part_step * p.gt;
    const float2* ml = p.part_ml + (int64_t)seg.x * p.gt + u.y;
    const float* po = p.part_o + ((int64_t)seg.x * p.gt + u.y) * Dh;
    if (warp == 0) {
      float m = -CUDART_INF_F;
      for (int i = lane; i < seg.y; i += 32) m = fmaxf(m, ml[i * step].x);
      m = warp_max(m);
      const float ref = m == -CUDART_INF_F ? 0.f : m;
      float l = 0.f;
      for (int i = lane; i < seg.y; i += 32) {
        const float2 v = ml[i * step];
        const float f = ex2(v.x - ref);
        s_f[i] = f;
        l += v.y * f;
      }
      l = warp_sum(l);
      if (lane == 0) s_l = l;
    }
    __syncthreads();
    const float inv = s_l == 0.f ? 0.f : 1.f / s_l;
    // ways threads share a column of the output, each every ways-th part
    const int ways = JT / Dh > 0 ? JT / Dh : 1;
    const int way = tid / Dh, d = tid - way * Dh;
    float acc = 0.f;
    if (way < ways)
      for (int i = way; i < seg.y; i += ways) acc += s_f[i] * po[i * step * Dh + d];
    s_red[tid] = acc;
    __syncthreads();
    if (tid < Dh) {
      for (int w = 1; w < ways; ++w) acc += s_red[w * Dh + tid];
      store_out(out + tid, s_l == 0.f ? 0.f : acc * inv);
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
    // a warp per head: the parts' (m, l) to the head's
    for (int h = warp; h < p.a.H; h += JT / 32) {
      const int2 u = unit_of(p, h);
      const int2 seg = p.seg[(int64_t)b * p.units + u.x];
      const int64_t step = (int64_t)p.part_step * p.gt;
      const float2* ml = p.part_ml + (int64_t)seg.x * p.gt + u.y;
      float m = -CUDART_INF_F;
      for (int i = lane; i < seg.y; i += 32) m = fmaxf(m, ml[i * step].x);
      m = warp_max(m);
      const float ref = m == -CUDART_INF_F ? 0.f : m;
      float l = 0.f;
      for (int i = lane; i < seg.y; i += 32) {
        const float2 v = ml[i * step];
        l += v.y * ex2(v.x - ref);
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
    for (int h = 0; h < p.a.H; ++h) w += ex2(sc[(int64_t)h * p.cap] - s_ml[h].x) * s_ml[h].y;
    w_out[j] = w_in[j] + w;
  } else if (w_out != w_in) {
    w_out[j] = w_in[j];
  }
}

// ── host ─────────────────────────────────────────────────────────────────────

struct Plan {
  PagedParams p;
  bool ring;      // rows go through the ring, else the generic kernel
  bool parts;     // more than one part per unit is possible (or weights): join runs
  int vec, nv;    // generic kernel
  int64_t w_blocks, n_parts;
  size_t off_ml, off_o, off_s, bytes;
};

constexpr int NWARP = 4;        // warps of a streaming block
constexpr int NWARP_DIRECT = 8; // warps that share a unit (4 with rows of 512 bytes)

bool aligned16(const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

// Streaming blocks: what shared memory holds of NWARP rings on every SM.
int stream_blocks(int row_bytes) {
  const int sms = num_sms() > 0 ? num_sms() : 148;
  const int blocks = sms * (row_bytes >= 512 ? 1 : 2 + (row_bytes == 64));
  return blocks < kMaxParts / NWARP ? blocks : kMaxParts / NWARP;
}

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
  if (p.cap > INT32_MAX - 64) return CK_ERR_INVALID_ARG;  // (positions of a tile stay int32)
  if (a.w_out != nullptr && (a.w_in == nullptr || a.w_width < p.cap)) return CK_ERR_INVALID_ARG;
  p.qk_scale = a.scale * 1.4426950408889634f;
  p.page_shift = 0;
  while (((int64_t)1 << p.page_shift) < a.page_size) ++p.page_shift;
  p.page_mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << p.page_shift) - a.page_size)) /
                              (uint64_t)a.page_size + 1);
  const int64_t es = a.dtype == CK_F32 ? 4 : 2;
  pl.ring = (a.Dh == 32 || a.Dh == 64 || a.Dh == 128) && aligned16(a.pool) && aligned16(a.q) &&
            (a.page_ld * es) % 16 == 0 && (a.row_ld * es) % 16 == 0 && (a.q_ld_b * es) % 16 == 0 &&
            (a.q_ld_h * es) % 16 == 0;
  if (pl.ring && a.dtype == CK_BF16) {
    p.gt = p.G <= 4 ? 4 : (p.G <= 8 ? 8 : 16);
  } else {
    p.gt = p.G == 1 ? 1 : 4;
    const bool v4 = aligned16(a.pool) && a.page_ld % 4 == 0 && a.row_ld % 4 == 0 && a.Dh % 4 == 0;
    pl.vec = v4 && a.Dh > 32 ? (a.dtype == CK_F32 && a.Dh <= 64 ? 2 : 4) : 1;
    pl.nv = a.Dh <= 32 * pl.vec ? 1 : (pl.vec == 4 ? 2 : 8);
  }
  p.units = a.Hkv * ((p.G + p.gt - 1) / p.gt);
  const int sms = num_sms() > 0 ? num_sms() : 148;
  const int64_t seqs = (int64_t)(a.B > 0 ? a.B : 0) * p.units;
  p.chunk = 0;
  p.n_chunks = 1;
  if (pl.ring) {
    // One block a unit and no parts (one launch) for short tables, as long as
    // every block finds an SM: against runs and a join, us a call (captured), 8 heads
    // of 64 in bf16 4.3 / 7.6 at 300 positions, 7.1 / 7.8 at 1024, 11.7 / 9.8 at 2048;
    // 4 heads of 64 in fp32 5.3 / 7.4 at 300, 11.1 / 8.9 at 1000.
    pl.parts = a.w_out != nullptr || p.cap > 1024 || p.cap * a.Dh * es > 128 * 1024 || seqs > sms;
    const int workers = stream_blocks(a.Dh * (int)es) * NWARP;
    p.runs = workers / (p.units < workers ? p.units : workers);
    p.part_step = p.units;
    pl.n_parts = seqs + (int64_t)p.runs * p.units;
  } else {
    // enough blocks for several rounds over the SMs, at least 64 positions each
    int64_t chunk = (p.cap * seqs + 8 * sms - 1) / (8 * sms);
    chunk = (chunk + 63) / 64 * 64;
    if (chunk < 64) chunk = 64;
    if (chunk > 1024) chunk = 1024;
    if (chunk < (p.cap + 1023) / 1024) chunk = (p.cap + 1023) / 1024;
    p.chunk = (int32_t)chunk;
    p.n_chunks = p.cap > chunk ? (int32_t)((p.cap + chunk - 1) / chunk) : 1;
    pl.parts = p.n_chunks > 1 || a.w_out != nullptr;
    pl.n_parts = seqs * p.n_chunks;
    p.part_step = 1;
    p.runs = 0;
  }
  pl.w_blocks = a.w_out != nullptr ? (a.w_width + JT - 1) / JT : 0;
  if (pl.n_parts > INT32_MAX || (int64_t)a.B * (a.H + pl.w_blocks) > INT32_MAX)
    return CK_ERR_UNSUPPORTED;
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  const size_t np = pl.parts ? (size_t)pl.n_parts * p.gt : 0;
  pl.off_ml = up(pl.parts ? (size_t)seqs * 8 : 0);
  pl.off_o = pl.off_ml + up(np * 8);
  pl.off_s = pl.off_o + up(np * (size_t)a.Dh * 4);
  pl.bytes = pl.off_s + up(a.w_out != nullptr ? (size_t)a.B * a.H * (size_t)p.cap * 4 : 0);
  return CK_OK;
}

template <typename T, int DH, int GT, int NW, bool DIRECT>
int launch_stream(const PagedParams& p, int blocks, cudaStream_t st) {
  constexpr int rings = NW * (Ring<T, DH>::BYTES + Heads<T, DH, GT>::Q_FLOATS * 4);
  constexpr int fin = DIRECT ? NW * GT * 8 + NW * GT * DH * 4 : 0;
  constexpr int smem = rings > fin ? rings : fin;
  static_assert(smem <= 220 * 1024, "ring budget");
  auto kern = paged_stream_kernel<T, DH, GT, NW, DIRECT>;
  if (!smem_attr_ready(reinterpret_cast<const void*>(kern), smem)) return record_cuda_error();
  return launch_pdl(kern, dim3((unsigned)blocks), dim3(NW * 32), smem, st, p);
}

template <typename T, int DH, int GT>
int run_ring(const Plan& pl, cudaStream_t st) {
  const int seqs = pl.p.a.B * pl.p.units;
  constexpr int direct = DH * sizeof(T) >= 512 ? NWARP : NWARP_DIRECT;
  if (!pl.parts) return launch_stream<T, DH, GT, direct, true>(pl.p, seqs, st);
  return launch_stream<T, DH, GT, NWARP, false>(pl.p, stream_blocks(DH * (int)sizeof(T)), st);
}

template <typename T, int GT>
int run_dh(const Plan& pl, cudaStream_t st) {
  if (pl.p.a.Dh == 32) return run_ring<T, 32, GT>(pl, st);
  if (pl.p.a.Dh == 64) return run_ring<T, 64, GT>(pl, st);
  return run_ring<T, 128, GT>(pl, st);
}

template <typename T, int VEC, int NV>
int launch_simt(const PagedParams& p, cudaStream_t st) {
  const int smem = kSub * 8 + NWARP * p.gt * 8 + NWARP * p.gt * p.a.Dh * 4;
  const dim3 grid((unsigned)(p.a.B * p.n_chunks * p.units));
  if (p.gt == 1) return launch_pdl(paged_simt_kernel<T, VEC, NV, 1, NWARP>, grid, dim3(NWARP * 32), smem, st, p);
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
  p.seg = pl.parts ? reinterpret_cast<int2*>(w) : nullptr;
  p.part_ml = reinterpret_cast<float2*>(w + pl.off_ml);
  p.part_o = reinterpret_cast<float*>(w + pl.off_o);
  p.scores = a.w_out != nullptr ? reinterpret_cast<float*>(w + pl.off_s) : nullptr;
  const bool bf = a.dtype == CK_BF16;
  if (pl.ring) {
    if (bf)
      rc = p.gt == 4   ? run_dh<__nv_bfloat16, 4>(pl, st)
           : p.gt == 8 ? run_dh<__nv_bfloat16, 8>(pl, st)
                       : run_dh<__nv_bfloat16, 16>(pl, st);
    else
      rc = p.gt == 1 ? run_dh<float, 1>(pl, st) : run_dh<float, 4>(pl, st);
  } else if (bf) {
    if (pl.vec == 4)
      rc = pl.nv == 1 ? launch_simt<__nv_bfloat16, 4, 1>(p, st) : launch_simt<__nv_bfloat16, 4, 2>(p, st);
    else
      rc = pl.nv == 1 ? launch_simt<__nv_bfloat16, 1, 1>(p, st) : launch_simt<__nv_bfloat16, 1, 8>(p, st);
  } else if (pl.vec == 4) {
    rc = pl.nv == 1 ? launch_simt<float, 4, 1>(p, st) : launch_simt<float, 4, 2>(p, st);
  } else if (pl.vec == 2) {
    rc = launch_simt<float, 2, 1>(p, st);
  } else {
    rc = pl.nv == 1 ? launch_simt<float, 1, 1>(p, st) : launch_simt<float, 1, 8>(p, st);
  }
  if (rc != CK_OK || !pl.parts) return rc;
  const int out_blocks = a.B * a.H;
  const dim3 grid((unsigned)(out_blocks + (int64_t)a.B * pl.w_blocks));
  const size_t smem = a.w_out != nullptr ? (size_t)a.H * 8 : 0;
  const int chunked = pl.ring ? 0 : 1;
  if (bf)
    return launch_pdl(join_kernel<__nv_bfloat16>, grid, dim3(JT), smem, st, p, out_blocks,
                      (int)pl.w_blocks, chunked);
  return launch_pdl(join_kernel<float>, grid, dim3(JT), smem, st, p, out_blocks, (int)pl.w_blocks,
                    chunked);
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
