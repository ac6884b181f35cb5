// Eviction from a paged row pool by accumulated weight.
//
// A sequence of n rows over its budget keeps the `budget` best: the rows whose
// position is among the newest (position > newest - recent) first, then by
// weight, largest first (NaN last), equal ones by slot. Rows are not kept in
// order (attention over them has no order; `positions` says which is which):
// the kept rows behind the budget fill the holes before it, both in ascending
// slot order. Only those rows move, sources lie behind the budget and
// destinations before it, so every move is independent of every other; a
// session that gave one row too many moves one row.
//
// select_kernel: a cluster of CS CTAs per sequence finds the budget-th largest
// key by radix selection (8 bits a pass, most significant first) and numbers
// holes and movers. Each CTA holds a contiguous part of the slots, its keys in
// shared memory when they fit; histograms and per-warp counts are exchanged
// through distributed shared memory, so the slots' order decides every rank
// and no result depends on timing. move_kernel copies the rows, a warp a row.
//
// Bytes: weights and positions once (8 B a slot), 2 row reads / writes a mover.
#include "common.cuh"
#include "kernels.h"

namespace ck {

namespace {

constexpr int ST = 1024;         // threads of a selecting CTA
constexpr int SW = ST / 32;
constexpr int kKeyCap = 49152;   // keys a CTA keeps in shared memory
constexpr uint32_t kProtected = 0xFFFFFFFFu;

struct EvictParams {
  ck_evict_args a;
  int64_t cap;        // page_table_width * page_size
  int32_t max_moves;  // per sequence
  int32_t* counts;    // [B] moves
  int32_t* holes;     // [B][max_moves]
  int32_t* movers;    // [B][max_moves]
  int32_t key_cap;    // keys per CTA that shared memory holds
  int32_t move_blocks;  // move_kernel: blocks per sequence
};

// Order-preserving key of a weight: NaN lowest, -0 as +0; below kProtected.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ uint32_t cl_ld(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <int CS>
__global__ void __launch_bounds__(ST, 1) evict_select_kernel(const EvictParams p) {
  __shared__ uint32_t s_hist[4][256];
  __shared__ uint32_t s_sum[256];
  __shared__ int32_t s_max[1];
  __shared__ int32_t s_cnt[3][SW];  // per warp: equal keys, holes, movers
  __shared__ uint32_t s_pick[2];
  extern __shared__ uint32_t s_key[];
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = CS > 1 ? (int)cl_rank() : 0;
  const int b = blockIdx.x / CS;
  const ck_evict_args& a = p.a;
  const int64_t raw = a.lengths[b];
  const bool bad = raw < 0 || raw > p.cap;
  if (bad && rank == 0 && tid == 0) set_status(CK_ERR_INDEX, b, (int)raw);
  const int n = bad ? 0 : (int)raw;
  const int budget = a.budget;
  const float* w_in = a.w_in + (int64_t)b * a.w_in_ld;
  const int32_t* pos_in = a.pos_in + (int64_t)b * a.pos_in_ld;
  float* w_out = a.w_out + (int64_t)b * a.w_out_ld;
  int32_t* pos_out = a.pos_out + (int64_t)b * a.pos_out_ld;
  const int kept_n = min(n, budget);

  // tables of the rows that stay where they are (holes are written further
  // down), and with fill the columns behind them
  auto copy_tables = [&]() {
    const int end = a.fill ? a.out_width : kept_n;
    if (a.w_out != a.w_in)
      for (int j = rank * ST + tid; j < end; j += CS * ST) w_out[j] = j < kept_n ? w_in[j] : 0.f;
    if (a.pos_out != a.pos_in)
      for (int j = rank * ST + tid; j < end; j += CS * ST) pos_out[j] = j < kept_n ? pos_in[j] : -1;
  };
  if (n <= budget) {  // (the whole cluster: n is the sequence's)
    copy_tables();
    if (rank == 0 && tid == 0) {
      a.lengths_out[b] = (int32_t)raw;
      if (p.counts != nullptr) p.counts[b] = 0;
    }
    return;
  }

  // this CTA's slots [s0, s1), this warp's [w0, w1): contiguous, in order
  const int per_warp = ((n + CS * SW - 1) / (CS * SW) + 31) / 32 * 32;
  const int s0 = min(n, rank * SW * per_warp);
  const int s1 = min(n, s0 + SW * per_warp);
  const int w0 = min(n, s0 + warp * per_warp);
  const int w1 = min(s1, w0 + per_warp);
  const bool cached = SW * per_warp <= p.key_cap;

  for (int i = tid; i < 4 * 256; i += ST) (&s_hist[0][0])[i] = 0u;
  if (tid == 0) s_max[0] = INT32_MIN;
  __syncthreads();
  int64_t guard = INT64_MAX;  // positions above it are protected
  if (a.recent > 0) {
    int mx = INT32_MIN;
    for (int j = w0 + lane; j < w1; j += 32) mx = max(mx, pos_in[j]);
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) atomicMax(&s_max[0], mx);
    if (CS > 1) {
      cl_sync();
      mx = INT32_MIN;
#pragma unroll
      for (int r = 0; r < CS; ++r) mx = max(mx, (int)cl_ld(cl_map(&s_max[0], r)));
    } else {
      __syncthreads();
      mx = s_max[0];
    }
    guard = (int64_t)mx - a.recent;
  }
  auto make_key = [&](int j) -> uint32_t {
    if (a.recent > 0 && (int64_t)pos_in[j] > guard) return kProtected;
    return weight_key(w_in[j]);
  };
  auto key_at = [&](int j) -> uint32_t { return cached ? s_key[j - s0] : make_key(j); };

  // radix selection of the budget-th largest key
  uint32_t prefix = 0u;
  uint32_t want = (uint32_t)budget;  // rank of the wanted key among those under the prefix
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    for (int j = w0 + lane; j - lane < w1; j += 32) {
      uint32_t k = 0u;
      bool in = j < w1;
      if (in) {
        if (pass == 0) {
          k = make_key(j);
          if (cached) s_key[j - s0] = k;
        } else {
          k = key_at(j);
          in = (k >> (shift + 8)) == (prefix >> (shift + 8));
        }
      }
      // lanes with the same digit add once (the first digit is a handful of
      // exponents: one address would take most of the adds)
      const uint32_t digit = in ? (k >> shift) & 255u : 256u;
      const uint32_t peers = __match_any_sync(0xffffffffu, digit);
      if (in && (peers & ((1u << lane) - 1u)) == 0u) atomicAdd(&s_hist[pass][digit], __popc(peers));
    }
    if (CS > 1) cl_sync(); else __syncthreads();
    if (tid < 256) {
      uint32_t h = 0u;
      if (CS > 1) {
#pragma unroll
        for (int r = 0; r < CS; ++r) h += cl_ld(cl_map(&s_hist[pass][tid], r));
      } else {
        h = s_hist[pass][tid];
      }
      s_sum[tid] = h;
    }
    __syncthreads();
    if (warp == 0) {
      // lane owns digits 255 - 8 lane down to 248 - 8 lane
      uint32_t own[8], tot = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        own[i] = s_sum[255 - 8 * lane - i];
        tot += own[i];
      }
      uint32_t before = tot;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      before -= tot;
      if (before < want && want <= before + tot) {
        uint32_t acc = before;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (acc < want && want <= acc + own[i]) {
            s_pick[0] = (uint32_t)(255 - 8 * lane - i);
            s_pick[1] = want - acc;
          }
          acc += own[i];
        }
      }
    }
    __syncthreads();
    prefix |= s_pick[0] << shift;
    want = s_pick[1];
    __syncthreads();
  }
  // kept: key > prefix, and the first `want` slots whose key equals it

  int eq = 0;
  for (int j = w0 + lane; j < w1; j += 32) eq += key_at(j) == prefix;
  eq = __reduce_add_sync(0xffffffffu, eq);
  if (lane == 0) s_cnt[0][warp] = eq;
  // prefix over the warps of every CTA before this one and of this CTA
  auto base_of = [&](int which) -> int {
    if (CS > 1) cl_sync(); else __syncthreads();
    int sum = 0;
    if (CS > 1) {
      for (int r = 0; r < rank; ++r) sum += (int)cl_ld(cl_map(&s_cnt[which][lane], r));
    }
    if (lane < warp) sum += s_cnt[which][lane];
    return __reduce_add_sync(0xffffffffu, sum);
  };
  const int eq_base = base_of(0);

  auto sweep = [&](int& nh, int& nm, bool write) {
    int e = eq_base;
    for (int jb = w0; jb < w1; jb += 32) {
      const int j = jb + lane;
      const bool in = j < w1;
      const uint32_t k = in ? key_at(j) : 0u;
      const bool is_eq = in && k == prefix;
      const uint32_t em = __ballot_sync(0xffffffffu, is_eq);
      const uint32_t lt = (1u << lane) - 1u;
      const bool keep = in && (k > prefix || (is_eq && (uint32_t)(e + __popc(em & lt)) < want));
      e += __popc(em);
      const bool hole = in && !keep && j < budget;
      const bool mover = keep && j >= budget;
      const uint32_t hm = __ballot_sync(0xffffffffu, hole);
      const uint32_t mm = __ballot_sync(0xffffffffu, mover);
      if (write) {
        if (hole) p.holes[(int64_t)b * p.max_moves + nh + __popc(hm & lt)] = j;
        if (mover) p.movers[(int64_t)b * p.max_moves + nm + __popc(mm & lt)] = j;
      }
      nh += __popc(hm);
      nm += __popc(mm);
    }
  };
  int nh = 0, nm = 0;
  sweep(nh, nm, false);
  if (lane == 0) {
    s_cnt[1][warp] = nh;
    s_cnt[2][warp] = nm;
  }
  int hbase = base_of(1);
  int mbase = base_of(2);
  copy_tables();  // (the holes' entries are overwritten after the next barrier)
  nh = hbase;
  nm = mbase;
  sweep(nh, nm, true);
  if (rank == CS - 1 && warp == SW - 1 && lane == 0) {
    p.counts[b] = nh;  // the last warp ends with the totals; holes == movers
    a.lengths_out[b] = budget;
  }
  __threadfence();
  if (CS > 1) cl_sync(); else __syncthreads();
  const int total = __ldcg(p.counts + b);
  for (int i = rank * ST + tid; i < total; i += CS * ST) {
    const int h = __ldcg(p.holes + (int64_t)b * p.max_moves + i);
    const int m = __ldcg(p.movers + (int64_t)b * p.max_moves + i);
    w_out[h] = w_in[m];
    pos_out[h] = pos_in[m];
  }
  if (CS > 1) cl_sync();  // no CTA leaves while another may read its counts
}

// Rows of the movers into the holes: a warp a row, VEC bytes a lane.
template <typename V>
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p, int64_t row_vecs) {
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x / p.move_blocks;
  const int lane = threadIdx.x & 31;
  const int w = (blockIdx.x - b * p.move_blocks) * 8 + (threadIdx.x >> 5);
  const int total = p.counts[b];
  const ck_evict_args& a = p.a;
  const int32_t* table = a.page_table + (int64_t)b * a.page_table_ld;
  auto row_of = [&](int j) -> int64_t {
    const int slot = j / a.page_size;
    const int32_t page = table[slot];
    if (page < 0 || page >= a.num_pages) {
      if (lane == 0) set_status(CK_ERR_INDEX, b, page);
      return -1;
    }
    return ((int64_t)page * a.page_ld + (int64_t)(j - slot * a.page_size) * a.row_ld) * a.elem_bytes;
  };
  uint8_t* pool = reinterpret_cast<uint8_t*>(a.pool);
  for (int i = w; i < total; i += p.move_blocks * 8) {
    const int64_t to = row_of(p.holes[(int64_t)b * p.max_moves + i]);
    const int64_t from = row_of(p.movers[(int64_t)b * p.max_moves + i]);
    if (to < 0 || from < 0) continue;
    const V* src = reinterpret_cast<const V*>(pool + from);
    V* dst = reinterpret_cast<V*>(pool + to);
    int64_t c = lane;
    for (; c + 96 < row_vecs; c += 128) {
      V v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = src[c + 32 * u];
#pragma unroll
      for (int u = 0; u < 4; ++u) dst[c + 32 * u] = v[u];
    }
    for (; c < row_vecs; c += 32) dst[c] = src[c];
  }
}

struct EvictPlan {
  EvictParams p;
  int cs;
  size_t off_holes, off_movers, bytes;
};

int make_plan(const ck_evict_args& a, EvictPlan& pl) {
  if (a.elem_bytes != 2 && a.elem_bytes != 4) return CK_ERR_UNSUPPORTED;
  if (a.B < 0 || a.num_pages < 0 || a.page_size <= 0 || a.page_table_width < 0 || a.width <= 0 ||
      a.budget < 1 || a.recent < 0 || a.recent > a.budget)
    return CK_ERR_INVALID_ARG;
  EvictParams& p = pl.p;
  p.a = a;
  p.cap = (int64_t)a.page_table_width * a.page_size;
  if (p.cap > INT32_MAX / 2) return CK_ERR_INVALID_ARG;
  if (a.in_width < p.cap || a.out_width < (a.budget < p.cap ? a.budget : p.cap))
    return CK_ERR_INVALID_ARG;
  const int64_t behind = p.cap - a.budget;
  p.max_moves = behind <= 0 ? 0 : (int32_t)(behind < a.budget ? behind : a.budget);
  // A cluster of 8 per sequence once a CTA's threads would take several slots each.
  pl.cs = p.cap > 4096 ? 8 : 1;
  if ((int64_t)a.B * 8 > INT32_MAX) return CK_ERR_UNSUPPORTED;
  const int64_t per_cta = (p.cap + pl.cs - 1) / pl.cs + 32 * SW;
  p.key_cap = (int32_t)(per_cta < kKeyCap ? per_cta : kKeyCap);
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  const size_t list = up((size_t)a.B * p.max_moves * 4);
  pl.off_holes = up((size_t)a.B * 4);
  pl.off_movers = pl.off_holes + list;
  pl.bytes = p.max_moves > 0 ? pl.off_movers + list : 0;
  return CK_OK;
}

template <int CS>
int launch_select(const EvictParams& p, cudaStream_t st) {
  auto kern = evict_select_kernel<CS>;
  if (!smem_attr_ready(reinterpret_cast<const void*>(kern), kKeyCap * 4)) return record_cuda_error();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.a.B * CS));
  cfg.blockDim = dim3(ST);
  cfg.dynamicSmemBytes = (size_t)p.key_cap * 4;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return launch_cfg(cfg, kern, p);
}

}  // namespace

int evict_by_weight(const ck_evict_args& a, void* ws, size_t ws_bytes, cudaStream_t st) {
  EvictPlan pl;
  int rc = make_plan(a, pl);
  if (rc != CK_OK) return rc;
  if (a.B == 0) return CK_OK;
  EvictParams& p = pl.p;
  if (a.fill && (a.w_out == a.w_in || a.pos_out == a.pos_in)) return CK_ERR_INVALID_ARG;
  if (!a.lengths || !a.lengths_out || !a.w_in || !a.w_out || !a.pos_in || !a.pos_out)
    return CK_ERR_INVALID_ARG;
  if (p.cap > 0 && ((a.num_pages > 0 && !a.pool) || !a.page_table)) return CK_ERR_INVALID_ARG;
  if (pl.bytes > 0 && (ws == nullptr || ws_bytes < pl.bytes ||
                       (reinterpret_cast<uintptr_t>(ws) & 15u) != 0))
    return CK_ERR_WORKSPACE;
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  p.counts = p.max_moves > 0 ? reinterpret_cast<int32_t*>(w) : nullptr;
  p.holes = reinterpret_cast<int32_t*>(w + pl.off_holes);
  p.movers = reinterpret_cast<int32_t*>(w + pl.off_movers);
  rc = pl.cs == 1 ? launch_select<1>(p, st) : launch_select<8>(p, st);
  if (rc != CK_OK || p.max_moves == 0) return rc;
  // blocks for the longest possible list, and no more than fill the card
  const int64_t need = (p.max_moves + 7) / 8;
  int64_t fill = (8 * (int64_t)num_sms() + a.B - 1) / a.B;
  if (fill < 1) fill = 1;
  p.move_blocks = (int32_t)(need < fill ? need : fill);
  const int64_t row_bytes = (int64_t)a.width * a.elem_bytes;
  const dim3 grid((unsigned)((int64_t)a.B * p.move_blocks));
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.pool) | (uintptr_t)(a.page_ld * a.elem_bytes) |
                         (uintptr_t)(a.row_ld * a.elem_bytes) | (uintptr_t)row_bytes;
  if (bits % 16 == 0) return launch_pdl(evict_move_kernel<uint4>, grid, dim3(256), 0, st, p, row_bytes / 16);
  if (bits % 4 == 0) return launch_pdl(evict_move_kernel<uint32_t>, grid, dim3(256), 0, st, p, row_bytes / 4);
  return launch_pdl(evict_move_kernel<uint16_t>, grid, dim3(256), 0, st, p, row_bytes / 2);
}

}  // namespace ck

extern "C" size_t ck_evict_workspace_bytes(const ck_evict_args* args) {
  ck::EvictPlan pl;
  return args != nullptr && ck::make_plan(*args, pl) == CK_OK ? pl.bytes : 0;
}

extern "C" int ck_evict_by_weight(const ck_evict_args* args, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  if (args == nullptr) return CK_ERR_INVALID_ARG;
  return ck::evict_by_weight(*args, workspace, workspace_bytes,
                             reinterpret_cast<cudaStream_t>(stream));
}
