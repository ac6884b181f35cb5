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
// holes and movers. A warp holds a contiguous part of the slots, their keys in
// shared memory when they fit; histograms and per-warp counts are exchanged
// through distributed shared memory, so the slots' order decides every rank and
// no result depends on timing. move_kernel then moves the rows with their
// weights and positions, a warp a row.
//
// Bytes: weights and positions once (8 B a slot), a row read and written a mover.
// Measured (captured): 32 sequences, one row too many each, 8.1 us a call; 24 sequences of 700
// to 16384 slots down to 1000, rows of 3 KB, 34 us, of which 18 select and the rest
// moves 88 MB; one sequence of 131072 slots 39 us (26 select). The selection is bound
// by its barriers, the moves by the chain of index, page and row.
#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace ck {

namespace {

constexpr int ST = 512;          // threads of a selecting CTA
constexpr int SW = ST / 32;
constexpr int kKeyCap = 49152;   // slots whose key a CTA keeps in shared memory
constexpr int kBulkRoom = 24576; // shared memory of a warp that moves rows by bulk copies
// Bytes of the longest row moved that way: against copies through registers, us a
// call, 512 moves in each of 32 sequences of 2 KB rows 17.0 / 21.1, 500 in 16 of
// 4 KB 16.9 / 17.3, of 8 KB 25.0 / 23.7.
constexpr int kBulkRow = 4096;
constexpr int kListed = 1024;    // sequences that the moving kernel lists at a time
// Rows, and bytes of them, that the selecting kernel moves itself at most. Against a
// second launch, us a call: 32 sequences of 2 KB rows, 1 move 7.8 / 10.4, 128 moves
// 14.0 / 15.5, 256 moves 17.8 / 14.2; 16 of 4 KB rows, 100 moves 16.2 / 14.3, of 8
// KB 24.2 / 16.2. (The bound is on what the table allows, a step moves a row.)
constexpr int kFewMoves = 128;
constexpr int64_t kFewBytes = 512 * 1024;
constexpr uint32_t kProtected = 0xFFFFFFFFu;

struct EvictParams {
  ck_evict_args a;
  int64_t cap;        // page_table_width * page_size
  int32_t max_moves;  // per sequence
  int32_t* counts;    // [B] moves
  int32_t* holes;     // [B][max_moves]
  int32_t* movers;    // [B][max_moves]
  int32_t key_cap;    // slots per CTA that shared memory holds
  int32_t move_blocks;  // move_kernel: blocks; 0: select_kernel moves the rows
  int32_t vec_bytes;    // bytes that a lane copies at a time
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

// One move of sequence b: the weight and position at once, and the byte offsets
// of its rows in the pool (-1 for a page outside it, which is recorded).
__device__ __forceinline__ void start_move(const EvictParams& p, int b, int hole, int mover,
                                           int64_t& from, int64_t& to) {
  const ck_evict_args& a = p.a;
  const int32_t* table = a.page_table + (int64_t)b * a.page_table_ld;
  auto row_of = [&](int j) -> int64_t {
    const int slot = j / a.page_size;
    const int32_t page = table[slot];
    if (page < 0 || page >= a.num_pages) {
      set_status(CK_ERR_INDEX, b, page);
      return -1;
    }
    return ((int64_t)page * a.page_ld + (int64_t)(j - slot * a.page_size) * a.row_ld) * a.elem_bytes;
  };
  to = row_of(hole);
  from = row_of(mover);
  a.w_out[(int64_t)b * a.w_out_ld + hole] = a.w_in[(int64_t)b * a.w_in_ld + mover];
  a.pos_out[(int64_t)b * a.pos_out_ld + hole] = a.pos_in[(int64_t)b * a.pos_in_ld + mover];
}

// The rows of the lanes' moves (cnt of them), one after the other by the whole
// warp, 8 vectors a lane in flight.
template <typename V>
__device__ __forceinline__ void copy_rows_of(const EvictParams& p, int cnt, int64_t from, int64_t to) {
  const int lane = threadIdx.x & 31;
  const int64_t vecs = (int64_t)p.a.width * p.a.elem_bytes / (int64_t)sizeof(V);
  uint8_t* pool = reinterpret_cast<uint8_t*>(p.a.pool);
  for (int k = 0; k < cnt; ++k) {
    const int64_t f = __shfl_sync(0xffffffffu, from, k), t = __shfl_sync(0xffffffffu, to, k);
    if (f < 0 || t < 0) continue;
    const V* src = reinterpret_cast<const V*>(pool + f);
    V* dst = reinterpret_cast<V*>(pool + t);
    for (int64_t c = lane; c < vecs; c += 8 * 32) {
      V v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c + 32 * u < vecs) v[u] = src[c + 32 * u];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (c + 32 * u < vecs) dst[c + 32 * u] = v[u];
    }
  }
}

// Moves w, w + workers, ... of one sequence, a lane each, then their rows.
template <typename V>
__device__ __forceinline__ void move_rows(const EvictParams& p, int b, const int32_t* holes,
                                          const int32_t* movers, int total, int w, int workers) {
  const int lane = threadIdx.x & 31;
  const int per = max(1, min(32, (total + workers - 1) / workers));
  for (int64_t i0 = (int64_t)w * per; i0 < total; i0 += (int64_t)workers * per) {
    const int cnt = (int)min((int64_t)per, total - i0);
    int64_t from = -1, to = -1;
    if (lane < cnt) start_move(p, b, holes[i0 + lane], movers[i0 + lane], from, to);
    copy_rows_of<V>(p, cnt, from, to);
  }
}

__device__ __forceinline__ int4 cl_ld4(uint32_t addr) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

template <int CS>
__global__ void __launch_bounds__(ST, 2) evict_select_kernel(const EvictParams p) {
  constexpr int WARPS = CS * SW;  // warps of the cluster
  __shared__ uint32_t s_hist[4][256];
  __shared__ uint32_t s_sum[256];
  __shared__ int32_t s_max;
  __shared__ uint32_t s_pick[4][3];  // digit, rank among its keys, its keys
  __shared__ int4 s_cnt[SW];       // per warp: front keys equal, greater; back equal, greater
  __shared__ int4 s_all[WARPS];    // the same of the whole cluster
  __shared__ int32_t s_list[2][CS == 1 ? kFewMoves : 1];  // holes, movers that one CTA moves itself
  extern __shared__ __align__(16) uint32_t s_key[];  // [key_cap]
  grid_dep_wait();
  grid_dep_launch();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = CS > 1 ? (int)cl_rank() : 0;
  const int b = blockIdx.x / CS;
  const ck_evict_args& a = p.a;
  if (CS == 1 && p.move_blocks == 0)  // the rows' addresses are needed at the end: fetch them now
    for (int i = tid * 32; i < a.page_table_width; i += ST * 32)
      asm volatile("prefetch.global.L2 [%0];" ::"l"(a.page_table + (int64_t)b * a.page_table_ld + i));
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

  // tables of the rows that stay where they are (move_kernel overwrites the
  // holes'), and with fill the columns behind them (out_width may be INT32_MAX)
  auto copy_tables = [&]() {
    const int end = a.fill ? a.out_width : kept_n;
    if (a.w_out != a.w_in)
      for (int64_t j = rank * ST + tid; j < end; j += CS * ST) w_out[j] = j < kept_n ? w_in[j] : 0.f;
    if (a.pos_out != a.pos_in)
      for (int64_t j = rank * ST + tid; j < end; j += CS * ST) pos_out[j] = j < kept_n ? pos_in[j] : -1;
  };
  if (n <= budget) {  // (the whole cluster: n is the sequence's)
    copy_tables();
    if (rank == 0 && tid == 0) {
      a.lengths_out[b] = (int32_t)raw;
      if (p.move_blocks > 0) p.counts[b] = 0;
    }
    return;
  }

  // this CTA's slots begin at s0, this warp's are [w0, w1): contiguous, in order
  const int per_warp = ((n + WARPS - 1) / WARPS + 31) / 32 * 32;
  const int s0 = min(n, rank * SW * per_warp);
  const int w0 = min(n, s0 + warp * per_warp);
  const int w1 = min(n, w0 + per_warp);
  const bool cached = SW * per_warp <= p.key_cap;

  for (int i = tid; i < 4 * 256; i += ST) (&s_hist[0][0])[i] = 0u;
  if (tid == 0) s_max = INT32_MIN;
  // one pass over the tables, 8 slots a lane in flight
  int mx = INT32_MIN;
  for (int jb = w0 + lane; jb - lane < w1; jb += 8 * 32) {
    float w[8];
    int32_t q[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = jb + 32 * u;
      q[u] = j < w1 && a.recent > 0 ? __ldg(pos_in + j) : INT32_MIN;
      w[u] = j < w1 && cached ? __ldg(w_in + j) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int j = jb + 32 * u;
      mx = max(mx, q[u]);
      if (j < w1 && cached) s_key[j - s0] = weight_key(w[u]);
    }
  }
  int64_t guard = INT64_MAX;  // positions above it are protected
  __syncthreads();
  if (a.recent > 0) {
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (lane == 0) atomicMax(&s_max, mx);
    if (CS > 1) {
      cl_sync();
      mx = lane < CS ? (int)cl_ld(cl_map(&s_max, lane)) : INT32_MIN;
      mx = __reduce_max_sync(0xffffffffu, mx);
    } else {
      __syncthreads();
      mx = s_max;
    }
    guard = (int64_t)mx - a.recent;
  }
  // keys of the slots, from here on with the protection applied
  if (cached && a.recent > 0) {
#pragma unroll 8
    for (int j = w0 + lane; j < w1; j += 32)
      if ((int64_t)__ldg(pos_in + j) > guard) s_key[j - s0] = kProtected;
  }
  __syncwarp();
  auto make_key = [&](int j) -> uint32_t {
    if (cached) return s_key[j - s0];
    if (a.recent > 0 && (int64_t)__ldg(pos_in + j) > guard) return kProtected;
    return weight_key(__ldg(w_in + j));
  };

  // radix selection of the budget-th largest key
  uint32_t prefix = 0u;
  bool found = false;
  uint32_t want = (uint32_t)budget;  // rank of the wanted key among those under the prefix
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const int shift = 24 - 8 * pass;
    // adds of 1 with no result: the lanes that meet in a bin are counted by the
    // hardware, however few exponents the first digit has
    auto count = [&](uint32_t k) {
      if (pass == 0 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&s_hist[pass][(k >> shift) & 255u], 1u);
    };
    if (cached) {
      int j = w0 + 4 * lane;
#pragma unroll 2
      for (; j + 3 < w1; j += 128) {
        const uint4 k = *reinterpret_cast<const uint4*>(s_key + (j - s0));
        count(k.x);
        count(k.y);
        count(k.z);
        count(k.w);
      }
      for (int i = 0; i < 4; ++i)
        if (j + i < w1) count(s_key[j + i - s0]);
    } else {
#pragma unroll 4
      for (int j = w0 + lane; j < w1; j += 32) count(make_key(j));
    }
    if (CS > 1) cl_sync(); else __syncthreads();
    if (CS > 1) {
      if (tid < 256) {
        uint32_t h = 0u;
#pragma unroll
        for (int r = 0; r < CS; ++r) h += cl_ld(cl_map(&s_hist[pass][tid], r));
        s_sum[tid] = h;
      }
      __syncthreads();
    }
    if (CS == 1 || warp == 0) {  // (one CTA: every warp for itself, no second barrier)
      // lane owns digits 255 - 8 lane down to 248 - 8 lane
      const uint32_t* sum = CS > 1 ? s_sum : s_hist[pass];
      uint32_t own[8], tot = 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        own[i] = sum[255 - 8 * lane - i];
        tot += own[i];
      }
      uint32_t before = tot;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      before -= tot;
      uint32_t digit = 0u, left = 0u, keys = 0u;
      const bool here = before < want && want <= before + tot;
      if (here) {
        uint32_t acc = before;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (acc < want && want <= acc + own[i]) {
            digit = (uint32_t)(255 - 8 * lane - i);
            left = want - acc;
            keys = own[i];
          }
          acc += own[i];
        }
      }
      const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
      digit = __shfl_sync(0xffffffffu, digit, src);
      left = __shfl_sync(0xffffffffu, left, src);
      keys = __shfl_sync(0xffffffffu, keys, src);
      if (CS > 1) {
        if (lane == 0) {
          s_pick[pass][0] = digit;
          s_pick[pass][1] = left;
          s_pick[pass][2] = keys;
        }
      } else {
        prefix |= digit << shift;
        want = left;
        found = left == keys;
      }
    }
    if (CS > 1) {
      __syncthreads();
      prefix |= s_pick[pass][0] << shift;
      want = s_pick[pass][1];
      found = want == s_pick[pass][2];
    }
    if (found && pass < 3) {
      // every key under this prefix is kept (with weights all different, mostly
      // one key after three digits): the keys above prefix - 1
      prefix -= 1u;  // (not 0: that would keep all n > budget rows)
      want = 0u;
      break;
    }
  }
  // kept: key > prefix, and the first `want` slots whose key equals it

  int4 c = make_int4(0, 0, 0, 0);
#pragma unroll 8
  for (int j = w0 + lane; j < w1; j += 32) {
    const uint32_t k = make_key(j);
    const bool back = j >= budget;
    c.x += !back && k == prefix;
    c.y += !back && k > prefix;
    c.z += back && k == prefix;
    c.w += back && k > prefix;
  }
  c.x = __reduce_add_sync(0xffffffffu, c.x);
  c.y = __reduce_add_sync(0xffffffffu, c.y);
  c.z = __reduce_add_sync(0xffffffffu, c.z);
  c.w = __reduce_add_sync(0xffffffffu, c.w);
  if (lane == 0) s_cnt[warp] = c;
  if (CS > 1) cl_sync(); else __syncthreads();
  for (int i = tid; i < WARPS; i += ST) {
    if (CS > 1) s_all[i] = cl_ld4(cl_map(&s_cnt[i % SW], i / SW));
    else s_all[i] = s_cnt[i];
  }
  copy_tables();
  __syncthreads();
  // What the warps before this one hold: equal keys, of which the first `want`
  // are kept, holes and movers. Equal keys come in slot order, so of a warp's
  // kept ones those in front come first.
  const int me = rank * SW + warp;
  int eq_base = 0, hole_base = 0, mover_base = 0, moves = 0;
  {
    int eq_sum = 0;
    for (int i0 = 0; i0 < WARPS; i0 += 32) {
      const int i = i0 + lane;
      const int4 v = i < WARPS ? s_all[i] : make_int4(0, 0, 0, 0);
      int eq = v.x + v.z, run = eq;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += u;
      }
      const int kept_eq = max(0, min(eq, (int)want - (eq_sum + run - eq)));
      const int kept_front = min(kept_eq, v.x);
      const int f0 = min(n, i * per_warp), f1 = min(n, f0 + per_warp);
      const int front = i < WARPS ? max(0, min(f1, budget) - min(f0, budget)) : 0;
      const int holes = front - v.y - kept_front;
      const int movers = v.w + kept_eq - kept_front;
      const bool mine = i < me;
      eq_base += __reduce_add_sync(0xffffffffu, mine ? eq : 0);
      hole_base += __reduce_add_sync(0xffffffffu, mine ? holes : 0);
      mover_base += __reduce_add_sync(0xffffffffu, mine ? movers : 0);
      moves += __reduce_add_sync(0xffffffffu, holes);
      eq_sum += __shfl_sync(0xffffffffu, run, 31);
    }
  }
  const uint32_t lt = (1u << lane) - 1u;
  const bool here = CS == 1 && p.move_blocks == 0;
  int32_t* holes = here ? s_list[0] : p.holes + (int64_t)b * p.max_moves;
  int32_t* movers = here ? s_list[1] : p.movers + (int64_t)b * p.max_moves;
  for (int jb = w0; jb < w1; jb += 32) {
    const int j = jb + lane;
    const bool in = j < w1;
    const uint32_t k = in ? make_key(j) : 0u;
    const bool is_eq = in && k == prefix;
    const uint32_t em = __ballot_sync(0xffffffffu, is_eq);
    const bool keep = in && (k > prefix || (is_eq && eq_base + __popc(em & lt) < (int)want));
    eq_base += __popc(em);
    const bool hole = in && !keep && j < budget;
    const bool mover = keep && j >= budget;
    const uint32_t hm = __ballot_sync(0xffffffffu, hole);
    const uint32_t mm = __ballot_sync(0xffffffffu, mover);
    if (hole) holes[hole_base + __popc(hm & lt)] = j;
    if (mover) movers[mover_base + __popc(mm & lt)] = j;
    hole_base += __popc(hm);
    mover_base += __popc(mm);
  }
  if (rank == 0 && tid == 0) {
    if (p.move_blocks > 0) p.counts[b] = moves;
    a.lengths_out[b] = budget;
  }
  if (p.move_blocks > 0) {
    if (CS > 1) cl_sync();  // no CTA leaves while another may read its counts
    return;
  }
  // a handful of movers at most: moved here
  if (CS > 1) {
    __threadfence();
    cl_sync();
  } else {
    __syncthreads();
  }
  switch (p.vec_bytes) {
    case 16: move_rows<uint4>(p, b, holes, movers, moves, me, WARPS); break;
    case 4: move_rows<uint32_t>(p, b, holes, movers, moves, me, WARPS); break;
    default: move_rows<uint16_t>(p, b, holes, movers, moves, me, WARPS);
  }
}

// The same through shared memory by bulk copies, a lane issuing its move's: the
// moves of lanes [first, first + slots), whose rows fill the warp's `room`. False
// when the copies did not come in time (recorded): the barrier is not used again.
__device__ __forceinline__ bool copy_rows_bulk(const EvictParams& p, int first, int slots, int64_t from,
                                               int64_t to, uint32_t room, uint64_t* bar,
                                               uint32_t& phase) {
  const int lane = threadIdx.x & 31;
  const uint32_t row = (uint32_t)(p.a.width * p.a.elem_bytes);
  uint8_t* pool = reinterpret_cast<uint8_t*>(p.a.pool);
  const bool mine = lane >= first && lane < first + slots && from >= 0 && to >= 0;
  const uint32_t rows = __popc(__ballot_sync(0xffffffffu, mine));
  if (rows == 0u) return true;
  if (lane == 0) mbar_arrive_expect_tx(bar, rows * row);
  __syncwarp();
  const uint32_t at = room + (uint32_t)(lane - first) * row;
  if (mine)
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(at),
        "l"(pool + from), "r"(row), "r"(smem_u32(bar))
        : "memory");
  const bool ok = __all_sync(0xffffffffu, mbar_wait_park(bar, phase, nullptr, 40));
  phase ^= 1u;
  if (!ok) {  // no copy may land after this block's exit: the same time for them again
    mbar_wait_park(bar, phase ^ 1u, nullptr, 41);
    return false;
  }
  if (mine) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(pool + to),
                 "r"(at), "r"(row)
                 : "memory");
    bulk_commit();
    bulk_wait_read<0>();  // before the next rows come into this place
  }
  __syncwarp();
  return true;
}

// Every sequence's moves as one list, an equal share of it to every warp: a
// batch has sequences with thousands of moves beside sequences with none. The
// blocks are one round of what the SMs hold. BULK (rows of a multiple of 16
// bytes, aligned, at most kBulkRow): rows go through shared memory by bulk
// copies, a lane issuing a row's, which keeps 192 KB an SM in flight; else
// through registers, V at a time.
template <typename V, bool BULK>
__global__ void __launch_bounds__(BULK ? 128 : 256) evict_move_kernel(const EvictParams p) {
  constexpr int NW = BULK ? 4 : 8;
  __shared__ int64_t s_end[kListed];  // moves up to and with each sequence
  __shared__ int64_t s_warp[NW];
  __shared__ __align__(8) uint64_t s_bar[NW];
  extern __shared__ __align__(128) uint8_t s_rows[];  // BULK: [NW][kBulkRoom]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (BULK && tid < NW) {
    mbar_init(&s_bar[tid], 1);
    fence_mbar_init();
    fence_proxy_async_smem();
  }
  grid_dep_wait();
  grid_dep_launch();
  uint32_t phase = 0;
  bool ok = true;  // of the warp
  const int slots = BULK ? (int)min((int64_t)32, (int64_t)kBulkRoom / (p.a.width * p.a.elem_bytes)) : 32;  // rows at a time
  for (int b0 = 0; b0 < p.a.B; b0 += kListed) {
    const int n = min(kListed, p.a.B - b0);
    // sums over the sequences: neighbouring ones a thread
    constexpr int PER = kListed / (32 * NW);
    int64_t own[PER], run = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = tid * PER + i;
      run += k < n ? p.counts[b0 + k] : 0;
      own[i] = run;
    }
    int64_t before = run;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += v;
    }
    __syncthreads();  // (the sums of the sequences before these have been read; the barriers are set)
    if (lane == 31) s_warp[warp] = before;
    __syncthreads();
    before -= run;
    for (int v = 0; v < warp; ++v) before += s_warp[v];
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (tid * PER + i < n) s_end[tid * PER + i] = before + own[i];
    __syncthreads();
    const int64_t total = s_end[n - 1];
    const int64_t workers = (int64_t)gridDim.x * NW, w = (int64_t)blockIdx.x * NW + warp;
    const int per = (int)max((int64_t)1, min((int64_t)32, (total + workers - 1) / workers));
    for (int64_t i0 = w * per; i0 < total; i0 += workers * per) {
      const int cnt = (int)min((int64_t)per, total - i0);
      int64_t from = -1, to = -1;
      if (lane < cnt) {
        int lo = 0, hi = n - 1;  // the first sequence that ends behind this move
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          if (s_end[mid] > i0 + lane) hi = mid; else lo = mid + 1;
        }
        const int64_t k = i0 + lane - (lo > 0 ? s_end[lo - 1] : 0);
        const int64_t at = (int64_t)(b0 + lo) * p.max_moves + k;
        start_move(p, b0 + lo, p.holes[at], p.movers[at], from, to);
      }
      if constexpr (BULK) {
        for (int k = 0; k < cnt && ok; k += slots)
          ok = copy_rows_bulk(p, k, slots, from, to, smem_u32(s_rows) + warp * kBulkRoom, &s_bar[warp],
                              phase);
      } else {
        copy_rows_of<V>(p, cnt, from, to);
      }
    }
  }
  if (BULK) bulk_wait<0>();  // this lane's stores are done
}

struct EvictPlan {
  EvictParams p;
  int cs;
  bool few;  // one launch
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
  // CTAs per sequence, measured on B200 (whole call, us, by CTAs): 24 sequences
  // of 4096 slots 28.7 / 28.7 / 32.8 (1 / 4 / 8), of 16384 slots 45.1 / 32.8 /
  // 34.8; one of 16384 slots 34.8 / 22.5 / 22.5, one of 131072 47.1 / 41.0 (8 /
  // 16). 16 CTAs only where they all find an SM: 24 sequences of 16384 slots
  // took 57.3.
  pl.cs = p.cap <= 2048 ? 1 : (p.cap <= 16384 ? 4 : 8);
  if (p.cap > 65536 && 16 * (int64_t)a.B <= num_sms()) pl.cs = 16;
  if ((int64_t)a.B * 16 > INT32_MAX) return CK_ERR_UNSUPPORTED;
  const int64_t per_cta = (p.cap + pl.cs - 1) / pl.cs + 32 * SW;
  p.key_cap = (int32_t)(per_cta < kKeyCap ? per_cta : kKeyCap);
  auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
  const size_t list = up((size_t)a.B * p.max_moves * 4);
  pl.off_holes = up((size_t)a.B * 4);
  pl.off_movers = pl.off_holes + list;
  // (one CTA a sequence and few movers: they never leave shared memory)
  pl.few = p.max_moves <= kFewMoves && (int64_t)p.max_moves * a.width * a.elem_bytes <= kFewBytes;
  pl.bytes = p.max_moves > 0 && !(pl.cs == 1 && pl.few) ? pl.off_movers + list : 0;
  return CK_OK;
}

template <int CS>
int launch_select(const EvictParams& p, cudaStream_t st) {
  auto kern = evict_select_kernel<CS>;
  if (!smem_attr_ready(reinterpret_cast<const void*>(kern), kKeyCap * 4)) return record_cuda_error();
  if (CS > 8) {  // more than the portable 8 CTAs: allowed once per device
    static std::atomic<uint64_t> allowed{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return record_cuda_error();
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if ((allowed.load(std::memory_order_relaxed) & bit) == 0) {
      if (cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return record_cuda_error();
      allowed.fetch_or(bit, std::memory_order_relaxed);
    }
  }
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
  // (tables without a column have no address)
  if (!a.lengths || !a.lengths_out || (p.cap > 0 && (!a.w_in || !a.pos_in)) ||
      ((p.cap > 0 || a.fill) && (!a.w_out || !a.pos_out)))
    return CK_ERR_INVALID_ARG;
  if (p.cap > 0 && ((a.num_pages > 0 && !a.pool) || !a.page_table)) return CK_ERR_INVALID_ARG;
  if (pl.bytes > 0 && (ws == nullptr || ws_bytes < pl.bytes ||
                       (reinterpret_cast<uintptr_t>(ws) & 15u) != 0))
    return CK_ERR_WORKSPACE;
  uint8_t* w = reinterpret_cast<uint8_t*>(ws);
  p.counts = reinterpret_cast<int32_t*>(w);
  p.holes = reinterpret_cast<int32_t*>(w + pl.off_holes);
  p.movers = reinterpret_cast<int32_t*>(w + pl.off_movers);
  const uintptr_t bits = reinterpret_cast<uintptr_t>(a.pool) | (uintptr_t)(a.page_ld * a.elem_bytes) |
                         (uintptr_t)(a.row_ld * a.elem_bytes) |
                         (uintptr_t)((int64_t)a.width * a.elem_bytes);
  p.vec_bytes = bits % 16 == 0 ? 16 : (bits % 4 == 0 ? 4 : 2);
  // One round of blocks (two or three an SM), or fewer where the lists cannot be that
  // long. A short list (sessions that stay at their budget)
  // is moved by the selecting kernel, without a second launch.
  const bool bulk = p.vec_bytes == 16 && (int64_t)a.width * a.elem_bytes <= kBulkRow;
  const int64_t need = ((int64_t)a.B * p.max_moves + 3) / 4, fill = (bulk ? 2 : 3) * (int64_t)num_sms();
  p.move_blocks = pl.few ? 0 : (int32_t)(need < fill ? need : fill);
  rc = pl.cs == 1   ? launch_select<1>(p, st)
       : pl.cs == 4 ? launch_select<4>(p, st)
       : pl.cs == 8 ? launch_select<8>(p, st)
                    : launch_select<16>(p, st);
  if (rc != CK_OK || p.move_blocks == 0) return rc;
  const dim3 grid((unsigned)p.move_blocks);
  if (bulk) {
    auto kern = evict_move_kernel<uint4, true>;
    if (!smem_attr_ready(reinterpret_cast<const void*>(kern), 4 * kBulkRoom)) return record_cuda_error();
    return launch_pdl(kern, grid, dim3(128), 4 * kBulkRoom, st, p);
  }
  if (p.vec_bytes == 16) return launch_pdl(evict_move_kernel<uint4, false>, grid, dim3(256), 0, st, p);
  if (p.vec_bytes == 4) return launch_pdl(evict_move_kernel<uint32_t, false>, grid, dim3(256), 0, st, p);
  return launch_pdl(evict_move_kernel<uint16_t, false>, grid, dim3(256), 0, st, p);
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
