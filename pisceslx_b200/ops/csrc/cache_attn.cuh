// Attention of new tokens over cached ones (sm_100a): causal, grouped heads, keys and values in bf16 pages (of 8-bit pages what the
// tokens see is widened to bf16 first, by cache_widen_kernel), an optional window with a few first tokens that stay visible.
//
// Query position p of a sequence sees key j <= p if there is no window w, or j > p - w, or j < first.  With n cached tokens, the
// new ones among them, the last query sits at n - 1.
//
// Rows of a query tile are the (token, query head) pairs that share a key head: 128 / G tokens of its G heads, so that a tile is
// full from 128 / G tokens on and keys and values are read once for all heads of the group.  One persistent CTA per SM walks
// (query block, sequence, key head, key range) items, heavy blocks first.  A block has two query tiles or one; the key tiles of a
// lone query tile are dealt out to both halves of the CTA in turn.  What few query blocks leave idle is used by cutting their
// keys into ranges, whose unnormalised sums a second kernel joins.  Only key tiles with a visible key are walked: those of the
// first tokens, then those from the block's first windowed key on.
//
// Roles (the pipeline is that of attention_fwd.cuh):
//   warps 0..3  softmax of tile 0, warps 4..7 of tile 1 (or of every other key tile): a thread owns a row = a TMEM lane
//   warp 8      TMA: query tiles and keys, one copy for each `box` rows of a page; warp 10: values
//   warp 9      MMA: S = Q K^T (SS), O += P V (TS), one thread's products in order
//   warp 11     gives its registers away
// TMEM columns: [0,128) S0/P0, [128,256) S1/P1, [256,256+D) O0, [384,384+D) O1.
//
// 32 query heads over 8 of 128: 512 tokens of 16384 158 us (856 TFLOP/s; 82 at the measured peak), 4096 of 32768 over 8-bit pages
// 2035 us (1010 TFLOP/s; 1254).  The kernel for prompts (attention_fwd.cuh), whose pipeline this is, takes a prompt without a prefix
// 8 to 9 % faster (16384 tokens 1926 us for 2085, 4096 127 for 140): pages in boxes, slots looked up, keys cleared.  The rest of the
// distance to the peak both have: a step, a key tile for both query tiles, takes 3700 cycles here where its products take 2048, since
// the softmax of a half (2000) and its products (1000, and as much behind the other's) follow one another.  Scores of a half's next
// tile ahead of that take tensor memory that only parts of 64 keys leave free, and then its products read the query tile twice as
// often (180 us).  Weights handed over in two portions: 161 us.  An item costs 6 us to begin and to end besides, and a short call is
// uneven: 128 of 148 SMs have work in the first of these.
//
// What a page holds past the end of a sequence, or in front of everything that the block sees, may be anything: its scores are
// masked and its values cleared (a zero weight times NaN is NaN).
#pragma once
#include "attention_math.cuh"
#include "cache_ops.h"
#include "chain.cuh"
#include "per_device.h"
#include "sm100.cuh"
#include "tensormap.h"

namespace yv {

struct CacheWidenArgs {
  const void *k, *v, *k_scale, *v_scale;
  void *ko, *vo;
  const int *table, *lens, *cu_q;
  int table_width, block, num_blocks, hk, room, max_q, window, first;
  uint32_t* status;
};

struct CacheAttnParams {
  CUtensorMap tma_q;             // (d, query head, token), box (64, G, 128 / G)
  CUtensorMap tma_k, tma_v;      // (d, key head, slot), box (64, 1, box)
  __nv_bfloat16* o;
  int64_t o_ld;
  float *po, *pml;
  const int *cu_q, *table, *lens;   // without a table key j of sequence b has the slot b * room + CacheRoom::row(j)
  int64_t total_q, items;
  int hq, hk, group, per_tile, batch, max_q, block, box, num_blocks, table_width;
  int window, first, two, splits, zero_rest, first_row, room;
  float scale_log2;
  uint32_t* status;
};

constexpr int kCaTile = 128;                    // rows of a query tile, keys of a key tile
// pairs of 16 whose 2^x is a polynomial (512 of 16384 tokens: 2 160 us, 3 157, 4 159, 6 162)
constexpr int kCaPoly = 3;
constexpr float kCaMask = -1.0e30f;
constexpr float kCaRescale = 8.0f;              // log2 units

template <int D>
struct CacheAttn {
  static constexpr int kThreads = 384;
  // registers of the softmax warps and of the others: together what the block was launched with (3 x 168)
  static constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
  static constexpr int kBytes = kCaTile * D * 2;                     // a tile of Q, K or V
  static constexpr int kStages = D == 64 ? 3 : 2;
  static constexpr int kTotal = kBytes * (2 + 2 * kStages) + kCaTile * 8 + 256 + 1024;
};

// Item of round r of a CTA; every other round runs backwards, so that no CTA gets the heaviest item of each.
__device__ __forceinline__ int64_t ca_item_of(int64_t r) {
  return r * gridDim.x + ((r & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
}

// Clears rows of o that belong to no sequence: behind the last one (zero_rest & 1), in front of the first (& 2).
template <int D, int THREADS>
__device__ __forceinline__ void ca_zero(const CacheAttnParams& p) {
  if (p.zero_rest == 0) return;
  const int64_t vecs = static_cast<int64_t>(p.hq) * D / 8, me = static_cast<int64_t>(blockIdx.x) * THREADS + threadIdx.x;
  auto clear = [&](int64_t from, int64_t to) {
    for (int64_t i = max(from, int64_t(0)) * vecs + me; i < min(to, p.total_q) * vecs; i += static_cast<int64_t>(gridDim.x) * THREADS)
      *reinterpret_cast<uint4*>(p.o + i / vecs * p.o_ld + i % vecs * 8) = make_uint4(0, 0, 0, 0);
  };
  if ((p.zero_rest & 1) != 0) clear(p.cu_q != nullptr ? p.cu_q[p.batch] : p.first_row + p.batch, p.total_q);
  if ((p.zero_rest & 2) != 0 && p.cu_q != nullptr) clear(0, p.cu_q[0]);
}

// The key tiles that a block of queries walks, as a list: those of the first tokens, then those from the window's first key on.
struct CacheTiles {
  int lo, last, first_end;           // keys that any row of the block sees: [0, first_end) and [lo, last]
  int ns, w0, begin;                 // tiles in front of the window's first one, that one, first entry of this key range in the list

  // queries at positions from .. to; range `split` of `splits`.  Returns the entry behind the last one.
  __device__ __forceinline__ int set(int from, int to, int window, int first, int split, int splits) {
    last = to;
    lo = window > 0 ? max(from - window + 1, 0) : 0;
    first_end = window > 0 ? min(first, lo) : 0;
    w0 = lo / kCaTile;
    ns = min((first_end + kCaTile - 1) / kCaTile, w0);
    const int all = list_end(last);
    begin = static_cast<int>(static_cast<int64_t>(all) * split / splits);
    return static_cast<int>(static_cast<int64_t>(all) * (split + 1) / splits);
  }
  // entries of the list up to the tile with key `k`
  __device__ __forceinline__ int list_end(int k) const {
    if (k < 0) return 0;
    const int tile = k / kCaTile;
    return tile < w0 ? min(ns, tile + 1) : ns + tile - w0 + 1;
  }
  // first key of the tile at a place of the range
  __device__ __forceinline__ int first_key(int at) const {
    at += begin;
    return (at < ns ? at : w0 + at - ns) * kCaTile;
  }
  __device__ __forceinline__ bool seen(int key) const { return key <= last && (key >= lo || key < first_end); }
  // whether any of n keys from `key` on is seen, and whether all of a tile are
  __device__ __forceinline__ bool any(int key, int n) const { return key <= last && (key + n > lo || key < first_end); }
  __device__ __forceinline__ bool whole(int key) const {
    return key + kCaTile - 1 <= last && (key >= lo || key + kCaTile <= first_end);
  }
};

// Rows that the keys which a sequence's new tokens see have among the `room` of it that are widened: those of the first tokens' tiles,
// then those from the window's first tile on (of CacheTiles the list for all new tokens, in whole tiles; a block's list is a part of it).
struct CacheRoom {
  int keep, skip;                    // keys below keep have rows of their own number, others lie skip rows further in front
  __device__ __forceinline__ CacheRoom(int from, int window, int first) {
    CacheTiles t;
    t.set(from, from, window, first, 0, 1);
    keep = t.ns * kCaTile;
    skip = (t.w0 - t.ns) * kCaTile;
  }
  __device__ __forceinline__ int row(int key) const { return key < keep ? key : key - skip; }
  __device__ __forceinline__ int key(int row) const { return row < keep ? row : row + skip; }
};

// Rows of q and cached tokens of sequence b; what is out of range is reported (if `report`) and counts as empty.
__device__ __forceinline__ void ca_sequence(const CacheAttnParams& p, int b, int& q_begin, int& q_len, int& k_len, bool report) {
  q_begin = p.cu_q != nullptr ? p.cu_q[b] : p.first_row + b;
  const int q_end = p.cu_q != nullptr ? p.cu_q[b + 1] : q_begin + 1;
  q_len = q_end - q_begin;
  if (q_begin < 0 || q_end > p.total_q || q_len < 0 || q_len > p.max_q) {
    if (report && p.status != nullptr) atomicOr(p.status, kStatusBadArgument);
    q_len = 0;
  }
  k_len = p.lens[b];
  if (k_len < 0 || static_cast<int64_t>(k_len) > static_cast<int64_t>(p.table_width) * p.block) {
    if (report && p.status != nullptr) atomicOr(p.status, kStatusIndexOutOfRange);
    k_len = 0;
  }
}

struct CacheItem : CacheTiles {
  int b, kvh, split;
  int t0, q_begin, q_len, shift;     // first token of the block; a sequence's rows of q; key of query i is i + shift
  int n[2];                          // key tiles of the two halves
  bool second, shared;               // there is a second query tile; both halves work on the first

  __device__ __forceinline__ bool load(const CacheAttnParams& p, int64_t r) {
    const int64_t w = ca_item_of(r);
    if (w >= p.items) return false;
    const int per = p.hk * p.batch * p.splits;
    const int rank = static_cast<int>(w / per);
    int rest = static_cast<int>(w - static_cast<int64_t>(rank) * per);
    b = rest / (p.hk * p.splits);
    rest -= b * p.hk * p.splits;
    split = rest / p.hk;
    kvh = rest - split * p.hk;
    int k_len;
    ca_sequence(p, b, q_begin, q_len, k_len, threadIdx.x == 0);
    const int tokens = p.per_tile << p.two;
    const int blk = (q_len + tokens - 1) / tokens - 1 - rank;                    // late (heavy) blocks first
    if (blk < 0) return false;
    t0 = blk * tokens;
    second = p.two != 0 && t0 + p.per_tile < q_len;
    shift = k_len - q_len;
    const int end = set(t0 + shift, min(t0 + tokens, q_len) - 1 + shift, p.window, p.first, split, p.splits);
    n[0] = min(max(list_end(min(t0 + p.per_tile, q_len) - 1 + shift) - begin, 0), end - begin);
    n[1] = second ? end - begin : 0;
    shared = !second && n[0] > 1;
    if (shared) {
      n[1] = n[0] / 2;
      n[0] -= n[1];
    }
    return true;
  }
  __device__ __forceinline__ int count(int t) const { return t == 0 ? n[0] : n[1]; }
  __device__ __forceinline__ int tiles() const { return shared ? n[0] + n[1] : n[0] > n[1] ? n[0] : n[1]; }
  __device__ __forceinline__ int steps() const { return n[0] > n[1] ? n[0] : n[1]; }
  // place of a half's step j among the item's tiles
  __device__ __forceinline__ int place(int t, int j) const { return shared ? 2 * j + t : j; }
  __device__ __forceinline__ bool last_reader(int t, int j) const { return shared || t == 1 || j >= n[1]; }
};

// Flat slot of a key of sequence b; at a table entry outside the pool (reported) some valid one.
__device__ __forceinline__ int ca_slot(const CacheAttnParams& p, int b, int key) {
  const int bi = key / p.block;
  int page = p.table[static_cast<int64_t>(b) * p.table_width + bi];
  if (page < 0 || page >= p.num_blocks) {
    if (p.status != nullptr) atomicOr(p.status, kStatusIndexOutOfRange);
    page = 0;
  }
  return page * p.block + (key - bi * p.block);
}

template <int D>
__global__ void __launch_bounds__(CacheAttn<D>::kThreads, 1) cache_attn_kernel(const __grid_constant__ CacheAttnParams p) {
  using S = CacheAttn<D>;
  constexpr int kStages = S::kStages;
  constexpr int kSlabs = D / 64;
  constexpr uint32_t kSlab = kCaTile * 128;            // 128 rows x 64 columns
  constexpr uint32_t kIdescQK = make_idesc_bf16(128, 128, false, false);
  constexpr uint32_t kIdescPV = make_idesc_bf16(128, D, false, true);
  constexpr uint32_t kTmemCols = 512;
  constexpr uint32_t kOCol = 256;

  extern __shared__ uint8_t ca_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ca_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;                                  // [2]
  uint8_t* sK = sQ + 2 * S::kBytes;
  uint8_t* sV = sK + kStages * S::kBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + kStages * S::kBytes);
  uint64_t* q_full = bars;                 // [2]
  uint64_t* q_empty = bars + 2;            // [2]
  uint64_t* s_full = bars + 4;             // [2]
  uint64_t* p_full = bars + 6;             // [2]
  uint64_t* o_full = bars + 8;             // [2]
  uint64_t* k_full = bars + 10;            // [kStages]
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* ml_full = v_empty + kStages;   // shared: the second half's maxima and sums are in ml
  uint64_t* ml_empty = ml_full + 1;        //         they and its O have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ml_empty + 1);
  float2* ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(bars) + 256);     // [128] per row

  constexpr bool kWarpIssues = D == 128;               // as in attention_fwd.cuh
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&p.tma_q);
    tma_prefetch_desc(&p.tma_k);
    tma_prefetch_desc(&p.tma_v);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_full[t], 4);
      mbar_init(&o_full[t], 1);
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    mbar_init(ml_full, 4);
    mbar_init(ml_empty, 4);
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  // the tensor memory is this kernel's before the next one may begin
  chain_next();
  chain_wait();
  ca_zero<D, S::kThreads>(p);
  const uint32_t tmem_base = *tmem_slot;

  if (warp >= 8) regs_give<S::kOtherRegs>();
  if (warp == 8 || warp == 10) {
    // ------------------------------------ copies --------------------------------------------
    // The whole warp walks the items: its lanes look up the slots of the next 32 copies at a time, ahead of their use (looked up one
    // by one, each costs the latency of a load: 16 streams of 32 pages 168 us).
    // Keys and values have a warp each: a tile of keys that is wanted early does not wait until the values in front of it have room.
    const bool keys = warp == 8;
    const CUtensorMap* map = keys ? &p.tma_k : &p.tma_v;
    uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
    uint8_t* ring = keys ? sK : sV;
    const uint32_t lead = elect_one() ? 1u : 0u;
    bool ok = true;
    uint32_t kv = 0, nq[2] = {0u, 0u};            // key tiles and Q tiles so far
    const int boxes = kCaTile / p.box, per_look = 32 / boxes;              // copies of a tile, tiles of a look
    for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
      CacheItem it;
      if (!it.load(p, r)) continue;
      const int n = it.tiles();
      // slot of copy `lane` of the tiles from j0 on; negative where no key of it is seen (the keys stay where they are)
      auto look = [&](int j0) {
        const int j = j0 + lane / boxes;
        if (j >= n) return -1;
        const int a = it.first_key(j) + (lane % boxes) * p.box;
        if (!it.any(a, p.box)) return -1;
        return p.table != nullptr ? ca_slot(p, it.b, a) : it.b * p.room + CacheRoom(it.shift, p.window, p.first).row(a);
      };
      int rows = look(0), next = -1;
      for (int t = 0; t < 2 && ok; ++t) {
        if (!keys || it.count(t) == 0) continue;
        ok = mbar_wait_warp(&q_empty[t], (nq[t] & 1u) ^ 1u, p.status);
        if (!ok) break;
        ++nq[t];
        if (lead) {
          mbar_expect_tx(&q_full[t], static_cast<uint32_t>(p.per_tile * p.group) * D * 2);
#pragma unroll
          for (int c = 0; c < kSlabs; ++c)
            tma_load_3d(sQ + t * S::kBytes + c * kSlab, &p.tma_q, &q_full[t], c * 64, it.kvh * p.group,
                        it.q_begin + it.t0 + (it.shared ? 0 : t * p.per_tile));
        }
        __syncwarp();
      }
      for (int j = 0; j < n && ok; ++j, ++kv) {
        const int in = j % per_look;
        if (in == 0) {
          if (j > 0) rows = next;
          next = look(j + per_look);
        }
        const uint32_t s = kv % kStages, ph = (kv / kStages) & 1u;
        const uint32_t here = __ballot_sync(0xFFFFFFFFu, rows >= 0 && lane / boxes == in);
        const uint32_t bytes = static_cast<uint32_t>(__popc(here)) * p.box * D * 2;
        ok = mbar_wait_warp(&empty[s], ph ^ 1u, p.status);
        if (!ok) break;
        if (lead) mbar_expect_tx(&full[s], bytes);
        for (int i = 0; i < boxes; ++i) {
          const int row = __shfl_sync(0xFFFFFFFFu, rows, in * boxes + i);
          if (lead && row >= 0) {
#pragma unroll
            for (int c = 0; c < kSlabs; ++c)
              tma_load_3d(ring + s * S::kBytes + c * kSlab + i * p.box * 128, map, &full[s], c * 64, it.kvh, row);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 9) {
    // ------------------------------------ products ------------------------------------------
    const uint32_t lead = elect_one() ? 1u : 0u;
    auto commit = [&](uint64_t* bar) {
      if (kWarpIssues) tc_commit_if(lead, bar); else tc_commit(bar);
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return kWarpIssues ? mbar_wait_warp(bar, parity, p.status) : mbar_wait(bar, parity, p.status);
    };
    if (kWarpIssues || lead != 0u) {
      bool ok = true;
      uint32_t kv = 0, nq[2] = {0u, 0u}, np[2] = {0u, 0u};   // key tiles, Q tiles and P tiles so far
      for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
        CacheItem it;
        if (!it.load(p, r)) continue;
        // S_t of step j; the products execute in order, so it follows the P V that read the same columns
        auto issue_qk = [&](int t, int j) -> bool {
          const uint32_t at = kv + it.place(t, j), s = at % kStages;
          if (!wait(&k_full[s], (at / kStages) & 1u)) return false;
          tc_fence_after_sync();
          const uint32_t aQ = smem_u32(sQ + t * S::kBytes), aK = smem_u32(sK + s * S::kBytes);
          const uint32_t tS = tmem_base + static_cast<uint32_t>(t * 128);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t off = (kk / 4) * kSlab + (kk % 4) * 32;
            const uint64_t dq = make_smem_desc(aQ + off, 16, 1024), dk = make_smem_desc(aK + off, 16, 1024);
            if (kWarpIssues) tc_mma_f16_ss_if(lead, tS, dq, dk, kIdescQK, kk != 0 ? 1u : 0u);
            else tc_mma_f16_ss(tS, dq, dk, kIdescQK, kk != 0 ? 1u : 0u);
          }
          commit(&s_full[t]);
          if (j + 1 == it.count(t)) commit(&q_empty[t]);
          if (it.last_reader(t, j)) commit(&k_empty[s]);
          return true;
        };
        for (int t = 0; t < 2 && ok; ++t) {
          if (it.count(t) == 0) continue;
          ok = wait(&q_full[t], nq[t] & 1u);
          if (!ok) break;
          ++nq[t];
          ok = issue_qk(t, 0);
        }
        for (int j = 0; j < it.steps() && ok; ++j) {
          for (int t = 0; t < 2 && ok; ++t) {
            if (j >= it.count(t)) continue;
            const uint32_t at = kv + it.place(t, j), s = at % kStages;
            ok = wait(&p_full[t], np[t] & 1u);
            if (!ok) break;
            ++np[t];
            ok = wait(&v_full[s], (at / kStages) & 1u);
            if (!ok) break;
            tc_fence_after_sync();
            const uint32_t aV = smem_u32(sV + s * S::kBytes);
            const uint32_t tP = tmem_base + static_cast<uint32_t>(t * 128);
            const uint32_t tO = tmem_base + kOCol + static_cast<uint32_t>(t * 128);
#pragma unroll
            for (int kk = 0; kk < kCaTile / 16; ++kk) {
              const uint64_t dv = make_smem_desc(aV + kk * 2048, kSlab, 1024);
              if (kWarpIssues) tc_mma_f16_ts_if(lead, tO, tP + kk * 8, dv, kIdescPV, (j | kk) != 0 ? 1u : 0u);
              else tc_mma_f16_ts(tO, tP + kk * 8, dv, kIdescPV, (j | kk) != 0 ? 1u : 0u);
            }
            if (j + 1 == it.count(t)) commit(&o_full[t]);
            if (it.last_reader(t, j)) commit(&v_empty[s]);
            if (j + 1 < it.count(t)) ok = issue_qk(t, j + 1);
          }
        }
        kv += it.tiles();
      }
    }
  } else if (warp < 8) {
    // ------------------------------------ softmax / epilogue --------------------------------
    regs_take<S::kSoftmaxRegs>();
    const int t = warp >> 2;                          // query tile of this warp
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;              // row inside the tile
    const int tok = row / p.group, g = row - tok * p.group;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + static_cast<uint32_t>(t * 128);
    const uint32_t tO = tmem_base + lane_off + kOCol + static_cast<uint32_t>(t * 128);
    bool ok = true;
    uint32_t ns = 0, no0 = 0, no1 = 0, nx = 0, kv = 0;   // score tiles, finished items of the halves, shared items, key tiles so far
    for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
      CacheItem it;
      if (!it.load(p, r)) continue;
      const int n_kv = it.count(t);
      const int q_tok = it.t0 + (it.shared ? 0 : t * p.per_tile) + tok;          // token inside the sequence
      const bool valid = tok < p.per_tile && q_tok < it.q_len && (t == 0 || it.second);
      const bool live = tok < p.per_tile && q_tok < it.q_len;                    // the row of a shared tile lives in both halves
      const bool warp_live = __any_sync(0xFFFFFFFFu, live);
      // last visible key, and the window's first; rows that do not exist are not masked (nobody looks at them)
      const int hi = live ? q_tok + it.shift : 0x7FFFFFFF;
      const int low = live && p.window > 0 ? hi - p.window + 1 : 0;
      float m_used = -1.0e29f;                        // running maximum (log2 domain); above kCaMask, so masked scores give 0
      float l_sum = 0.f;
      for (int j = 0; j < n_kv && ok; ++j, ++ns) {
        ok = mbar_wait(&s_full[t], ns & 1u, p.status);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        tc_fence_after_sync();
        const int key0 = it.first_key(it.place(t, j));
        if (warp_live) {
          uint32_t sreg[128];
          {
            uint32_t(&c0)[32] = *reinterpret_cast<uint32_t(*)[32]>(&sreg[0]);
            uint32_t(&c1)[32] = *reinterpret_cast<uint32_t(*)[32]>(&sreg[32]);
            uint32_t(&c2)[32] = *reinterpret_cast<uint32_t(*)[32]>(&sreg[64]);
            uint32_t(&c3)[32] = *reinterpret_cast<uint32_t(*)[32]>(&sreg[96]);
            tmem_ld32(tS, c0);
            tmem_ld32(tS + 32, c1);
            tmem_ld32(tS + 64, c2);
            tmem_ld32(tS + 96, c3);
            tc_wait_ld();
          }
          if (__any_sync(0xFFFFFFFFu, key0 + kCaTile - 1 > hi || (key0 < low && key0 + kCaTile > p.first))) {
            // a bit for each visible key (compared one by one, with branches, a masked tile took 13000 cycles)
            const int end = hi - key0, from = low - key0, head = p.first - key0;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              auto below = [&](int n) { return n <= 32 * w ? 0u : n >= 32 * w + 32 ? 0xFFFFFFFFu : (1u << (n - 32 * w)) - 1u; };
              const uint32_t bits = (end >= 127 ? 0xFFFFFFFFu : below(end + 1)) & (~below(from) | below(head));
#pragma unroll
              for (int i = 0; i < 32; ++i) sreg[32 * w + i] = (bits >> i) & 1u ? sreg[32 * w + i] : 0xFF800000u;      // -inf: 2^(-inf) = 0
            }
          }
          float m4[4] = {kCaMask, kCaMask, kCaMask, kCaMask};
#pragma unroll
          for (int i = 0; i < 128; i += 8) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              m4[c] = max_nan(m4[c], max_nan(__uint_as_float(sreg[i + 2 * c]), __uint_as_float(sreg[i + 2 * c + 1])));
          }
          float mx = max_nan(max_nan(m4[0], m4[1]), max_nan(m4[2], m4[3]));
          mx = (mx <= 0.5f * kCaMask) ? kCaMask : mx * p.scale_log2;
          mx += mx - mx;                              // a NaN or an infinite score makes the whole row NaN
          float alpha = 1.f;
          bool rescale = false;
          if (!(mx <= m_used + kCaRescale)) {         // lazy: the reference maximum moves in large steps only
            alpha = exp2f(m_used - mx);
            m_used = mx;
            rescale = (j > 0) && live;
          }
          if (__any_sync(0xFFFFFFFFu, rescale)) {
            // O holds sums relative to the old maximum; the products that wrote it precede the scores just read
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t ov[32];
              tmem_ld32(tO + c * 32, ov);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
              tmem_st32(tO + c * 32, ov);
            }
          }
          float2 rs2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          const float2 sc2 = make_float2(p.scale_log2, p.scale_log2);
          const float2 nm2 = make_float2(-m_used, -m_used);
#pragma unroll
          for (int hlf = 0; hlf < 2; ++hlf) {
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const int at = hlf * 64 + 2 * i;
              const float2 x = __ffma2_rn(make_float2(__uint_as_float(sreg[at]), __uint_as_float(sreg[at + 1])), sc2, nm2);
              const float2 e = ex2_pair<kCaPoly, false>(at / 2, x);
              rs2[i & 1] = __fadd2_rn(rs2[i & 1], e);
              pk[i] = pack_bf16(e.x, e.y);
            }
            tmem_st32(tS + hlf * 32, pk);
          }
          tc_wait_st();
          const float2 rs = __fadd2_rn(rs2[0], rs2[1]);
          l_sum = l_sum * alpha + (rs.x + rs.y);
        }
        if (!it.whole(key0)) {                 // clear the values of keys that no row sees
          const uint32_t at = kv + it.place(t, j), s = at % kStages;
          ok = mbar_wait(&v_full[s], (at / kStages) & 1u, p.status);
          ok = __all_sync(0xFFFFFFFFu, ok);
          if (!ok) break;
          if (!it.seen(key0 + row)) {
#pragma unroll
            for (int c = 0; c < kSlabs; ++c) {
              uint4* vr = reinterpret_cast<uint4*>(sV + s * S::kBytes + c * kSlab + row * 128);
#pragma unroll
              for (int i = 0; i < 8; ++i) vr[i] = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);       // one arrival per warp
      }
      kv += it.tiles();
      // ---- epilogue ----
      const uint32_t done0 = no0 & 1u, done1 = no1 & 1u, turn = nx & 1u;
      no0 += it.n[0] > 0 ? 1u : 0u;
      no1 += it.n[1] > 0 ? 1u : 0u;
      if (it.shared) {
        ++nx;
        if (t == 1) {
          // hand this half's maxima and sums over; its O stays where it is until it has been read
          if (ok) {
            ml[row] = make_float2(m_used, l_sum);
            __syncwarp();
            if (lane == 0) mbar_arrive(ml_full);
            ok = mbar_wait(ml_empty, turn, p.status);
            ok = __all_sync(0xFFFFFFFFu, ok);
            tc_fence_after_sync();
          }
          continue;
        }
        if (ok) {
          // in this order: once the second half has handed over, its earlier items' products are known to have landed
          ok = mbar_wait(ml_full, turn, p.status) && mbar_wait(&o_full[1], done1, p.status);
          ok = __all_sync(0xFFFFFFFFu, ok);
        }
      }
      if (ok && n_kv > 0) {
        ok = mbar_wait(&o_full[t], t == 0 ? done0 : done1, p.status);
        ok = __all_sync(0xFFFFFFFFu, ok);
      }
      if (!ok) break;
      tc_fence_after_sync();
      if (warp_live) {
        float f0 = 1.f, f1 = 0.f;                     // factors of the halves' sums
        if (it.shared) {
          const float2 other = ml[row];
          const float m = max_nan(m_used, other.x);
          f0 = exp2f(m_used - m);
          f1 = exp2f(other.x - m);
          m_used = m;
          l_sum = l_sum * f0 + other.y * f1;
        }
        const int64_t at = it.q_begin + q_tok;        // row of q, when it is valid
        const int h = it.kvh * p.group + g;
        float* prow = nullptr;
        if (p.splits > 1) {
          const int64_t part = (static_cast<int64_t>(it.split) * p.total_q + at) * p.hq + h;
          prow = p.po + part * D;
          if (valid) *reinterpret_cast<float2*>(p.pml + part * 2) = make_float2(m_used, l_sum);
        } else {
          const float inv_l = (l_sum > 0.f) ? 1.f / l_sum : 0.f;
          f0 *= inv_l;
          f1 *= inv_l;
        }
        __nv_bfloat16* orow = p.o + at * p.o_ld + static_cast<int64_t>(h) * D;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {            // a loop, since short items run it once each: the code has to stay small
          uint32_t ov[32];
          if (n_kv > 0) {
            tmem_ld32(tO + c * 32, ov);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = 0u;
          }
          if (it.shared) {
            uint32_t o1[32];
            tmem_ld32(tO + 128 + c * 32, o1);
            tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f0 + __uint_as_float(o1[i]) * f1);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * f0);
          }
          if (valid && prow != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(prow + c * 32 + i * 4) = make_uint4(ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
          } else if (valid) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint4 v;
              v.x = pack_bf16(__uint_as_float(ov[8 * i + 0]), __uint_as_float(ov[8 * i + 1]));
              v.y = pack_bf16(__uint_as_float(ov[8 * i + 2]), __uint_as_float(ov[8 * i + 3]));
              v.z = pack_bf16(__uint_as_float(ov[8 * i + 4]), __uint_as_float(ov[8 * i + 5]));
              v.w = pack_bf16(__uint_as_float(ov[8 * i + 6]), __uint_as_float(ov[8 * i + 7]));
              *reinterpret_cast<uint4*>(orow + c * 32 + i * 8) = v;
            }
          }
        }
      }
      tc_fence_before_sync();                         // O is read before the next item's first P is announced
      if (it.shared) {
        __syncwarp();
        if (lane == 0) mbar_arrive(ml_empty);
      }
    }
  }

  tc_fence_before_sync();
  block_settle(p.status);
  if (warp == 9) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// Two e4m3 codes in the high bytes of the halves of t -> the bits of bf16 numbers that are 2^-120 times as large: the exponent and
// mantissa fields line up (4 + 3 bits above a bf16 mantissa's low 4), subnormal codes become bf16 subnormals.
__device__ __forceinline__ uint32_t ca_widen(uint32_t t) { return (t & 0x80008000u) | ((t >> 4) & 0x07F007F0u); }

__device__ __forceinline__ uint32_t ca_mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// 16 codes -> 16 bf16 numbers, exactly: times 2^(120 + E), E = byte - 127.  `most`: no byte of the calling warp's group of rows is
// above it.  Beyond 134 (E > 7: keys or values past 57344) bf16 has no such factor and it comes in two; 255 gives NaN.
__device__ __forceinline__ void ca_values(uint4 c, uint32_t most, uint32_t byte, uint4& lo, uint4& hi) {
  const uint32_t w[4] = {c.x, c.y, c.z, c.w};
  const uint32_t f = (most <= 134u ? (byte + 120u) << 7 : byte == 255u ? 0x7FC0u : min(byte + 120u, 254u) << 7) * 0x10001u;
  uint32_t r[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = ca_mul2(ca_widen(__byte_perm(w[i], 0, 0x1404)), f);
    r[2 * i + 1] = ca_mul2(ca_widen(__byte_perm(w[i], 0, 0x3424)), f);
  }
  if (most > 134u) {
    const uint32_t f2 = (byte == 255u ? 127u : 127u + max(byte, 134u) - 134u) * (0x10001u << 7);
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = ca_mul2(r[i], f2);
  }
  lo = make_uint4(r[0], r[1], r[2], r[3]);
  hi = make_uint4(r[4], r[5], r[6], r[7]);
}

// Keys and values that the new tokens of a sequence see, from 8-bit pages to bf16 rows [sequence, room, hk, D], see CacheRoom (what
// they do not see is left alone).  A group of D / 16 lanes per row.  Bound by bytes: 3 for each number.
template <int D>
__global__ void __launch_bounds__(256) cache_widen_kernel(const CacheWidenArgs a) {
  constexpr int kLanes = D / 16;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes, b = blockIdx.y;
  const int row = static_cast<int>(at / (2 * a.hk));
  int r = static_cast<int>(at - static_cast<int64_t>(row) * 2 * a.hk);
  const int n = a.lens[b], new_tokens = a.cu_q != nullptr ? a.cu_q[b + 1] - a.cu_q[b] : 1;
  // what is out of range is reported by the attention kernel, and read by nobody
  if (row >= a.room || row >= n || static_cast<int64_t>(n) > static_cast<int64_t>(a.table_width) * a.block || new_tokens < 0 || new_tokens > a.max_q) return;
  const int from = n - new_tokens, key = CacheRoom(from, a.window, a.first).key(row);
  if (key >= n || (a.window > 0 && key <= from - a.window && key >= a.first)) return;
  const bool val = r >= a.hk;
  if (val) r -= a.hk;
  const int bi = key / a.block, off = key - bi * a.block;
  int page = a.table[static_cast<int64_t>(b) * a.table_width + bi];
  if (page < 0 || page >= a.num_blocks) {
    if (lane == 0 && a.status != nullptr) atomicOr(a.status, kStatusIndexOutOfRange);
    page = 0;
  }
  const uint4 c = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(val ? a.v : a.k) +
                                                       ((static_cast<int64_t>(page) * a.block + off) * a.hk + r) * D) + lane);
  const uint32_t byte = __ldg(static_cast<const uint8_t*>(val ? a.v_scale : a.k_scale) + (static_cast<int64_t>(page) * a.hk + r) * a.block + off);
  uint4 lo, hi;
  ca_values(c, byte, byte, lo, hi);
  uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(val ? a.vo : a.ko) +
                                        ((static_cast<int64_t>(b) * a.room + row) * a.hk + r) * D) + 2 * lane;
  dst[0] = lo;
  dst[1] = hi;
}

// Joins the key ranges of a query head: a warp for each of the tokens x hq rows.  A range without a visible key has a sum of zero
// and is passed over (its part of po was written all the same).
template <int D>
__global__ void __launch_bounds__(128) cache_attn_merge_kernel(const CacheAttnParams p) {
  chain_next();
  chain_wait();
  const int begin = p.cu_q != nullptr ? p.cu_q[0] : p.first_row, end = p.cu_q != nullptr ? p.cu_q[p.batch] : p.first_row + p.batch;
  const int64_t row = static_cast<int64_t>(begin) * p.hq + static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (begin < 0 || row >= static_cast<int64_t>(end) * p.hq || row >= p.total_q * p.hq) return;
  const int64_t step = p.total_q * p.hq;
  float m = -1.0e29f;
  for (int s = 0; s < p.splits; ++s) m = max_nan(m, p.pml[(s * step + row) * 2]);
  constexpr int E = D / 32;
  float acc[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = *reinterpret_cast<const float2*>(p.pml + (s * step + row) * 2);
    const float f = ex2(ml.x - m);
    const float* src = p.po + (s * step + row) * D + lane * E;
    l += ml.y * f;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(src + e);
      acc[e] += v.x * f;
      acc[e + 1] += v.y * f;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.o + row / p.hq * p.o_ld + row % p.hq * D + lane * E);
#pragma unroll
  for (int e = 0; e < E; e += 2) dst[e / 2] = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
}

}  // namespace yv
