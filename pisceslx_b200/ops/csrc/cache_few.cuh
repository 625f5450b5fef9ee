// Attention of few new tokens over cached ones (sm_100a): decode steps, drafts, short turns.  The arithmetic is that of
// cache_attn.cuh; the keys are the rows of the products here, so that a tile of 128 of them meets 16, 32 or 64 (token, query head)
// rows N instead of 128, and what bounds the kernel is the bytes of keys and values:
//
//   S^T[128 keys, N]  = K[128 keys, D] Q[N, D]^T            (SS, K-major)
//   O^T[D, N]        += V[128 keys, D]^T P[N, 128 keys]^T   (SS, V as stored is MN-major)
//
// 8-bit pages: S^T takes the key codes as they are (kind::f8f6f4).  A query row is scaled by a power of two like a cached row and
// held as two e4m3 numbers, q = q1 + q2 / 16: four bits of the eight that a bf16 number has each, so the two are exact for numbers
// down to 2^-14 of the row's largest, and within 2^-22 of that one below.  They are 2 N columns of one product; a key's exponent
// and a row's are factors of the sums.  Values are widened to bf16, exactly, by four warps between the copy and the product (P has
// to keep weights of very different sizes, for which 4 bits and an exponent of e4m3 are too few).
//
// One persistent CTA per SM walks (token chunk, key head, key range, sequence) items; barriers and rings run on across items, so
// that the copies never stop.  Warps:
//   0..3   softmax: thread t owns key t of a tile (TMEM lane t of S^T) and output dimension t; the reference maximum of a row is
//          shared, moves in large steps, and the tile's threads meet at one vote on whether it has to
//   4, 5   one lane issues S^T (two tiles ahead, two buffers), one the product with the values (two P buffers)
//   6      TMA: a stage holds a tile of keys and values (and, of 8-bit pages, their exponent bytes)
//   7      rows of the next item's queries: two buffers
//   8..11  (8-bit pages) values to bf16, two buffers
#pragma once
#include "cache_attn.cuh"
#include "chain.cuh"

namespace yv {

struct CacheFewParams {
  CUtensorMap tma_k, tma_v;          // (D, key head, slot): bf16 box (64, 1, box), codes box (D, 1, box)
  const __nv_bfloat16* q;
  int64_t q_ld;
  const uint8_t *ks, *vs;
  CacheAttnParams a;                 // per_tile = tokens of a chunk, items, splits and what the sequences need
  int chunks;
};

template <int D, bool F8, int N>
struct CacheFew {
  static constexpr int kThreads = F8 ? 384 : 256;
  static constexpr int kHalf = kCaTile * D * (F8 ? 1 : 2);           // keys, or values, of a stage
  static constexpr int kStage = 2 * kHalf;                           // values, then keys
  static constexpr int kQ = 2 * N * D;                               // bf16 rows, or two rows of codes
  static constexpr int kP = N * kCaTile * 2;
  static constexpr int kWide = F8 ? kCaTile * D * 2 : 0;             // values in bf16
  static constexpr int kQBufs = N == 16 ? 2 : 1;                     // what more would take a stage away
  static constexpr int kFixed = kQBufs * kQ + 2 * (kP + kWide);
  static constexpr int kRest = 256 + 4 * 2 * kCaTile + 10 * N * 4;   // barriers, exponent bytes, row tables
  static constexpr int kMost = (227 * 1024 - 1024 - kRest - kFixed) / kStage;
  static constexpr int kStages = kMost < 4 ? kMost : 4;
  static constexpr int kTotal = kFixed + kStages * kStage + kRest + 1024;
  static constexpr uint32_t kSCols = F8 ? 2 * N : N;                 // columns of a score buffer
  static constexpr uint32_t kCols = 2 * kSCols + 2 * N <= 64 ? 64 : 2 * kSCols + 2 * N <= 128 ? 128 : 2 * kSCols + 2 * N <= 256 ? 256 : 512;
  static_assert(kStages >= 2 && kTotal <= 227 * 1024 && 2 * kSCols + 2 * N <= 512, "room");
};

struct CacheFewItem : CacheTiles {
  int b, kvh, split, t0, q_begin, q_len, shift, n;
  __device__ __forceinline__ bool load(const CacheFewParams& p, int64_t r) {
    const int64_t w = ca_item_of(r);
    if (w >= p.a.items) return false;
    // chunks of the same keys run at the same time: the second reads them from the L2
    int rest = static_cast<int>(w);
    const int chunk = rest % p.chunks;
    rest /= p.chunks;
    kvh = rest % p.a.hk;
    rest /= p.a.hk;
    split = rest % p.a.splits;
    b = rest / p.a.splits;
    int k_len;
    ca_sequence(p.a, b, q_begin, q_len, k_len);
    t0 = chunk * p.a.per_tile;
    if (t0 >= q_len) return false;
    shift = k_len - q_len;
    n = set(t0 + shift, min(t0 + p.a.per_tile, q_len) - 1 + shift, p.a.window, p.a.first, split, p.a.splits);
    n -= begin;
    return true;
  }
};

// Swizzled K-major operand whose rows are 64 bytes: groups of 8 rows are 512 bytes apart, 16-byte places are exchanged by bits 1, 2
// of the row.
__device__ __forceinline__ uint64_t make_smem_desc_rows64(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>(512 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(4) << 61;
  return d;
}

// Barrier over the 128 softmax threads with an OR of `v` (lanes that left a wait at different times are brought together first).
__device__ __forceinline__ bool few_any(bool v) {
  uint32_t any;
  __syncwarp();
  asm volatile(
      "{\n"
      ".reg .pred pin, pout;\n"
      "setp.ne.u32 pin, %1, 0;\n"
      "bar.red.or.pred pout, 1, 128, pin;\n"
      "selp.u32 %0, 1, 0, pout;\n"
      "}\n"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(v))
      : "memory");
  return any != 0u;
}

template <int D, bool F8, int N>
__global__ void __launch_bounds__(CacheFew<D, F8, N>::kThreads, 1) cache_few_kernel(const __grid_constant__ CacheFewParams fp) {
  using S = CacheFew<D, F8, N>;
  const CacheAttnParams& p = fp.a;
  constexpr int kStages = S::kStages;
  constexpr uint32_t kSlab = kCaTile * 128;                          // 128 rows x 64 columns of bf16
  constexpr uint32_t kIdescS = F8 ? make_idesc_e4m3(128, 2 * N) : make_idesc_bf16(128, N, false, false);
  constexpr uint32_t kIdescPV = make_idesc_bf16(128, N, true, false);

  extern __shared__ uint8_t cf_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(cf_raw) + 1023) & ~uintptr_t(1023));
  // At D = 64 the products with the values read a second slab of 64 rows behind the first, whose results nobody looks at: widened
  // values have the ring behind them, values of a stage its keys.
  uint8_t* sWide = smem;                                             // [2]
  uint8_t* sRing = sWide + 2 * S::kWide;
  uint8_t* sP = sRing + kStages * S::kStage;                         // [2]
  uint8_t* sQ = sP + 2 * S::kP;                                      // [kQBufs]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sQ + S::kQBufs * S::kQ);
  uint64_t* full = bars;                     // [kStages] keys, values and exponent bytes have landed
  uint64_t* empty = bars + kStages;          // [kStages]
  uint64_t* s_full = bars + 2 * kStages;     // [2]
  uint64_t* p_full = s_full + 2;             // [2] weights are stored and all scores read
  uint64_t* pv_done = p_full + 2;            // [2]
  uint64_t* v_full = pv_done + 2;            // [2] widened values
  uint64_t* q_full = v_full + 2;             // [2] query rows and their tables
  uint64_t* t_empty = q_full + 2;            // [2] tables
  uint64_t* o_empty = t_empty + 2;           // [2]
  uint64_t* q_empty = o_empty + 2;           // [kQBufs] query rows
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_empty + 2);
  uint8_t* sByte = reinterpret_cast<uint8_t*>(bars) + 256;                               // [kStages][2][128]
  int* sHi = reinterpret_cast<int*>(sByte + kStages * 2 * kCaTile);                      // [2][N] last visible key of a row, -1 = none
  float* sFactor = reinterpret_cast<float*>(sHi + 2 * N);                                // [2][N] a row's power of two times the scale
  float* sM = sFactor + 2 * N;                                                           // [N] reference maxima
  float* sMax = sM + N;                                                                  // [N] new ones
  float* sRed = sMax + N;                                                                // [4][N]

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
  if (tid == 0) {
    tma_prefetch_desc(&fp.tma_k);
    tma_prefetch_desc(&fp.tma_v);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], F8 ? 9 : 1);      // 8 bits: the score product, four softmax warps, four widening ones; else the P V product
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&q_full[i], 1);
      mbar_init(&t_empty[i], 4);
      mbar_init(&q_empty[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, S::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  // the tensor memory is this kernel's before the next one may begin
  chain_next();
  chain_wait();
  if (p.zero_rest != 0) {                                            // rows that belong to no sequence
    const int64_t used = p.cu_q != nullptr ? p.cu_q[p.batch] : p.batch, vecs = static_cast<int64_t>(p.hq) * D / 8;
    for (int64_t i = (used < 0 ? 0 : used) * vecs + static_cast<int64_t>(blockIdx.x) * S::kThreads + tid; i < p.total_q * vecs;
         i += static_cast<int64_t>(gridDim.x) * S::kThreads)
      *reinterpret_cast<uint4*>(p.o + i / vecs * p.o_ld + i % vecs * 8) = make_uint4(0, 0, 0, 0);
  }

  auto stage_v = [&](uint32_t s) { return sRing + s * S::kStage; };
  auto stage_k = [&](uint32_t s) { return sRing + s * S::kStage + S::kHalf; };
  const uint32_t tO = tmem_base + 2 * S::kSCols;                     // two buffers of N columns behind the scores'

  if (warp == 6) {
    // ------------------------------------ copies --------------------------------------------
    const uint32_t lead = elect_one() ? 1u : 0u;
    const int boxes = kCaTile / p.box, per_look = 32 / boxes;
    uint32_t g = 0;                                                  // tiles so far
    bool ok = true;
    for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
      CacheFewItem it;
      if (!it.load(fp, r)) continue;
      // slot of copy `lane` of the tiles from j0 on; negative where no key of it is seen
      auto look = [&](int j0) {
        const int j = j0 + lane / boxes;
        if (j >= it.n) return -1;
        const int key = it.first_key(j) + (lane % boxes) * p.box;
        return it.any(key, p.box) ? ca_slot(p, it.b, key) : -1;
      };
      int rows = look(0), next = -1;
      for (int j = 0; j < it.n && ok; ++j, ++g) {
        const int in = j % per_look;
        if (in == 0) {
          if (j > 0) rows = next;
          next = look(j + per_look);
        }
        const uint32_t s = g % kStages;
        const uint32_t here = __ballot_sync(0xFFFFFFFFu, rows >= 0 && lane / boxes == in);
        ok = mbar_wait_warp(&empty[s], ((g / kStages) & 1u) ^ 1u, p.status);
        if (!ok) break;
        if (lead) mbar_expect_tx(&full[s], static_cast<uint32_t>(__popc(here)) * p.box * (F8 ? 2 * D + 2 : 4 * D));
        for (int i = 0; i < boxes; ++i) {
          const int row = __shfl_sync(0xFFFFFFFFu, rows, in * boxes + i);
          if (!lead || row < 0) continue;
          if constexpr (F8) {
            tma_load_3d(stage_k(s) + i * p.box * D, &fp.tma_k, &full[s], 0, it.kvh, row);
            tma_load_3d(stage_v(s) + i * p.box * D, &fp.tma_v, &full[s], 0, it.kvh, row);
            const int page = row / p.block;
            const int64_t at = (static_cast<int64_t>(page) * p.hk + it.kvh) * p.block + (row - page * p.block);
            bulk_load_1d(sByte + s * 2 * kCaTile + i * p.box, fp.ks + at, p.box, &full[s]);
            bulk_load_1d(sByte + s * 2 * kCaTile + kCaTile + i * p.box, fp.vs + at, p.box, &full[s]);
          } else {
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_3d(stage_k(s) + c * kSlab + i * p.box * 128, &fp.tma_k, &full[s], c * 64, it.kvh, row);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) tma_load_3d(stage_v(s) + c * kSlab + i * p.box * 128, &fp.tma_v, &full[s], c * 64, it.kvh, row);
          }
        }
        __syncwarp();
      }
    }
  } else if (warp == 7) {
    // ------------------------------------ query rows ----------------------------------------
    uint32_t items = 0;
    bool ok = true;
    for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
      CacheFewItem it;
      if (!it.load(fp, r)) continue;
      if (it.n == 0) continue;
      const uint32_t tb = items & 1u, qb = items % S::kQBufs;
      ok = mbar_wait_warp(&q_empty[qb], ((items / S::kQBufs) & 1u) ^ 1u, p.status) &&
           mbar_wait_warp(&t_empty[tb], ((items >> 1) & 1u) ^ 1u, p.status);
      if (!ok) break;
      ++items;
      constexpr int E = D / 32;                                      // numbers of a lane
      uint8_t* dst = sQ + qb * S::kQ;
#pragma unroll 8
      for (int i = 0; i < N; ++i) {
        const int tok = i / p.group, h = i - tok * p.group;
        const bool there = tok < p.per_tile && it.t0 + tok < it.q_len;
        uint32_t w[E / 2];
#pragma unroll
        for (int e = 0; e < E / 2; ++e) w[e] = 0;
        if (there) {
          const __nv_bfloat16* src = fp.q + static_cast<int64_t>(it.q_begin + it.t0 + tok) * fp.q_ld +
                                     static_cast<int64_t>(it.kvh * p.group + h) * D + lane * E;
          if constexpr (E == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            w[0] = x.x;
            w[1] = x.y;
          } else {
            w[0] = *reinterpret_cast<const uint32_t*>(src);
          }
        }
        float factor = p.scale_log2;
        if constexpr (F8) {
          uint32_t top = 0;
#pragma unroll
          for (int e = 0; e < E / 2; ++e) top = max(top, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));
          top = __reduce_max_sync(0xFFFFFFFFu, top);
          const bool finite = top < 0x7F80u;
          const int byte = finite ? max(0, static_cast<int>(top >> 7) - 8 + ((top & 0x7Fu) > 0x60u ? 1 : 0)) : 127;
          const float inv = __int_as_float((254 - byte) << 23);      // 2^-E
          factor = finite ? factor * (byte == 0 ? __int_as_float(0x00400000) : __int_as_float(byte << 23)) : __int_as_float(0x7FC00000);
          uint32_t c1 = 0, c2 = 0;
#pragma unroll
          for (int e = 0; e < E / 2; ++e) {
            const float2 x = make_float2(__uint_as_float(w[e] << 16) * inv, __uint_as_float(w[e] & 0xFFFF0000u) * inv);
            const __nv_fp8x2_storage_t a = __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3);
            const float2 y = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(a, __NV_E4M3)));
            const __nv_fp8x2_storage_t b =
                __nv_cvt_float2_to_fp8x2(make_float2((x.x - y.x) * 16.f, (x.y - y.y) * 16.f), __NV_SATFINITE, __NV_E4M3);
            c1 |= static_cast<uint32_t>(a) << (16 * e);
            c2 |= static_cast<uint32_t>(b) << (16 * e);
          }
          if (!finite) c1 = c2 = 0;
          // rows i and N + i
          if constexpr (D == 128) {
            const uint32_t at = ((((lane >> 2) ^ (i & 7)) << 4) | ((lane & 3) << 2));
            *reinterpret_cast<uint32_t*>(dst + i * 128 + at) = c1;
            *reinterpret_cast<uint32_t*>(dst + (N + i) * 128 + at) = c2;
          } else {
            const uint32_t at = ((((lane >> 3) ^ ((i >> 1) & 3)) << 4) | ((lane & 7) << 1));
            *reinterpret_cast<uint16_t*>(dst + i * 64 + at) = static_cast<uint16_t>(c1);
            *reinterpret_cast<uint16_t*>(dst + (N + i) * 64 + at) = static_cast<uint16_t>(c2);
          }
        } else if constexpr (E == 4) {
          const int c = lane >> 1;
          *reinterpret_cast<uint2*>(dst + (c >> 3) * (N * 128) + i * 128 + (((c & 7) ^ (i & 7)) << 4) + ((lane & 1) << 3)) = make_uint2(w[0], w[1]);
        } else {
          *reinterpret_cast<uint32_t*>(dst + i * 128 + (((lane >> 2) ^ (i & 7)) << 4) + ((lane & 3) << 2)) = w[0];
        }
        if (lane == 0) {
          sHi[tb * N + i] = there ? it.t0 + tok + it.shift : -1;
          sFactor[tb * N + i] = factor;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[tb]);
    }
  } else if (warp == 4) {
    // ------------------------------------ scores --------------------------------------------
    if (elect_one()) {
      uint32_t g = 0, items = 0;
      bool ok = true;
      for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
        CacheFewItem it;
        if (!it.load(fp, r) || it.n == 0) continue;
        const uint32_t qb = items % S::kQBufs;
        ok = mbar_wait(&q_full[items & 1u], (items >> 1) & 1u, p.status);
        ++items;
        const uint32_t aQ = smem_u32(sQ + qb * S::kQ);
        for (int j = 0; j < it.n && ok; ++j, ++g) {
          const uint32_t s = g % kStages, sb = g & 1u;
          // the buffer's scores, of tile g - 2, have been read
          ok = mbar_wait(&full[s], (g / kStages) & 1u, p.status) && (g < 2 || mbar_wait(&p_full[sb], ((g >> 1) & 1u) ^ 1u, p.status));
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t aK = smem_u32(stage_k(s)), tS = tmem_base + sb * S::kSCols;
          if constexpr (F8) {
#pragma unroll
            for (int kk = 0; kk < D / 32; ++kk) {
              if constexpr (D == 128)
                tc_mma_f8_ss(tS, make_smem_desc(aK + kk * 32, 16, 1024), make_smem_desc(aQ + kk * 32, 16, 1024), kIdescS, kk != 0 ? 1u : 0u);
              else
                tc_mma_f8_ss(tS, make_smem_desc_rows64(aK + kk * 32), make_smem_desc_rows64(aQ + kk * 32), kIdescS, kk != 0 ? 1u : 0u);
            }
          } else {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              tc_mma_f16_ss(tS, make_smem_desc(aK + (kk / 4) * kSlab + (kk % 4) * 32, 16, 1024),
                            make_smem_desc(aQ + (kk / 4) * (N * 128) + (kk % 4) * 32, 16, 1024), kIdescS, kk != 0 ? 1u : 0u);
          }
          tc_commit(&s_full[sb]);
          if (F8) tc_commit(&empty[s]);
          if (j + 1 == it.n) tc_commit(&q_empty[qb]);
        }
      }
    }
  } else if (warp == 5) {
    // ------------------------------------ weights times values ------------------------------
    if (elect_one()) {
      uint32_t g = 0, items = 0;
      bool ok = true;
      for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
        CacheFewItem it;
        if (!it.load(fp, r) || it.n == 0) continue;
        const uint32_t ob = items & 1u;
        ok = mbar_wait(&o_empty[ob], ((items >> 1) & 1u) ^ 1u, p.status);
        ++items;
        for (int j = 0; j < it.n && ok; ++j, ++g) {
          const uint32_t s = g % kStages, pb = g & 1u, ph = (g >> 1) & 1u;
          ok = (F8 ? mbar_wait(&v_full[pb], ph, p.status) : mbar_wait(&full[s], (g / kStages) & 1u, p.status)) &&
               mbar_wait(&p_full[pb], ph, p.status);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t aV = F8 ? smem_u32(sWide + pb * S::kWide) : smem_u32(stage_v(s)), aP = smem_u32(sP + pb * S::kP);
#pragma unroll
          for (int kk = 0; kk < kCaTile / 16; ++kk)
            tc_mma_f16_ss(tO + ob * N, make_smem_desc(aV + kk * 2048, kSlab, 1024),
                          make_smem_desc(aP + (kk / 4) * (N * 128) + (kk % 4) * 32, 16, 1024), kIdescPV, (j | kk) != 0 ? 1u : 0u);
          tc_commit(&pv_done[pb]);
          if (!F8) tc_commit(&empty[s]);
        }
      }
    }
  } else if (F8 && warp >= 8) {
    // ------------------------------------ values to bf16 ------------------------------------
    constexpr int kLanes = D / 16;                                   // lanes of a row, 16 codes each
    constexpr int kStep = 128 / kLanes;
    const int c = (tid - 256) % kLanes, row0 = (tid - 256) / kLanes;
    // 16 codes fill two 16-byte places of a swizzled row.  Where 8 lanes work on one row, those of the second slab start with the
    // odd place: the 8 stores then meet 8 different groups of banks.
    const bool odd_first = D == 128 && c >= 4;
    uint32_t g = 0;
    bool ok = true;
    for (int64_t r = 0; r * gridDim.x < p.items && ok; ++r) {
      CacheFewItem it;
      if (!it.load(fp, r)) continue;
      for (int j = 0; j < it.n && ok; ++j, ++g) {
        const uint32_t s = g % kStages, vb = g & 1u;
        const int key0 = it.first_key(j);
        ok = mbar_wait_warp(&full[s], (g / kStages) & 1u, p.status) &&
             (g < 2 || mbar_wait_warp(&pv_done[vb], ((g >> 1) & 1u) ^ 1u, p.status));
        if (!ok) break;
        const uint8_t* src = stage_v(s);
        const uint8_t* bytes = sByte + s * 2 * kCaTile + kCaTile;
        uint8_t* dst = sWide + vb * S::kWide + (c / 4) * kSlab;
#pragma unroll 4
        for (int row = row0; row < kCaTile; row += kStep) {
          uint4 a = make_uint4(0, 0, 0, 0), b = make_uint4(0, 0, 0, 0);
          if (it.seen(key0 + row))
            ca_values(*reinterpret_cast<const uint4*>(src + row * D + c * 16), ca_factors(bytes[row]), a, b);
          uint8_t* at = dst + row * 128;
          const int w = (2 * c) & 7, x = row & 7;
          *reinterpret_cast<uint4*>(at + (((w + (odd_first ? 1 : 0)) ^ x) << 4)) = odd_first ? b : a;
          *reinterpret_cast<uint4*>(at + (((w + (odd_first ? 0 : 1)) ^ x) << 4)) = odd_first ? a : b;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&v_full[vb]);
          mbar_arrive(&empty[s]);
        }
      }
    }
  } else if (warp < 4) {
    // ------------------------------------ softmax -------------------------------------------
    const uint32_t lane_off = static_cast<uint32_t>(warp * 32) << 16;
    uint32_t g = 0, items = 0;
    bool ok = true;
    for (int64_t r = 0; r * gridDim.x < p.items; ++r) {
      CacheFewItem it;
      if (!it.load(fp, r)) continue;
      const uint32_t tb = items & 1u;
      float l[N];
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = 0.f;
      if (it.n > 0) {
        ++items;
        if (tid < N) sM[tid] = -1.0e29f;
        ok = mbar_wait(&q_full[tb], ((items - 1) >> 1) & 1u, p.status);
        ok = !few_any(!ok);                                          // the maxima are set; all agree on whether a wait ran out
        if (!ok) break;
      }
      // rows are masked one by one only where some row does not see the whole tile
      const int hi_least = it.t0 + it.shift, hi_most = min(it.t0 + p.per_tile, it.q_len) - 1 + it.shift;
      // a warp whose wait ran out walks on, without waiting, to the next vote; all leave there together
      for (int j = 0; j < it.n; ++j, ++g) {
        const uint32_t s = g % kStages, sb = g & 1u, ph = (g >> 1) & 1u;
        const int key0 = it.first_key(j), key = key0 + tid;
        const bool seen = it.seen(key);
        const bool all = key0 + kCaTile - 1 <= hi_least &&
                         (p.window == 0 || key0 > hi_most - p.window || key0 + kCaTile <= p.first);
        ok = ok && mbar_wait(&s_full[sb], ph, p.status);
        if (F8 || !it.whole(key0)) ok = ok && mbar_wait(&full[s], (g / kStages) & 1u, p.status);
        ok = __all_sync(0xFFFFFFFFu, ok);                            // the aligned tcgen05 instructions need a converged warp
        float kf = p.scale_log2;
        if (F8 && ok) {
          const uint32_t byte = sByte[s * 2 * kCaTile + tid];
          kf = byte == 255u ? __int_as_float(0x7FC00000) : byte == 0u ? __int_as_float(0x00400000) : __int_as_float(static_cast<int>(byte) << 23);
        }
        float sc[N];
        bool high = false;
        if (ok) {
          tc_fence_after_sync();
          const uint32_t tS = tmem_base + lane_off + sb * S::kSCols;
#pragma unroll
          for (int n0 = 0; n0 < N; n0 += 16) {
            uint32_t a[16];
            tmem_ld16(tS + n0, a);
            if constexpr (F8) {
              uint32_t b[16];
              tmem_ld16(tS + N + n0, b);
              float f[16];
#pragma unroll
              for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(f + i) = *reinterpret_cast<const float4*>(sFactor + tb * N + n0 + i);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                sc[n0 + i] = fmaf(__uint_as_float(b[i]), 0.0625f, __uint_as_float(a[i])) * (kf * f[i]);
            } else {
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) sc[n0 + i] = __uint_as_float(a[i]) * kf;
            }
          }
          if (!all || !seen) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              const int hi = sHi[tb * N + i];
              const bool mine = seen && key <= hi && (p.window == 0 || key > hi - p.window || key < p.first);
              if (!mine) sc[i] = kCaMask;
            }
          }
#pragma unroll
          for (int i = 0; i < N; i += 4) {
            const float4 m = *reinterpret_cast<const float4*>(sM + i);
            high |= !(sc[i] <= m.x + kCaRescale) || !(sc[i + 1] <= m.y + kCaRescale) || !(sc[i + 2] <= m.z + kCaRescale) ||
                    !(sc[i + 3] <= m.w + kCaRescale);
          }
        }
        tc_fence_before_sync();
        // lazy: a reference maximum moves only when a score exceeds it by more than 2^8 (or is NaN)
        if (few_any(high || !ok)) {
          if (ok) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
              float v = sc[i];
#pragma unroll
              for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
              if (lane == 0) sRed[warp * N + i] = v;
            }
          }
          ok = !few_any(!ok);
          if (!ok) break;
          if (tid < N) {
            const float top = max_nan(max_nan(sRed[tid], sRed[N + tid]), max_nan(sRed[2 * N + tid], sRed[3 * N + tid]));
            sMax[tid] = !(top <= sM[tid] + kCaRescale) ? top : sM[tid];
          }
          // the products so far have landed
          if (j > 0) ok = mbar_wait(&pv_done[(g - 1) & 1u], ((g - 1) >> 1) & 1u, p.status);
          ok = !few_any(!ok);
          if (!ok) break;
          tc_fence_after_sync();
#pragma unroll
          for (int n0 = 0; n0 < N; n0 += 16) {
            uint32_t o[16];
            if (j > 0) {
              tmem_ld16(tO + lane_off + ((items - 1) & 1u) * N + n0, o);
              tc_wait_ld();
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float alpha = ex2(sM[n0 + i] - sMax[n0 + i]);
              l[n0 + i] *= alpha;
              if (j > 0) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            }
            if (j > 0) {
              tmem_st16(tO + lane_off + ((items - 1) & 1u) * N + n0, o);
              tc_wait_st();
            }
          }
          tc_fence_before_sync();
          few_any(false);                                            // everyone has read the old maxima
          if (tid < N) sM[tid] = sMax[tid];
          few_any(false);
        }
        if (g >= 2) {                                                // this P buffer was read by the product of tile g - 2
          ok = ok && mbar_wait(&pv_done[sb], ph ^ 1u, p.status);
          ok = __all_sync(0xFFFFFFFFu, ok);
        }
        if (ok) {
          uint8_t* sp = sP + sb * S::kP + (tid >> 6) * (N * 128) + ((tid & 7) << 1);
#pragma unroll
          for (int i0 = 0; i0 < N; i0 += 4) {
            float m[4];
            *reinterpret_cast<float4*>(m) = *reinterpret_cast<const float4*>(sM + i0);
#pragma unroll
            for (int i = i0; i < i0 + 4; ++i) {
              const __nv_bfloat16 w = __float2bfloat16(ex2(sc[i] - m[i - i0]));          // masked: 2^(-1e30 - m) = 0
              *reinterpret_cast<__nv_bfloat16*>(sp + i * 128 + ((((tid & 63) >> 3) ^ (i & 7)) << 4)) = w;
              l[i] += __bfloat162float(w);           // the sum takes the rounded weights that the tensor core multiplies
            }
          }
          if (!F8 && !it.whole(key0)) {
            if (!seen) {                             // values that no row sees are cleared (0 * NaN would be NaN)
#pragma unroll
              for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) reinterpret_cast<uint4*>(stage_v(s) + c * kSlab + tid * 128)[i] = make_uint4(0, 0, 0, 0);
            }
          }
          fence_proxy_async_smem();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&p_full[sb]);
            if (F8) mbar_arrive(&empty[s]);
          }
        }
      }
      if (it.n > 0) {
        if (ok) ok = mbar_wait(&pv_done[(g - 1) & 1u], ((g - 1) >> 1) & 1u, p.status);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          float v = l[i];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
          if (lane == 0) sRed[warp * N + i] = v;
        }
        ok = !few_any(!ok);
        if (!ok) break;                              // a wait ran out (the status word says so): the outputs are not written
        tc_fence_after_sync();
      }
      const int64_t step = p.total_q * p.hq;
#pragma unroll 1
      for (int n0 = 0; n0 < N; n0 += 16) {
        uint32_t o[16];
        if (it.n > 0) {
          tmem_ld16(tO + lane_off + ((items - 1) & 1u) * N + n0, o);
          tc_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int row = n0 + i, tok = row / p.group, h = row - tok * p.group;
          if (tok >= p.per_tile || it.t0 + tok >= it.q_len) continue;
          const int64_t at = it.q_begin + it.t0 + tok;
          const int head = it.kvh * p.group + h;
          const float sum = it.n > 0 ? sRed[row] + sRed[N + row] + sRed[2 * N + row] + sRed[3 * N + row] : 0.f;
          if (p.splits > 1) {
            const int64_t part = it.split * step + at * p.hq + head;
            if (tid < D) p.po[part * D + tid] = __uint_as_float(o[i]);
            if (tid == 0) *reinterpret_cast<float2*>(p.pml + part * 2) = make_float2(it.n > 0 ? sM[row] : -1.0e29f, sum);
          } else if (tid < D) {
            p.o[at * p.o_ld + static_cast<int64_t>(head) * D + tid] = __float2bfloat16(sum > 0.f ? __uint_as_float(o[i]) / sum : __uint_as_float(o[i]) * 0.f);
          }
        }
      }
      if (it.n > 0) {
        tc_fence_before_sync();
        few_any(false);                              // sRed, sM and the row tables have been read
        if (lane == 0) {
          mbar_arrive(&o_empty[(items - 1) & 1u]);
          mbar_arrive(&t_empty[tb]);
        }
      }
    }
  }

  tc_fence_before_sync();
  block_settle(p.status);                            // begins with a barrier
  if (warp == 0) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, S::kCols);
  }
}

}  // namespace yv
