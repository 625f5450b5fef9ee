// Attention of few new tokens over cached ones (sm_100a): decode steps, drafts, short turns.  The arithmetic is that of
// cache_attn.cuh; the keys are the rows of the products here, so that a tile of 128 of them meets R = 4 to 64 (token, query head)
// rows, N = max(R, 16) columns, instead of 128 (of bf16 pages up to 16 rows: see few_rows in cache.cu).  Few rows are bounded by the
// bytes of keys and values; from some 16 rows on by the chain from a tile's scores to its product with the values:
//
//   S^T[128 keys, N]  = K[128 keys, D] Q[N, D]^T            (SS, K-major)
//   O^T[D, N]        += V[128 keys, D]^T P[128 keys, N]     (SS; V as stored and P as a key's thread writes it are MN-major)
//
// 8-bit pages: S^T takes the key codes as they are (kind::f8f6f4).  A query row is scaled by a power of two like a cached row and
// held as two e4m3 numbers, q = q1 + q2 / 16: four bits of the eight that a bf16 number has each, so the two are exact for numbers
// down to 2^-14 of the row's largest, and within 2^-22 of that one below.  They are 2 N columns of one product; a key's exponent
// and a row's are factors of the sums.  Value codes are widened to fp16, which holds them all, by four warps between the copy and
// the product (one conversion for two codes; to bf16, with the exponent in it, took five operations and bounded the kernel); their
// exponents go into the weights, fp16 too: w = p 2^(E - Eref + 4) with a reference Eref at least E - 3, at most 2^15.  fp16 keeps 11
// bits of weights down to 2^-18 of the largest, and is off by 2^-29 of that below.  The largest may carry no weight for a row (its key is
// hidden from it, or unlikely), so this is for value rows of about one size: once the exponents that an item has met are kFewSpread
// apart, its tiles go as bf16, weights and values, with 8 bits of each weight as far as sums in 32 bits reach.
//
// The key tiles of all sequences and key heads form one line, which is cut into equal pieces, two for every SM: the kernel ends
// everywhere at the same time whatever the lengths are, and nothing but the lengths on the device decides.  A (sequence, head) that
// lies in one piece is finished there; one that is cut leaves its unnormalised sums, at most two such parts a piece, to a
// second kernel.  A CTA works on its two pieces tile by tile in turn, with a group of softmax warps for each, so that the
// copies go on while one of them ends an item.  Warps:
//   0..3, 4..7  softmax of a piece: thread t owns key t of a tile (TMEM lane t of S^T) and output dimension t; a row's reference
//               maximum is shared and moves in large steps, and the group meets at one vote a tile on whether it has to
//   8           one lane issues the products: of a tile with the values, then the scores of the piece's next tile
//   9           rows of the next items' queries (and, of 8 bits and up to 16 rows, their codes)
//   10, 11      TMA, a piece each: a stage holds a tile of keys and values (and, of 8-bit pages, their exponent bytes), and what the
//               other warps have to know of it
//   12..15      (8-bit pages) values to fp16
// Only warps 9 to 11 walk the line, and all loops are short: 16 warps in six roles share an instruction cache.  With a walk of both
// pieces in each of them a third of all stalls was for instructions and an 8-bit tile took 1.5 to 1.8 us; with one warp that
// copied for both pieces, 1.2.  For the same reason 16 rows at a time go through a loop that is not unrolled: with all 64 of a tile
// unrolled, in registers, what is done once an item cost more than its tiles (18 sequences of 2048 tokens, 16 new ones: 270 us;
// 16 of them take 59 in loops).
//
// 8-bit pages, 32 query heads over 8 of 128: 64 sequences of 2048 to 4096 tokens, a new one each, 95 us (4.2 TB/s of codes, 64 % of the
// measured copy rate; a tile takes an SM 0.85 us, its bytes 0.75); 8 of up to 8192 with 5 new ones 53 us (15.5 for the bytes; a tile 1.4
// us, 1.75 with 16 new ones).  Of each call 12 us or so are the beginning, the last parts and the join.  Scores of a piece's next tile
// ahead of a product with the values, in a second buffer, made it slower (one new token 1.11 us a tile for 0.83, four 1.41 for
// 1.04), and so did, from 32 rows on, loads of the next 16 rows' scores in front of the weights of these (2 to 5 %).
#pragma once
#include "cache_attn.cuh"
#include "chain.cuh"

namespace yv {

struct CacheFewParams {
  CUtensorMap tma_k, tma_v;          // (D, key head, slot): bf16 box (64, 1, box), codes box (D, 1, box)
  CUtensorMap tma_q;                 // (D, query head, token): box (64, G, R / G), for 8-bit pages (D, G, R / G) as it lies
  const uint8_t *ks, *vs;
  CacheAttnParams a;                 // po, pml: [piece][2][R][D] and [piece][2][R][2]
  int* pre;                          // [batch + 1] tiles in front of every sequence, for the second kernel
};
constexpr int kFewSequences = 512;   // of one launch
constexpr int kFewLeast = 2;         // tiles of a piece where SMs have one: below, more pieces cost more than they save
constexpr int kFewTwo = 4;           // tiles of a piece from which SMs have two

template <int D, bool F8, int R>
struct CacheFew {
  static constexpr int kN = R < 16 ? 16 : R;
  static constexpr int kThreads = F8 ? 512 : 384;
  static constexpr int kHalf = kCaTile * D * (F8 ? 1 : 2);           // keys, or values, of a stage
  static constexpr int kStage = 2 * kHalf;                           // values, then keys
  static constexpr int kQ = 2 * kN * D;                              // bf16 rows, or two rows of codes
  static constexpr int kP = kN * kCaTile * 2;
  static constexpr int kWide = F8 ? kCaTile * D * 2 : 0;             // values in fp16
  static constexpr int kRaw = F8 ? R * D * 2 : 0;                    // query rows before they become codes
  static constexpr int kFixed = 2 * (kQ + kP + kWide) + kRaw;        // each of the two pieces has its own
  static constexpr int kRest = 256 + 4 * (2 * kCaTile + 32) + 30 * kN * 4 + 128 + 13 * kFewSequences + 64;   // barriers, exponent bytes, tables
  static constexpr int kMost = (227 * 1024 - 1024 - kRest - kFixed) / kStage;
  static constexpr int kStages = kMost < 4 ? kMost : 4;
  // 8-bit stages are given back as soon as their keys are multiplied and the rest is read, where a piece's tiles keep to stages of
  // their own (an even number); else, in the order of the ring, by the product with the values.  A copying warp that waits for a
  // stage must not see it given back a turn too early.
  static constexpr bool kEarly = F8 && kStages % 2 == 0;
  // From 32 rows on the softmax warps make codes of their own item's query rows: one warp that does it for both pieces takes 8000
  // cycles for 64 rows, and an item's first scores wait for it.  Of few rows it is done ahead.
  static constexpr bool kOwnRows = F8 && R >= 32;
  static constexpr int kTotal = kFixed + kStages * kStage + kRest + 1024;
  static constexpr uint32_t kSCols = F8 ? 2 * kN : kN;               // columns of a score buffer
  static constexpr uint32_t kUsed = 2 * kSCols + 2 * kN;             // scores and sums of two pieces
  static constexpr uint32_t kCols = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
  static_assert(kStages >= 2 && kTotal <= 227 * 1024 && kUsed <= 512, "room");
};

// The line in n pieces: the first `more` have a tile more than the others (32-bit arithmetic and one division: every warp asks
// before it can begin).
struct CacheFewCuts {
  int each, more, n;
  __device__ __forceinline__ CacheFewCuts(int all, int n_) : each(all / n_), more(all - all / n_ * n_), n(n_) {}
  __device__ __forceinline__ int cut(int c) const { return c < n ? each * c + min(c, more) : each * n + more; }    // places in front of piece c
  __device__ __forceinline__ int tiles(int c) const { return c < n ? each + (c < more ? 1 : 0) : 0; }
  __device__ __forceinline__ int piece(int x) const {
    const int longer = (each + 1) * more;
    return x < longer ? x / (each + 1) : more + (x - longer) / each;
  }
};
__device__ __forceinline__ int few_pieces(int all, int ctas) {
  return all >= 2 * kFewTwo * ctas ? 2 * ctas : max(1, min(ctas, all / kFewLeast));
}

// What the roles know of the sequences, in shared memory.
struct CacheFewTable {
  int *pre, *q0, *len;               // [batch + 1] tiles of one head in front of a sequence, first row of q, cached tokens
  uint8_t* q_len;
};

// A walk along a piece [at, end) of the line: sequence by sequence, head by head.  A sequence whose tokens see nothing has one
// tile, of which nothing is seen.
struct CacheFewItem : CacheTiles {
  int at, start, end;                // place on the line; first and last place of the piece
  int b, kvh, q_begin, q_len, shift, n;
  int slot;                          // -1: whole, else which of the piece's parts

  __device__ __forceinline__ void begin_walk(const CacheAttnParams& p, const CacheFewTable& t, const CacheFewCuts& cuts, int piece) {
    start = at = cuts.cut(piece);
    end = start + cuts.tiles(piece);
    int low = 0, high = p.batch;     // the last sequence with pre <= at / hk
    while (high - low > 1) {
      const int mid = (low + high) / 2;
      if (t.pre[mid] * p.hk <= at) low = mid; else high = mid;
    }
    b = low;
  }
  __device__ __forceinline__ bool next(const CacheAttnParams& p, const CacheFewTable& t) {
    if (at >= end) return false;
    while (at >= t.pre[b + 1] * p.hk) ++b;
    const int tiles = t.pre[b + 1] - t.pre[b], place = at - t.pre[b] * p.hk;
    kvh = place / tiles;
    const int from = place - kvh * tiles;
    n = min(tiles - from, end - at);
    slot = n == tiles ? -1 : at == start ? 0 : 1;
    at += n;
    q_begin = t.q0[b];
    q_len = t.q_len[b];
    shift = t.len[b] - q_len;
    set(shift, q_len - 1 + shift, p.window, p.first, 0, 1);
    begin = from;
    return true;
  }
};

// What a copying warp says of the tile in a stage.
struct alignas(16) CacheFewTile {
  int key, flags, lo, last, first_end, pad[3];
  __device__ __forceinline__ bool seen(int k) const { return k <= last && (k >= lo || k < first_end); }
};
// Exponents of an item's seen values that fp16 weights hold: w = p 2^(E - Eref + 4) is off by 2^-25 where it is below 2^-14, and the
// largest of a row is 2^(4 - kFewSpread) at least.  That is 2^-22 of it for each key, at worst as far as one bf16 weight for
// 8192 keys that are all rounded alike.
constexpr int kFewSpread = 7;
// What bf16 values are held by: e4m3 codes keep their 3 bits of mantissa where they are in fp16, moved to bf16's place.
constexpr int kFewWidePower = 112;
enum : int {
  kFewGroup = 1,                     // the piece
  kFewFirst = 2, kFewLast = 4,       // of its item
  kFewWhole = 8,                     // some row sees each key
  kFewAll = 16,                      // every row sees every key
};

// A wait of few instructions (they are inlined in many places); the same limit as mbar_wait's.
__device__ __forceinline__ bool few_wait(uint64_t* bar, uint32_t parity, uint32_t* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 0; !mbar_try_wait(bar, parity); ++i) {
    if ((i & 0xFFu) != 0u) continue;
    const uint64_t now = globaltimer_ns();
    if (i == 0) t0 = now;
    else if (gave_up(status)) return false;
    else if (now - t0 > YV_WAIT_LIMIT_NS) {
      if (status != nullptr) atomicOr(status, kStatusWaitTimeout);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool few_wait_warp(uint64_t* bar, uint32_t parity, uint32_t* status) {
  return __all_sync(0xFFFFFFFFu, few_wait(bar, parity, status)) != 0;
}

// Place in the ring of tile k of a piece: the pieces take stages in turn, as long as both have tiles.
__device__ __forceinline__ uint32_t few_turn(uint32_t k, uint32_t group, uint32_t others) { return k + min(k + group, others); }

// Descriptor of a swizzled operand: rows of `bytes` 32, 64 or 128, groups of 8 rows one after the other (modes 6, 4, 2).  K-major
// rows hold consecutive k, MN-major ones consecutive columns of one k.  Within a row the 16-byte places are exchanged by the
// row's number: few_place.
template <int BYTES>
__device__ __forceinline__ uint64_t few_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>((8 * BYTES) >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(BYTES == 128 ? 2 : BYTES == 64 ? 4 : 6) << 61;
  return d;
}
template <int BYTES>
__device__ __forceinline__ int few_place(int row, int place) {
  return BYTES == 128 ? place ^ (row & 7) : BYTES == 64 ? place ^ ((row >> 1) & 3) : place ^ ((row >> 2) & 1);
}

// v[i] of all lanes joined: a lane's result is that of row lane / (32 / C).  Every step halves the rows that a lane holds.
template <int C, typename F>
__device__ __forceinline__ float few_across(const float (&in)[C], int lane, F&& join) {
  float v[C];
#pragma unroll
  for (int i = 0; i < C; ++i) v[i] = in[i];
#pragma unroll
  for (int step = 0; step < 5; ++step) {
    const int bit = 16 >> step, half = C >> (step + 1);
    const bool up = (lane & bit) != 0;
    if (half == 0) {
      v[0] = join(v[0], __shfl_xor_sync(0xFFFFFFFFu, v[0], bit));
    } else {
#pragma unroll
      for (int i = 0; i < half; ++i) {
        const float other = __shfl_xor_sync(0xFFFFFFFFu, up ? v[i] : v[i + half], bit);
        v[i] = join(up ? v[i + half] : v[i], other);
      }
    }
  }
  return v[0];
}

// four consecutive columns of this thread's TMEM lane
__device__ __forceinline__ void few_ld4(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}

__device__ __forceinline__ void few_st4(uint32_t at, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}

// 8 e4m3 codes -> 8 fp16 numbers, exactly
__device__ __forceinline__ uint4 few_halves(uint32_t a, uint32_t b) {
  uint4 r;
  asm("{\n"
      ".reg .b16 l, h;\n"
      "mov.b32 {l, h}, %4;\n"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n"
      "mov.b32 {l, h}, %5;\n"
      "cvt.rn.f16x2.e4m3x2 %2, l;\n"
      "cvt.rn.f16x2.e4m3x2 %3, h;\n"
      "}\n"
      : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
      : "r"(a), "r"(b));
  return r;
}

__device__ __forceinline__ uint32_t few_pack_half(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The fp16 numbers that e4m3 codes stand for to bf16 numbers 2^-kFewWidePower as large, exactly: a larger exponent field's bias.  (NaN
// does not stay one; it is in rows whose weights are NaN.)
__device__ __forceinline__ uint4 few_wide_values(uint4 v) {
  auto one = [](uint32_t h) { return (h & 0x80008000u) | ((h >> 3) & 0x0FF00FF0u); };
  return make_uint4(one(v.x), one(v.y), one(v.z), one(v.w));
}

// Values of a tile whose weights are bf16: widened to fp16 by other warps as ever, then changed in place by the 128 threads that made the
// weights.  Not inlined: the softmax warps' loop with this inside it was 8 % slower where it is not wanted (64 sequences of
// 3000 tokens 114 us for 106).  bf16 weights and values for every tile, without a reference exponent: 133.
__device__ __noinline__ bool few_widen_tile(uint64_t* bar, uint32_t parity, uint32_t* status, uint4* v, int n) {
  if (!few_wait_warp(bar, parity, status)) return false;
#pragma unroll 1
  for (int i = 0; i < n; i += kCaTile) v[i] = few_wide_values(v[i]);
  return true;
}

// 2^(byte - 127); byte 255 gives NaN
__device__ __forceinline__ float few_power(uint32_t byte) {
  return byte == 255u ? __int_as_float(0x7FC00000) : byte == 0u ? __int_as_float(0x00400000) : __int_as_float(static_cast<int>(byte) << 23);
}

// Query rows (bf16, as they lie) to two codes for each number and a power of two for each row: codes of what is left after the first
// ones, times 16, are rows N + i.  Four lanes for a row, eight rows at a time for a warp; `rows`: the table of rows, -1 = none.
template <int D, int N, int R>
__device__ __forceinline__ void few_query(const uint8_t* raw, uint8_t* dst, float* factor, const int* rows, float scale, int from, int step) {
  const int part = threadIdx.x & 3;
#pragma unroll 1
  for (int i = from + ((threadIdx.x & 31) >> 2); i < (R < 8 ? 8 : R); i += step) {
    const bool there = i < R && rows[i] >= 0;
    constexpr int kVecs = D / 32;                                    // 16-byte vectors of a lane
    uint4 x[kVecs];
    uint32_t m2 = 0;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      x[v] = there ? *reinterpret_cast<const uint4*>(raw + i * D * 2 + (part * kVecs + v) * 16) : make_uint4(0, 0, 0, 0);
      m2 = __vmaxu2(__vmaxu2(m2, x[v].x & 0x7FFF7FFFu), __vmaxu2(x[v].y & 0x7FFF7FFFu, __vmaxu2(x[v].z & 0x7FFF7FFFu, x[v].w & 0x7FFF7FFFu)));
    }
    uint32_t most = max(m2 & 0xFFFFu, m2 >> 16);
    most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
    most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, 2));
    const bool finite = most < 0x7F80u;
    const int byte = finite ? max(0, static_cast<int>(most >> 7) - 8 + ((most & 0x7Fu) > 0x60u ? 1 : 0)) : 127;
    const float inv = __int_as_float((254 - byte) << 23);            // 2^-E
#pragma unroll
    for (int v = 0; v < kVecs; v += 2) {
      const uint32_t w[8] = {x[v].x, x[v].y, x[v].z, x[v].w, x[v + 1].x, x[v + 1].y, x[v + 1].z, x[v + 1].w};
      uint32_t c1[4] = {0, 0, 0, 0}, c2[4] = {0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float2 f = make_float2(__uint_as_float(w[e] << 16) * inv, __uint_as_float(w[e] & 0xFFFF0000u) * inv);
        const __nv_fp8x2_storage_t a = __nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3);
        const float2 y = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(a, __NV_E4M3)));
        const __nv_fp8x2_storage_t b = __nv_cvt_float2_to_fp8x2(make_float2((f.x - y.x) * 16.f, (f.y - y.y) * 16.f), __NV_SATFINITE, __NV_E4M3);
        c1[e / 2] |= static_cast<uint32_t>(a) << (16 * (e & 1));
        c2[e / 2] |= static_cast<uint32_t>(b) << (16 * (e & 1));
      }
      // rows i and N + i (N is a multiple of 16: the same exchange of places)
      const int at = few_place<D>(i, (part * kVecs + v) / 2) << 4;
      if (i < R) {
        *reinterpret_cast<uint4*>(dst + i * D + at) = finite ? make_uint4(c1[0], c1[1], c1[2], c1[3]) : make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(dst + (N + i) * D + at) = finite ? make_uint4(c2[0], c2[1], c2[2], c2[3]) : make_uint4(0, 0, 0, 0);
      }
    }
    if (part == 0 && i < R) factor[i] = finite ? scale * few_power(byte) : __int_as_float(0x7FC00000);
  }
  fence_proxy_async_smem();
  __syncwarp();
}

// Barrier over `THREADS` threads with an OR of `v` (lanes that left a wait at different times are brought together first).
template <int THREADS>
__device__ __forceinline__ bool few_any(int id, bool v) {
  uint32_t any;
  __syncwarp();
  asm volatile(
      "{\n"
      ".reg .pred pin, pout;\n"
      "setp.ne.u32 pin, %1, 0;\n"
      "bar.red.or.pred pout, %2, %3, pin;\n"
      "selp.u32 %0, 1, 0, pout;\n"
      "}\n"
      : "=r"(any)
      : "r"(static_cast<uint32_t>(v)), "r"(id), "n"(THREADS)
      : "memory");
  return any != 0u;
}

template <int D, bool F8, int R>
__global__ void __launch_bounds__(CacheFew<D, F8, R>::kThreads, 1) cache_few_kernel(const __grid_constant__ CacheFewParams fp) {
  using S = CacheFew<D, F8, R>;
  const CacheAttnParams& p = fp.a;
  constexpr int kStages = S::kStages, N = S::kN;
  constexpr uint32_t kSlab = kCaTile * 128;                          // 128 rows x 64 columns of bf16
  constexpr int kPRow = N * 2;                                       // bytes of a key's weights
  constexpr uint32_t kIdescS = F8 ? make_idesc_e4m3(128, 2 * N) : make_idesc_bf16(128, N, false, false);
  constexpr uint32_t kIdescPV = make_idesc_bf16(128, N, true, true);
  constexpr uint32_t kIdescHalf = kIdescPV & ~((1u << 7) | (1u << 10));          // the format fields of fp16 are zero

  extern __shared__ uint8_t cf_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(cf_raw) + 1023) & ~uintptr_t(1023));
  // At D = 64 the products with the values read a second slab of 64 rows behind the first, whose results nobody looks at: widened
  // values have the ring behind them, values of a stage its keys.
  uint8_t* sWide = smem;                                             // [2]
  uint8_t* sRing = sWide + 2 * S::kWide;
  uint8_t* sP = sRing + kStages * S::kStage;                         // [2]
  uint8_t* sQ = sP + 2 * S::kP;                                      // [2]
  uint8_t* sRaw = sQ + 2 * S::kQ;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRaw + S::kRaw);
  uint64_t* full = bars;                     // [kStages] keys, values and exponent bytes have landed
  uint64_t* empty = bars + kStages;          // [kStages]
  // of a piece:
  uint64_t* s_full = bars + 2 * kStages;     // [2]
  uint64_t* p_full = s_full + 2;             // [2] weights are stored and all scores read
  uint64_t* pv_done = p_full + 2;            // [2]
  uint64_t* v_full = pv_done + 2;            // [2] widened values
  uint64_t* q_empty = v_full + 2;            // [2] query rows
  uint64_t* q_full = q_empty + 2;            // [2][2] query rows and their tables, of which there are two
  uint64_t* t_empty = q_full + 4;            // [2][2]
  uint64_t* raw_full = t_empty + 4;          // [2] query rows as they were (of a piece: kOwnRows)
  uint64_t* raw_empty = raw_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw_empty + 1);
  uint8_t* sByte = reinterpret_cast<uint8_t*>(bars) + 256;                               // [kStages][2][128]
  CacheFewTile* sTile = reinterpret_cast<CacheFewTile*>(sByte + kStages * 2 * kCaTile);  // [kStages]
  volatile int* sKind = reinterpret_cast<int*>(bars) + 60;                               // [2] the weights are: 1 an item's first, 2 bf16
  int4* sItem = reinterpret_cast<int4*>(sTile + kStages);                                // [2][2] first row of q, key head, slot
  int* sHi = reinterpret_cast<int*>(sItem + 4);                    // [2][2][N] last visible key of a row, -1 = none
  int* sRow = sHi + 4 * N;                                                               // [2][2][N] token << 8 | head of the group
  float* sFactor = reinterpret_cast<float*>(sRow + 4 * N);                               // [2][2][N] a row's power of two times the scale
  float* sM = sFactor + 4 * N;                                                           // [2][N] reference maxima
  float* sRed = sM + 2 * N;                                                              // [2][4][N] maxima of the warps; a new one goes to [0]
  float* sSum = sRed + 8 * N;                                                            // [2][4][N] sums of the warps
  int* sTop = reinterpret_cast<int*>(sSum + 8 * N);                                      // [2][8] largest exponent bytes, reference
  CacheFewTable tab;
  tab.pre = sTop + 16;
  tab.q0 = tab.pre + kFewSequences + 1;
  tab.len = tab.q0 + kFewSequences;
  tab.q_len = reinterpret_cast<uint8_t*>(tab.len + kFewSequences);

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xFFFFFFFFu, tid >> 5, 0);
  if (tid == 0) {
    tma_prefetch_desc(&fp.tma_k);
    tma_prefetch_desc(&fp.tma_v);
    tma_prefetch_desc(&fp.tma_q);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], S::kEarly ? 9 : 1);         // early: the score product, four softmax warps, four widening ones
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&v_full[i], 4);
      mbar_init(&q_empty[i], 1);
    }
    mbar_init(&raw_full[0], 1);
    mbar_init(&raw_full[1], 1);
    mbar_init(raw_empty, 4);
    for (int i = 0; i < 4; ++i) {
      mbar_init(&q_full[i], !F8 ? 2 : S::kOwnRows ? 4 : 1);     // the rows, and the tables where those are copied as they are
      mbar_init(&t_empty[i], 4);
    }
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(tmem_slot, S::kCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  // query rows that do not exist stay zero
  for (int i = tid; i < 2 * S::kQ / 16; i += S::kThreads) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  // the tensor memory is this kernel's before the next one may begin
  chain_next();
  chain_wait();
  ca_zero<D, S::kThreads>(p);
  // Tiles in front of every sequence: each thread adds up a few sequences, the warps scan those sums, and the warps' are added.
  {
    const int each = (p.batch + S::kThreads - 1) / S::kThreads, b0 = min(tid * each, p.batch), b1 = min(b0 + each, p.batch);
    int sum = 0;
    for (int b = b0; b < b1; ++b) {
      int q0, q_len, len;
      ca_sequence(p, b, q0, q_len, len, blockIdx.x == 0);
      CacheTiles tiles;
      const int n = tiles.set(len - q_len, len - 1, p.window, p.first, 0, 1);
      tab.q0[b] = q0;
      tab.q_len[b] = static_cast<uint8_t>(max(q_len, 0));
      tab.len[b] = len;
      tab.pre[b + 1] = q_len > 0 ? max(n, 1) : 0;
      sum += tab.pre[b + 1];
    }
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, scan, o);
      if (lane >= o) scan += v;
    }
    int* totals = reinterpret_cast<int*>(sRed);                      // [warps]
    if (lane == 31) totals[warp] = scan;
    __syncthreads();
    int ahead = scan - sum + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? totals[lane] : 0);
    for (int b = b0; b < b1; ++b) {
      ahead += tab.pre[b + 1];
      tab.pre[b + 1] = ahead;
    }
    if (tid == 0) tab.pre[0] = 0;
    __syncthreads();
  }
  if (blockIdx.x == 0)
    for (int b = tid; b <= p.batch; b += S::kThreads) fp.pre[b] = tab.pre[b];
  const int places = tab.pre[p.batch] * p.hk;
  const CacheFewCuts cuts(places, few_pieces(places, gridDim.x));

  auto stage_v = [&](uint32_t s) { return sRing + s * S::kStage; };
  auto stage_k = [&](uint32_t s) { return sRing + s * S::kStage + S::kHalf; };
  const uint32_t tO = tmem_base + 2 * S::kSCols;                     // [2] of N columns behind the scores

  // the longer one is the first
  const int extra = cuts.tiles(gridDim.x + blockIdx.x) > cuts.tiles(blockIdx.x) ? 1 : 0;
  auto piece_of = [&](uint32_t group) { return static_cast<int>(blockIdx.x + ((group ^ extra) != 0u ? gridDim.x : 0u)); };
  const int both = cuts.tiles(piece_of(0)) + cuts.tiles(piece_of(1));       // tiles of both pieces

  if (warp == 10 || warp == 11) {
    // ------------------------------------ copies --------------------------------------------
    const uint32_t grp = warp - 10, lead = elect_one() ? 1u : 0u;
    const int piece = piece_of(grp), boxes = kCaTile / p.box, per_look = 32 / boxes;
    const uint32_t others = both - cuts.tiles(piece);
    uint32_t k = 0;
    bool ok = true;
    CacheFewItem it;
    it.begin_walk(p, tab, cuts, piece);
    while (ok && it.next(p, tab)) {
      // lane i: slot of copy i of the next tiles and its place in the page (negative where no key of it is seen), looked up while
      // those of the tiles in front are used; a lone place for it, so that its code is there once
      int2 rows = {}, next = {};
      for (int j = -1, in = per_look - 1; j < it.n; ++j) {
        const bool look = ++in == per_look;
        if (look) {
          if (j >= 0) in = 0;
          rows = next;
        }
        if (j >= 0) {
          const uint32_t g = few_turn(k, grp, others), s = g % kStages;
          const uint32_t here = __ballot_sync(0xFFFFFFFFu, rows.x >= 0 && lane / boxes == in);
          ok = few_wait_warp(&empty[s], ((g / kStages) & 1u) ^ 1u, p.status);
          if (!ok) break;
          if (lead) {
            const int key0 = it.first_key(j);
            const bool whole = it.whole(key0);
            const bool all = whole && key0 + kCaTile - 1 <= it.shift &&
                             (p.window == 0 || key0 > it.q_len - 1 + it.shift - p.window || key0 + kCaTile <= p.first);
            sTile[s].key = key0;
            sTile[s].flags = static_cast<int>(grp) | (j == 0 ? kFewFirst : 0) | (j + 1 == it.n ? kFewLast : 0) | (whole ? kFewWhole : 0) |
                             (all ? kFewAll : 0);
            sTile[s].lo = it.lo;
            sTile[s].last = it.last;
            sTile[s].first_end = it.first_end;
            mbar_expect_tx(&full[s], static_cast<uint32_t>(__popc(here)) * p.box * (F8 ? 2 * D + 2 : 4 * D));
          }
          for (int i = 0; i < boxes; ++i) {
            const int row = __shfl_sync(0xFFFFFFFFu, rows.x, in * boxes + i), off = __shfl_sync(0xFFFFFFFFu, rows.y, in * boxes + i);
            if (!lead || row < 0) continue;
            if constexpr (F8) {
              const int64_t from = static_cast<int64_t>(row) * p.hk + it.kvh * p.block - off * (p.hk - 1);   // [page][head][place]
              tma_load_3d(stage_k(s) + i * p.box * D, &fp.tma_k, &full[s], 0, it.kvh, row);
              bulk_load_1d(sByte + s * 2 * kCaTile + i * p.box, fp.ks + from, p.box, &full[s]);
              tma_load_3d(stage_v(s) + i * p.box * D, &fp.tma_v, &full[s], 0, it.kvh, row);
              bulk_load_1d(sByte + s * 2 * kCaTile + kCaTile + i * p.box, fp.vs + from, p.box, &full[s]);
            } else {
#pragma unroll
              for (int c = 0; c < D / 64; ++c) tma_load_3d(stage_k(s) + c * kSlab + i * p.box * 128, &fp.tma_k, &full[s], c * 64, it.kvh, row);
#pragma unroll
              for (int c = 0; c < D / 64; ++c) tma_load_3d(stage_v(s) + c * kSlab + i * p.box * 128, &fp.tma_v, &full[s], c * 64, it.kvh, row);
            }
          }
          __syncwarp();
          ++k;
        }
        if (look) {
          const int at = (j < 0 ? 0 : j + per_look) + lane / boxes, key = it.first_key(at) + (lane % boxes) * p.box;
          next = at < it.n && it.any(key, p.box) ? make_int2(ca_slot(p, it.b, key), key % p.block) : make_int2(-1, 0);
          if (j < 0) in = per_look - 1;
        }
      }
    }
  } else if (warp == 9) {
    // ------------------------------------ query rows ----------------------------------------
    // Items of both pieces, in the order in which their first tiles are multiplied.
    const int n0 = cuts.tiles(piece_of(0));
    const uint32_t lead = elect_one() ? 1u : 0u;
    uint32_t items[2] = {0u, 0u}, k[2] = {0u, 0u}, fills = 0;        // items and tiles so far, copies of query rows
    CacheFewItem now, then;
    uint32_t grp = 0;
    now.begin_walk(p, tab, cuts, piece_of(0));
    then.begin_walk(p, tab, cuts, piece_of(1));
    for (;;) {
      const uint32_t turn0 = few_turn(k[0], 0, both - n0), turn1 = few_turn(k[1], 1, n0);
      const bool live0 = k[0] < static_cast<uint32_t>(n0), live1 = k[1] < static_cast<uint32_t>(both - n0);
      if (!live0 && !live1) break;
      const uint32_t want = !live0 || (live1 && turn1 < turn0) ? 1u : 0u;
      if (want != grp) {
        const CacheFewItem other = then;
        then = now;
        now = other;
        grp = want;
      }
      CacheFewItem& it = now;
      it.next(p, tab);
      const uint32_t item = grp != 0 ? items[1] : items[0], tb = grp * 2 + (item & 1u);
      if (!few_wait_warp(&q_empty[grp], (item & 1u) ^ 1u, p.status) || !few_wait_warp(&t_empty[tb], ((item >> 1) & 1u) ^ 1u, p.status)) break;
      if (lane == 0) sItem[tb] = make_int4(it.q_begin, it.kvh, it.slot, 0);
      for (int i = lane; i < R; i += 32) {
        const int tok = i / p.group;
        sHi[tb * N + i] = tok < it.q_len ? tok + it.shift : -1;
        sRow[tb * N + i] = tok < it.q_len ? tok << 8 | (i - tok * p.group) : -1;
      }
      __syncwarp();
      const int box = p.group * p.per_tile;                          // rows of the copy
      if constexpr (F8) {
        uint64_t* raw = &raw_full[S::kOwnRows ? grp : 0];
        if (S::kOwnRows && !few_wait_warp(raw_empty, (fills & 1u) ^ 1u, p.status)) break;
        if (lead) {
          mbar_expect_tx(raw, static_cast<uint32_t>(box) * D * 2);
          tma_load_3d(sRaw, &fp.tma_q, raw, 0, it.kvh * p.group, it.q_begin);
        }
        if (!S::kOwnRows) {
          if (!few_wait_warp(raw, fills & 1u, p.status)) break;
          few_query<D, N, R>(sRaw, sQ + grp * S::kQ, sFactor + tb * N, sRow + tb * N, p.scale_log2, 0, 8);
          if (lane == 0) mbar_arrive(&q_full[tb]);
        }
        ++fills;
      } else {
        if (lead) {
          mbar_expect_tx(&q_full[tb], static_cast<uint32_t>(box) * D * 2);
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
            tma_load_3d(sQ + grp * S::kQ + c * (N * 128), &fp.tma_q, &q_full[tb], c * 64, it.kvh * p.group, it.q_begin);
        }
        // the copy's arrival is announced above: this one is the tables'
        if (lane == 0) mbar_arrive(&q_full[tb]);
      }
      if (grp != 0) { ++items[1]; k[1] += it.n; } else { ++items[0]; k[0] += it.n; }
    }
  } else if (warp == 8) {
    // ------------------------------------ products ------------------------------------------
    if (elect_one()) {
      const uint32_t n0 = cuts.tiles(piece_of(0)), n1 = both - n0;
      uint32_t items0 = 0, items1 = 0;
      // scores of tile k of a piece
      auto scores = [&](uint32_t i, uint32_t k) -> bool {
        const uint32_t g = few_turn(k, i, i != 0 ? n0 : n1), s = g % kStages;
        if (!few_wait(&full[s], (g / kStages) & 1u, p.status)) return false;
        const int flags = sTile[s].flags;
        const uint32_t item = i != 0 ? items1 : items0;
        if ((flags & kFewFirst) != 0 && !few_wait(&q_full[i * 2 + (item & 1u)], (item >> 1) & 1u, p.status)) return false;
        tc_fence_after_sync();
        const uint32_t aK = smem_u32(stage_k(s)), aQ = smem_u32(sQ + i * S::kQ), tS = tmem_base + i * S::kSCols;
        if constexpr (F8) {
#pragma unroll
          for (int kk = 0; kk < D / 32; ++kk)
            tc_mma_f8_ss(tS, few_desc<D>(aK + kk * 32), few_desc<D>(aQ + kk * 32), kIdescS, kk != 0 ? 1u : 0u);
        } else {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            tc_mma_f16_ss(tS, few_desc<128>(aK + (kk / 4) * kSlab + (kk % 4) * 32), few_desc<128>(aQ + (kk / 4) * (N * 128) + (kk % 4) * 32),
                          kIdescS, kk != 0 ? 1u : 0u);
        }
        tc_commit(&s_full[i]);
        if (S::kEarly) tc_commit(&empty[s]);
        if ((flags & kFewLast) != 0) {
          tc_commit(&q_empty[i]);
          if (i != 0) ++items1; else ++items0;
        }
        return true;
      };
      uint32_t k0 = 0, k1 = 0;                                       // tiles of the pieces
      // the first scores of both, then tile by tile in the order of the ring; a lone call of `scores`, so that its code is there once
      for (int g = -2; g < both; ++g) {
        uint32_t i, next;
        if (g < 0) {
          i = g + 2;
          next = 0;
        } else {
          i = k0 >= n0 || (k1 < n1 && k1 < k0) ? 1u : 0u;
          const uint32_t k = i != 0 ? k1 : k0, at = few_turn(k, i, i != 0 ? n0 : n1), s = at % kStages;
          // the weights are stored and the scores read; of 8 bits the stage may be another tile's by now
          if (!few_wait(&p_full[i], k & 1u, p.status) || (F8 && !few_wait(&v_full[i], k & 1u, p.status))) break;
          tc_fence_after_sync();
          const uint32_t aV = F8 ? smem_u32(sWide + i * S::kWide) : smem_u32(stage_v(s)), aP = smem_u32(sP + i * S::kP);
          const int kind = sKind[i];
          const uint32_t more = (kind & 1) == 0 ? 1u : 0u, idesc = !F8 || (kind & 2) != 0 ? kIdescPV : kIdescHalf;
#pragma unroll
          for (int kk = 0; kk < kCaTile / 16; ++kk)
            tc_mma_f16_ss(tO + i * N, make_smem_desc(aV + kk * 2048, kSlab, 1024), few_desc<kPRow>(aP + kk * 16 * kPRow), idesc,
                          kk != 0 ? 1u : more);
          tc_commit(&pv_done[i]);
          if (!S::kEarly) tc_commit(&empty[s]);
          next = k + 1;
          if (i != 0) ++k1; else ++k0;
        }
        if (next < (i != 0 ? n1 : n0) && !scores(i, next)) break;
      }
    }
  } else if (warp >= 12) {
    if constexpr (F8) {
      // ------------------------------------ values to fp16 ----------------------------------
      constexpr int kLanes = D / 16;                                   // lanes of a row, 16 codes each
      constexpr int kStep = 128 / kLanes, kRows = kCaTile / kStep;
      const int c = (tid - 384) % kLanes, row0 = (tid - 384) / kLanes;
      // 16 codes fill two 16-byte places of a swizzled row.  Where 8 lanes work on one row, those of the second slab start with the
      // odd place: the 8 stores then meet 8 different groups of banks.  kStep is a multiple of 8: a thread's rows are all alike.
      const int w = (2 * c) & 7, odd_first = D == 128 && c >= 4 ? 1 : 0;
      const uint32_t place0 = (c / 4) * kSlab + row0 * 128 + (((w + odd_first) ^ (row0 & 7)) << 4);
      const uint32_t place1 = (c / 4) * kSlab + row0 * 128 + (((w + 1 - odd_first) ^ (row0 & 7)) << 4);
      uint32_t k0 = 0, k1 = 0, s = 0, ph = 0;                        // tiles of the pieces
      for (int g = 0; g < both; ++g) {
        if (!few_wait_warp(&full[s], ph, p.status)) break;
        const uint8_t* src = stage_v(s) + row0 * D + c * 16;
        uint4 x[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) x[i] = *reinterpret_cast<const uint4*>(src + i * kStep * D);
        const int flags = sTile[s].flags;
        if ((flags & kFewWhole) == 0) {                              // values that no row sees are cleared (0 * NaN would be NaN)
          const CacheFewTile tile = sTile[s];
#pragma unroll
          for (int i = 0; i < kRows; ++i)
            if (!tile.seen(tile.key + row0 + i * kStep)) x[i] = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
        if (S::kEarly && lane == 0) mbar_arrive(&empty[s]);
        const bool second = (flags & kFewGroup) != 0;
        const uint32_t i_side = second ? 1u : 0u, mine = second ? k1 : k0;
        if (mine > 0 && !few_wait_warp(&pv_done[i_side], (mine - 1) & 1u, p.status)) break;
        uint8_t* dst = sWide + i_side * S::kWide;
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
          const uint4 a = few_halves(x[i].x, x[i].y), b = few_halves(x[i].z, x[i].w);
          *reinterpret_cast<uint4*>(dst + place0 + i * kStep * 128) = odd_first ? b : a;
          *reinterpret_cast<uint4*>(dst + place1 + i * kStep * 128) = odd_first ? a : b;
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[i_side]);
        if (second) ++k1; else ++k0;
        if (++s == kStages) { s = 0; ph ^= 1u; }
      }
    }
  } else if (warp < 8) {
    // ------------------------------------ softmax -------------------------------------------
    const uint32_t grp = warp >> 2;                                  // the piece of this warp
    const int t = tid & 127, bar = 1 + grp;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem_base + lane_off + grp * S::kSCols, to = tO + lane_off + grp * N;
    float *m_mine = sM + grp * N, *red = sRed + grp * 4 * N;
    int* top = sTop + grp * 8;                                       // exponent bytes: [0..3] of the warps, [6] least, [7] reference
    uint8_t* sp = sP + grp * S::kP + t * kPRow;
    uint32_t k = 0, items = 0;                                       // tiles and items so far
    bool ok = true;
    const int piece = piece_of(grp);
    const uint32_t mine = cuts.tiles(piece), others = both - mine;
    constexpr int C = R < 16 ? R : 16;                               // rows at a time
    float* sums = sSum + (grp * 4 + (warp & 3)) * N;
    const int my_row = lane / (32 / C);                              // whose joined value this lane holds
    const bool my_turn = lane % (32 / C) == 0;
    bool pending = false;                                            // an item's tiles are done, its sums not yet written
    for (;; ++k) {
      if (S::kOwnRows && (k == 0 || pending) && k < mine) {          // before the sums are written: the next scores wait for it
        const uint32_t next = items + (pending ? 1u : 0u), tb = grp * 2 + (next & 1u);
        ok = ok && few_wait_warp(&raw_full[grp], next & 1u, p.status);
        if (ok) {
          few_query<D, N, R>(sRaw, sQ + grp * S::kQ, sFactor + tb * N, sRow + tb * N, p.scale_log2, (warp & 3) * 8, 32);
          if (lane == 0) {
            mbar_arrive(raw_empty);
            mbar_arrive(&q_full[tb]);
          }
        }
      }
      if (pending) {
        const uint32_t tb = grp * 2 + (items & 1u);
        // ---- the end of an item
        ok = ok && few_wait(&pv_done[grp], (k - 1u) & 1u, p.status);
        ok = !few_any<128>(bar, !ok);                // all sums are there
        if (!ok) break;                              // a wait ran out (the status word says so): the outputs are not written
        tc_fence_after_sync();
        const int4 item = sItem[tb];                 // first row of q, key head, slot
        ++items;
        const float back = F8 ? few_power(max(top[7], 0)) * 0.0625f : 1.f;                 // 2^(Eref - 4)
        const float* all = sSum + grp * 4 * N;
        // a row's factor, for rows of parts with its sum beside it, where the maxima of the warps were
        if (t < R) {
          const float sum = (all[t] + all[N + t]) + (all[2 * N + t] + all[3 * N + t]);
          red[t] = item.z >= 0 ? back : sum > 0.f ? back / sum : sum * 0.f;          // no visible key: 0, NaN stays
          if (item.z >= 0 && sRow[tb * N + t] >= 0)
            *reinterpret_cast<float2*>(p.pml + ((static_cast<int64_t>(piece) * 2 + item.z) * R + t) * 2) = make_float2(m_mine[t], sum);
        }
        few_any<128>(bar, false);
        float* part = p.po + (static_cast<int64_t>(piece) * 2 + item.z) * R * D + t;
        __nv_bfloat16* out = p.o + item.x * p.o_ld + static_cast<int64_t>(item.y * p.group) * D + t;
#pragma unroll 1
        for (int n0 = 0; n0 < R; n0 += C) {
          uint32_t o[16];
          tmem_ld16(to + n0, o);
          tc_wait_ld();
          float f[C];
          int at[C];
#pragma unroll
          for (int i = 0; i < C; i += 4) {
            *reinterpret_cast<float4*>(f + i) = *reinterpret_cast<const float4*>(red + n0 + i);
            *reinterpret_cast<int4*>(at + i) = *reinterpret_cast<const int4*>(sRow + tb * N + n0 + i);
          }
          if (t >= D) continue;
          if (item.z >= 0) {                         // rows that do not exist are not joined
#pragma unroll
            for (int i = 0; i < C; ++i) part[(n0 + i) * D] = __uint_as_float(o[i]) * f[i];
          } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
              if (at[i] >= 0) out[(at[i] >> 8) * p.o_ld + (at[i] & 255) * D] = __float2bfloat16(__uint_as_float(o[i]) * f[i]);
          }
        }
        tc_fence_before_sync();
        few_any<128>(bar, false);                    // sums, maxima and the row tables have been read
        if (lane == 0) mbar_arrive(&t_empty[tb]);
      }
      if (k >= mine) break;
      const uint32_t g = few_turn(k, grp, others), s = g % kStages, ph = k & 1u;
      const uint32_t tb = grp * 2 + (items & 1u);
      // a warp whose wait ran out (what it reads of the tile may then be anything) goes to the vote; the group leaves there together
      ok = ok && few_wait(&full[s], (g / kStages) & 1u, p.status);
      const int flags = sTile[s].flags, key = sTile[s].key + t;
      const bool first = (flags & kFewFirst) != 0;                   // the group's maxima, sums and reference are an earlier item's
      const bool seen = (flags & kFewWhole) != 0 || sTile[s].seen(key);
      if (first) ok = ok && few_wait(&q_full[tb], (items >> 1) & 1u, p.status);
      ok = ok && few_wait(&s_full[grp], ph, p.status);
      ok = __all_sync(0xFFFFFFFFu, ok);                              // the aligned tcgen05 instructions need a converged warp
      float kf = p.scale_log2;
      int vbyte = 0;
      bool high = false;
      float sc[C];
      // scores of C rows from n0 on (log2 domain)
      auto scores = [&](int n0) {
        uint32_t a[16];
        tmem_ld16(tS + n0, a);
        if constexpr (F8) {
          uint32_t b[16];
          tmem_ld16(tS + N + n0, b);
          float f[C];
#pragma unroll
          for (int i = 0; i < C; i += 4) *reinterpret_cast<float4*>(f + i) = *reinterpret_cast<const float4*>(sFactor + tb * N + n0 + i);
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < C; ++i) sc[i] = fmaf(__uint_as_float(b[i]), 0.0625f, __uint_as_float(a[i])) * (kf * f[i]);
        } else {
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < C; ++i) sc[i] = __uint_as_float(a[i]) * kf;
        }
        if ((flags & kFewAll) == 0) {
#pragma unroll
          for (int i = 0; i < C; ++i) {
            const int hi = sHi[tb * N + n0 + i];
            const bool mine = seen & (key <= hi) & ((p.window == 0) | (key > hi - p.window) | (key < p.first));
            sc[i] = mine ? sc[i] : kCaMask;
          }
        }
      };
      if (ok) {
        tc_fence_after_sync();
        if constexpr (F8) {
          kf = few_power(sByte[s * 2 * kCaTile + t]);
          vbyte = seen ? sByte[s * 2 * kCaTile + kCaTile + t] : 0;
          __syncwarp();
          if (S::kEarly && lane == 0) mbar_arrive(&empty[s]);
          const int2 ends = *reinterpret_cast<const int2*>(top + 6);
          // what is not seen has the byte 0, NaN (255) needs no reference
          high |= (vbyte > ends.y + 3) & (vbyte != 255) | seen & (vbyte < ends.x);
        }
        if constexpr (R == C) {
          scores(0);
#pragma unroll
          for (int i = 0; i < C; i += 4) {
            const float4 m = *reinterpret_cast<const float4*>(m_mine + i);
            high |= !(sc[i] <= m.x + kCaRescale) || !(sc[i + 1] <= m.y + kCaRescale) || !(sc[i + 2] <= m.z + kCaRescale) ||
                    !(sc[i + 3] <= m.w + kCaRescale);
          }
        }
      }
      // Lazy: a reference maximum moves only when a score exceeds it by more than 2^8 (or is NaN).  Scores of a few rows stay in
      // registers from one vote to the weights.  Those of many are read twice; there the weights are made at once, with the
      // references as they are, which is nearly always right, and made again where the vote says that one has to move.
      bool moves = first, out = false, wide = false;
      if constexpr (R == C) {
        tc_fence_before_sync();
        moves = few_any<128>(bar, high || first || !ok);
      }
      // the product of the group's last tile has landed: its P buffer is free, its sums may be rescaled
      if (k > 0) ok = ok && few_wait(&pv_done[grp], ph ^ 1u, p.status);
      ok = __all_sync(0xFFFFFFFFu, ok);
      for (;;) {
        if (moves) {
          if (ok) {
            tc_fence_after_sync();
#pragma unroll 1
            for (int n0 = 0; n0 < R; n0 += C) {
              if (R > C) scores(n0);
              const float v = few_across<C>(sc, lane, [](float x, float y) { return max_nan(x, y); });
              if (my_turn) red[(warp & 3) * N + n0 + my_row] = v;
            }
            if (F8) {
              const int v = __reduce_max_sync(0xFFFFFFFFu, vbyte == 255 ? 0 : vbyte);
              const int u = __reduce_min_sync(0xFFFFFFFFu, seen ? vbyte : 255);
              if (lane == 0) top[warp & 3] = v | u << 8;
            }
          }
          ok = !few_any<128>(bar, !ok);
          out = !ok;
          if (out) break;
          // a reference exponent that is passed by more than 3 moves as the maxima do; the least one moves a step more than it has to
          const int old_ref = !F8 ? 0 : first ? -1024 : top[7];
          int ref = 0, least = 0;
          if (F8) {
            const int most = max(max(top[0] & 255, top[1] & 255), max(top[2] & 255, top[3] & 255));
            ref = most > old_ref + 3 ? most : old_ref;
            least = min(min(top[0], top[1]) >> 8, min(top[2], top[3]) >> 8) - 1;         // the upper bytes order the words
            least = first ? least : min(least, top[6]);
            if (ref - least > kFewSpread) least = -1024;             // far enough: nothing below moves it
          }
          const float rescale = F8 ? ex2(static_cast<float>(old_ref - ref)) : 1.f;
          if (t < R) {
            const float now = max_nan(max_nan(red[t], red[N + t]), max_nan(red[2 * N + t], red[3 * N + t]));
            const float old = first ? -1.0e29f : m_mine[t];
            red[t] = !(now <= old + kCaRescale) ? now : old;
          }
          few_any<128>(bar, false);
          if (!first) {
            tc_fence_after_sync();
#pragma unroll 1
            for (int n0 = 0; n0 < R; n0 += 4) {
              uint32_t o[4];
              few_ld4(to + n0, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 4; ++i)
                o[i] = __float_as_uint(__uint_as_float(o[i]) * (ex2(m_mine[n0 + i] - red[n0 + i]) * rescale));
              few_st4(to + n0, o);
              tc_wait_st();
            }
            tc_fence_before_sync();
            if (my_turn)
              for (int n0 = my_row; n0 < R; n0 += C) sums[n0] *= ex2(m_mine[n0] - red[n0]);
          }
          few_any<128>(bar, false);                                  // everyone has read the old maxima
          if (t < R) m_mine[t] = red[t];
          if (F8 && t == 0) {
            top[6] = least;
            top[7] = ref;
          }
          few_any<128>(bar, false);
        }
        if (ok) {
          tc_fence_after_sync();
          // A key's weights are a row of P.  The sums take bf16 weights as rounded, as the tensor core multiplies them; fp16 ones, which
          // hold the value's exponent as well, before they are rounded.
          const int2 ends = *reinterpret_cast<const int2*>(top + 6);
          wide = F8 && ends.y - ends.x > kFewSpread;
          const float vf = vbyte == 255 ? __int_as_float(0x7FC00000) : ex2(static_cast<float>(vbyte - ends.y + (wide ? 4 + kFewWidePower : 4)));
#pragma unroll 1
          for (int n0 = 0; n0 < R; n0 += C) {
            if (R > C) scores(n0);
            uint32_t w[C / 2];
#pragma unroll
            for (int i = 0; i < C; i += 4) {
              const float4 m = *reinterpret_cast<const float4*>(m_mine + n0 + i);
              const float x[4] = {sc[i] - m.x, sc[i + 1] - m.y, sc[i + 2] - m.z, sc[i + 3] - m.w};
              const float e[4] = {ex2(x[0]), ex2(x[1]), ex2(x[2]), ex2(x[3])};       // masked: 0
              if (R > C) high |= !(x[0] <= kCaRescale) || !(x[1] <= kCaRescale) || !(x[2] <= kCaRescale) || !(x[3] <= kCaRescale);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if constexpr (F8) {
                  w[i / 2 + h] = few_pack_half(e[2 * h] * vf, e[2 * h + 1] * vf);
                  sc[i + 2 * h] = e[2 * h];
                  sc[i + 2 * h + 1] = e[2 * h + 1];
                } else {
                  w[i / 2 + h] = pack_bf16(e[2 * h], e[2 * h + 1]);
                  sc[i + 2 * h] = __uint_as_float(w[i / 2 + h] << 16);
                  sc[i + 2 * h + 1] = __uint_as_float(w[i / 2 + h] & 0xFFFF0000u);
                }
              }
            }
            if (F8 && wide) {                        // again, as bf16: a branch that is rarely taken costs less than two forms of each weight
#pragma unroll
              for (int i = 0; i < C; i += 2) w[i / 2] = pack_bf16(sc[i] * vf, sc[i + 1] * vf);
            }
            if constexpr (R == 4) {
              *reinterpret_cast<uint2*>(sp + (few_place<kPRow>(t, 0) << 4)) = make_uint2(w[0], w[1]);
            } else {
#pragma unroll
              for (int i = 0; i < C / 8; ++i)
                *reinterpret_cast<uint4*>(sp + (few_place<kPRow>(t, n0 / 8 + i) << 4)) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
            }
            const float v = few_across<C>(sc, lane, [](float x, float y) { return x + y; });
            if (my_turn) {
              if (R == C) sums[my_row] = first ? v : sums[my_row] + v;
              else red[(warp & 3) * N + n0 + my_row] = v;
            }
          }
        }
        if (R == C || moves) break;
        moves = few_any<128>(bar, high || !ok);
        if (!moves) break;
      }
      if (out) break;                                // the group leaves, and with it the kernel
      if (ok) {
        // the sums of this tile, which the same lanes have written
        if (R > C && my_turn)
          for (int n0 = my_row; n0 < R; n0 += C) sums[n0] = first ? red[(warp & 3) * N + n0] : sums[n0] + red[(warp & 3) * N + n0];
        if (!F8 && !seen) {                          // values that no row sees are cleared (0 * NaN would be NaN)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int i = 0; i < 8; ++i) reinterpret_cast<uint4*>(stage_v(s) + c * kSlab + t * 128)[i] = make_uint4(0, 0, 0, 0);
        }
        if (F8 && wide)
          ok = few_widen_tile(&v_full[grp], ph, p.status, reinterpret_cast<uint4*>(sWide + grp * S::kWide) + t, S::kWide / 16);
      }
      if (ok) {
        fence_proxy_async_smem();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if ((warp & 3) == 0) sKind[grp] = (first ? 1 : 0) | (wide ? 2 : 0);
          mbar_arrive(&p_full[grp]);
        }
      }
      pending = (flags & kFewLast) != 0;
    }
  }

  tc_fence_before_sync();
  block_settle(p.status);                            // begins with a barrier
  if (warp == 8) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, S::kCols);
  }
}

// Joins the parts of a (sequence, head) that was cut: a warp for a row; most blocks leave at once.
template <int D, int R>
__global__ void __launch_bounds__(128) cache_few_join_kernel(const CacheFewParams fp, int ctas) {
  const CacheAttnParams& p = fp.a;
  chain_next();
  chain_wait();
  const int b = blockIdx.y, kvh = blockIdx.x, row = blockIdx.z * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int all = fp.pre[p.batch] * p.hk, tiles = fp.pre[b + 1] - fp.pre[b], from = fp.pre[b] * p.hk + kvh * tiles;
  if (tiles == 0) return;
  const CacheFewCuts cuts(all, few_pieces(all, ctas));
  const int c0 = cuts.piece(from), c1 = cuts.piece(from + tiles - 1);
  if (c0 == c1) return;
  int q_begin, q_len, k_len;
  ca_sequence(p, b, q_begin, q_len, k_len, false);
  if (row >= q_len * p.group) return;
  const int first_slot = cuts.cut(c0) == from ? 0 : 1;
  auto part = [&](int c) { return (c * 2 + (c == c0 ? first_slot : 0)) * R + row; };
  float m = -1.0e29f;
  for (int c = c0 + lane; c <= c1; c += 32) m = max_nan(m, p.pml[part(c) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
  constexpr int E = D / 32;
  float acc[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 8
  for (int c = c0; c <= c1; ++c) {
    const float2 ml = *reinterpret_cast<const float2*>(p.pml + part(c) * 2);
    const float f = ex2(ml.x - m);
    const float* o = p.po + static_cast<int64_t>(part(c)) * D + lane * E;
    l += ml.y * f;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 v = *reinterpret_cast<const float2*>(o + e);
      acc[e] += v.x * f;
      acc[e + 1] += v.y * f;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int tok = row / p.group, h = row - tok * p.group;
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.o + (q_begin + tok) * p.o_ld + static_cast<int64_t>(kvh * p.group + h) * D + lane * E);
#pragma unroll
  for (int e = 0; e < E; e += 2) dst[e / 2] = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
}

}  // namespace yv
