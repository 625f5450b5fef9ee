// A paged cache in 8 bits: keys and values become e4m3 codes with one power of two for each token and head as they are written,
// and are read back.  Attention over such pages, or over pages in bf16: cache_attn.cuh.
//
// A row x of d numbers (one head of one token) is held as code_i 2^E: E is the smallest exponent at which the largest |x_i| does
// not pass 448, e4m3's largest number, and code_i = x_i 2^-E to the nearest e4m3 number (ties to even).  The codes are floating
// point, so a finer factor than a power of two would not make them more exact; a power of two makes the product x_i 2^-E exact,
// the row's byte an exponent, and the value read back a bf16 number without rounding.  A row with a number that is not finite gets
// the byte 255 and is read as NaN throughout.
#include <cuda_fp8.h>

#include "cache_attn.cuh"
#include "cache_few.cuh"
#include "cache_ops.h"
#include "sm100.cuh"

namespace yv {
namespace {

constexpr int kRowsThreads = 256;

// One group of d / 8 lanes per row: 16 bytes in, 8 bytes of codes out, a byte by the first lane.
// 8191 tokens of 8 heads of 128 (50 MB) take 17.5 us from a cold cache in a captured run of calls, a copy of as many bytes 18.1 in
// the same way (7.8 at the rate of a copy of gigabytes); 18.8 call by
// call.  Two or four rows a group, loaded ahead, 20.5 for 19.
template <int D, bool CHAIN>
__global__ void __launch_bounds__(kRowsThreads) cache_write_fp8_kernel(const CacheRowsArgs a) {
  constexpr int kLanes = D / 8;
  chain_start<CHAIN>();
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kRowsThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int per = 2 * a.hk;
  const int64_t t = at / per;
  if (t >= a.tokens) return;                                   // whole groups of lanes leave together
  const int r = static_cast<int>(at - t * per);
  const bool val = r >= a.hk;
  const int h = val ? r - a.hk : r;
  const int slot = a.slots[t];
  if (slot < 0) return;
  if (slot >= a.num_slots) {
    if (lane == 0 && a.status != nullptr) atomicOr(a.status, kStatusIndexOutOfRange);
    return;
  }
  const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(val ? a.v : a.k) + t * (val ? a.v_ld : a.k_ld) +
                             static_cast<int64_t>(h) * D + lane * 8;
  const uint4 x = *reinterpret_cast<const uint4*>(src);
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  // magnitudes of bf16 numbers are ordered as integers; what is not finite is above all others
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m2 = __vmaxu2(m2, w[i] & 0x7FFF7FFFu);
  uint32_t top = max(m2 & 0xFFFFu, m2 >> 16);
  const unsigned mask = ((1u << kLanes) - 1u) << (threadIdx.x & 31 & ~(kLanes - 1));      // a group leaves as one
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
  // top = 1.f 2^(X - 127) against 448 = 1.75 2^8
  const bool finite = top < 0x7F80u;
  const int byte = finite ? max(0, static_cast<int>(top >> 7) - 8 + ((top & 0x7Fu) > 0x60u ? 1 : 0)) : 255;
  const float inv = __int_as_float((254 - (finite ? byte : 127)) << 23);          // 2^-E
  uint32_t c[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t both = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t p = w[2 * i + j];
      const float2 f = make_float2(__uint_as_float(p << 16) * inv, __uint_as_float(p & 0xFFFF0000u) * inv);
      both |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3)) << (16 * j);
    }
    c[i] = finite ? both : 0x7F7F7F7Fu;
  }
  uint8_t* dst = static_cast<uint8_t*>(val ? a.v_codes : a.k_codes) + (static_cast<int64_t>(slot) * a.hk + h) * D + lane * 8;
  *reinterpret_cast<uint2*>(dst) = make_uint2(c[0], c[1]);
  if (lane == 0) {
    const int page = slot / a.block;
    static_cast<uint8_t*>(val ? a.v_scale : a.k_scale)[(static_cast<int64_t>(page) * a.hk + h) * a.block + slot - page * a.block] =
        static_cast<uint8_t>(byte);
  }
}

// 2^(byte - 127) in fp32
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7FC00000u : byte == 0u ? 0x00400000u : byte << 23);
}

template <int D>
__global__ void __launch_bounds__(kRowsThreads) cache_read_fp8_kernel(const CacheRowsArgs a) {
  constexpr int kLanes = D / 16;
  const int64_t at = (static_cast<int64_t>(blockIdx.x) * kRowsThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  const int per = 2 * a.hk;
  const int64_t t = at / per;
  if (t >= a.tokens) return;
  const int r = static_cast<int>(at - t * per);
  const bool val = r >= a.hk;
  const int h = val ? r - a.hk : r;
  const int slot = a.slots[t];
  uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  if (slot >= a.num_slots) {
    if (lane == 0 && a.status != nullptr) atomicOr(a.status, kStatusIndexOutOfRange);
  } else if (slot >= 0) {
    const uint4 c = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(val ? a.v_codes : a.k_codes) +
                                                    (static_cast<int64_t>(slot) * a.hk + h) * D + lane * 16);
    const int page = slot / a.block;
    const float s = scale_of(static_cast<const uint8_t*>(
        val ? a.v_scale : a.k_scale)[(static_cast<int64_t>(page) * a.hk + h) * a.block + slot - page * a.block]);
    const uint32_t codes[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(codes[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(__half2(two));
      w[i] = pack_bf16(f.x * s, f.y * s);
    }
  }
  __nv_bfloat16* dst = static_cast<__nv_bfloat16*>(val ? a.vo : a.ko) + (t * a.hk + h) * D + lane * 16;
  reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int rows_grid(const CacheRowsArgs& a, int lanes, unsigned* grid) {
  if (a.hk <= 0 || (a.d != 64 && a.d != 128) || a.block <= 0 || a.num_slots < 0 || a.num_slots >= (1ll << 31)) return -1;
  const int64_t blocks = (a.tokens * 2 * a.hk * lanes + kRowsThreads - 1) / kRowsThreads;
  if (blocks > 0x7FFFFFFFll) return -2;
  *grid = static_cast<unsigned>(blocks);
  return 0;
}

}  // namespace

int launch_cache_write_fp8(const CacheRowsArgs& in, cudaStream_t stream) {
  CacheRowsArgs a = in;
  if (a.tokens <= 0) return 0;
  if (a.tokens == 1) a.k_ld = a.v_ld = 0;                      // a single row has no pitch
  unsigned grid = 0;
  const int r = rows_grid(a, a.d / 8, &grid);
  if (r != 0) return r;
  if (((a.k_ld | a.v_ld) & 7) != 0 || !al16(a.k) || !al16(a.v) || !al16(a.k_codes) || !al16(a.v_codes)) return -3;
  const bool chain = grid <= kChainBlocks;
  if (a.d == 128)
    return launch_chained_if(chain, cache_write_fp8_kernel<128, true>, cache_write_fp8_kernel<128, false>, dim3(grid), dim3(kRowsThreads), 0, stream, a);
  return launch_chained_if(chain, cache_write_fp8_kernel<64, true>, cache_write_fp8_kernel<64, false>, dim3(grid), dim3(kRowsThreads), 0, stream, a);
}

int launch_cache_read_fp8(const CacheRowsArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0) return 0;
  unsigned grid = 0;
  const int r = rows_grid(a, a.d / 16, &grid);
  if (r != 0) return r;
  if (!al16(a.ko) || !al16(a.vo) || !al16(a.k_codes) || !al16(a.v_codes)) return -3;
  (a.d == 128 ? cache_read_fp8_kernel<128> : cache_read_fp8_kernel<64>)<<<grid, kRowsThreads, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}

namespace {

constexpr float kLog2e = 1.4426950408889634f;

int sm_count() {
  static PerDeviceInt count;
  if (!count.cur()) {
    int dev = 0, n = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
    count.cur() = n > 0 ? n : 148;
  }
  return count.cur();
}

// Tokens of a query tile, whether blocks have two tiles, and the items of one key range.
struct CacheGrid {
  int per_tile, two;
  int64_t items;
};
CacheGrid cache_grid(const CacheAttnArgs& a) {
  CacheGrid g;
  g.per_tile = kCaTile / (a.hq / a.hk);
  const int64_t heads = static_cast<int64_t>(a.hk) * a.batch, tiles = (a.max_q + g.per_tile - 1) / g.per_tile;
  g.two = tiles > 1;
  g.items = (g.two ? (tiles + 1) / 2 : tiles) * heads;
  return g;
}

int check(const CacheAttnArgs& a) {
  if (a.d != 64 && a.d != 128) return -1;
  if (a.hk <= 0 || a.hq <= 0 || a.hq % a.hk != 0 || a.hq / a.hk > kCaTile) return -2;
  if (a.block <= 0 || a.block % 16 != 0 || a.table_width <= 0 || a.num_blocks <= 0 ||
      static_cast<int64_t>(a.num_blocks) * a.block >= (1ll << 31) || static_cast<int64_t>(a.table_width) * a.block >= (1ll << 30)) return -3;
  if (a.window < 0 || a.first < 0 || !(a.scale > 0.f) || a.max_q <= 0) return -4;
  if (!al16(a.q) || !al16(a.o) || !al16(a.k) || !al16(a.v) || ((a.q_ld | a.o_ld) & 7) != 0) return -5;
  return 0;
}

template <int D>
int run_cache_attn(const CacheAttnParams& p, unsigned grid, cudaStream_t stream) {
  using S = CacheAttn<D>;
  static PerDeviceInt configured;
  if (!configured.cur()) {
    const cudaError_t e = cudaFuncSetAttribute(cache_attn_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured.cur() = 1;
  }
  return launch_chained(cache_attn_kernel<D>, dim3(grid), dim3(S::kThreads), S::kTotal, stream, 0, p);
}

// Key tiles that a block of queries can see at most.
int64_t most_tiles(const CacheAttnArgs& a) {
  int64_t keys = static_cast<int64_t>(a.table_width) * a.block;
  const int64_t seen = static_cast<int64_t>(a.window) + a.first + a.max_q;
  if (a.window > 0 && seen < keys) keys = seen;
  return (keys + kCaTile - 1) / kCaTile;
}

// Rows that 8-bit keys of a sequence take once they are widened: as many as its table has room for, or as the new tokens' window and
// the first tokens can see, in whole tiles (see CacheRoom; 512 new tokens with a window of 4096 over a table of 131072 tokens
// of 8 heads of 128: 19 MB for 537).
int widened_room(const CacheAttnArgs& a) {
  const int64_t all = static_cast<int64_t>(a.table_width) * a.block;
  if (a.window <= 0) return static_cast<int>(all);
  const int64_t tiles = (static_cast<int64_t>(a.first) + kCaTile - 1) / kCaTile + (static_cast<int64_t>(a.window) + a.max_q - 2) / kCaTile + 2;
  return static_cast<int>(tiles * kCaTile < all ? tiles * kCaTile : all);
}

// Rows (token, head of a group) that the kernel for few tokens holds, 0 where cache_attn_kernel takes the call.  That one would
// have to widen 8-bit pages first: 16 sequences of 8192 tokens with 16 new ones, 4 heads a group: 137 us here, 17 new ones there 250.
// Pages in bf16 it reads as they are, and its 128 rows cost no more than the keys' bytes.  It is the slower one where its key
// ranges are uneven or too short, that is for up to 16 rows and many sequences (64 of up to 3000 tokens, 8 key heads, one new one:
// 137 us against 121 here; 16 of 8192: 98 and 98) or for little in all (one of 2048 tokens: 16.4 and 13.8; of 8192: 29.6 and 28.7;
// of 32768: 49 and 53).  More rows it takes always (16 of 8192 tokens with 8 new ones: 98 us, 131 here).
constexpr int kFewMost = 64, kFewMostWide = 16;
int few_rows(const CacheAttnArgs& a) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * (a.hq / a.hk), heads = static_cast<int64_t>(a.batch) * a.hk;
  if (rows > (a.k_scale != nullptr ? kFewMost : kFewMostWide)) return 0;
  if (a.k_scale == nullptr && heads < sm_count() && heads * most_tiles(a) > 4 * sm_count()) return 0;
  int r = 4;
  while (r < rows) r *= 2;
  return r;
}

// What a miss fetches into the L2: no more than a row of one head.  Another head's is read by another SM, at another time (8-bit
// rows of 128 bytes, 64 sequences of 3000 tokens: 604 MB read where 414 are needed).
CUtensorMapL2promotion row_fetch(int bytes) {
  return bytes >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : bytes >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B : CU_TENSOR_MAP_L2_PROMOTION_L2_64B;
}

int page_map(CUtensorMap* m, const CacheAttnArgs& a, const void* pages, int64_t slots, int box) {
  return make_tmap_3d(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, pages, static_cast<uint64_t>(a.d), static_cast<uint64_t>(a.hk),
                      static_cast<uint64_t>(slots), static_cast<uint64_t>(a.d) * 2,
                      static_cast<uint64_t>(a.hk) * a.d * 2, 64, 1, static_cast<uint32_t>(box), CU_TENSOR_MAP_SWIZZLE_128B,
                      row_fetch(a.d * 2));
}

}  // namespace

namespace {

// Key ranges of a block: the number that takes the least time, by an estimate in us: 1.9 a step (D = 128) and 2 a range for each
// round of ranges over the SMs, 2 for the second kernel and its bytes at 3 TB/s (a fit to 17 calls: (new tokens of cached) 512 of
// 16384, 32 heads over 8, D = 128: one range 256 us, two 154, three 201, eight 184; 128 of 16384: 250, 141, 104, 57; 2048 of 32768:
// 971, 1051, 1079, 1164.  The estimate's choice was within 5 % of the best of 12 numbers in 15 of the calls, 26 % off at worst).
// Equal pieces of one line of all tiles, as in cache_few.cuh, balance better but lose: 166 for the first call and 1908 for 4096 of
// 32768, where ranges take 154 and 1740.  Blocks of one head that walk the same keys at the same time share them in the L2; pieces
// begin anywhere, and each tile then comes from far away or from DRAM (2.7 GB read where the cache holds 0.13).
int tile_splits(const CacheAttnArgs& a) {
  const CacheGrid g = cache_grid(a);
  const int sms = sm_count();
  // steps of an item: key tiles of a block of two query tiles, pairs of key tiles of a lone one
  const double steps = static_cast<double>(most_tiles(a)) / (g.two ? 1 : 2);
  const int64_t room = (int64_t(256) << 20) / (a.total_q * a.hq * a.d * 4 + 1);              // ranges that the scratch has room for
  const double sums = static_cast<double>(a.total_q) * a.hq * a.d * 8;                       // bytes written and read, per range
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 32 && (s == 1 || (s <= 2 * steps && s <= room)); ++s) {
    const double rounds = static_cast<double>((g.items * s + sms - 1) / sms);
    const double cost = rounds * (steps / s * 1.9 + 2) + (s > 1 ? 2 + s * sums / 3e6 : 0);
    if (s == 1 || cost < least) { best = s; least = cost; }
  }
  return best;
}

// Scratch: parts of cut sums, then what is widened or counted.
int64_t part_bytes(const CacheAttnArgs& a, int few) {
  const int64_t rows = few != 0 ? static_cast<int64_t>(sm_count()) * 4 * few : a.splits > 1 ? a.total_q * a.hq * a.splits : 0;
  return (rows * (a.d + 2) * 4 + 255) & ~int64_t(255);
}

}  // namespace

int64_t cache_attn_plan(CacheAttnArgs& a) {
  a.wide_batch = 0;
  if (a.total_q <= 0 || a.batch <= 0 || check(a) != 0) return 0;
  const int few = few_rows(a);
  if (few != 0) return part_bytes(a, few) + (kFewSequences + 1) * 4;
  if (a.splits <= 0) a.splits = tile_splits(a);
  int64_t bytes = part_bytes(a, 0);
  if (a.k_scale != nullptr) {
    // about a gigabyte at a time, one sequence at least
    const int64_t one = static_cast<int64_t>(widened_room(a)) * a.hk * a.d * 4, fit = (int64_t(1) << 30) / one;
    a.wide_batch = static_cast<int>(fit < 1 ? 1 : fit < a.batch ? fit : a.batch);
    bytes += one * a.wide_batch;
  }
  return bytes;
}

namespace {

int launch_merge(const CacheAttnParams& p, int d, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((p.total_q * p.hq + 3) / 4));
  return launch_chained(d == 128 ? cache_attn_merge_kernel<128> : cache_attn_merge_kernel<64>, grid, dim3(128), 0, stream, 0, p);
}

// What both kernels read of the sequences.
CacheAttnParams cache_params(const CacheAttnArgs& a) {
  CacheAttnParams p = {};
  p.group = a.hq / a.hk;
  p.o = static_cast<__nv_bfloat16*>(a.o); p.o_ld = a.o_ld;
  p.cu_q = a.cu_q; p.table = a.table; p.lens = a.lens;
  p.total_q = a.total_q;
  p.hq = a.hq; p.hk = a.hk; p.batch = a.batch; p.max_q = a.max_q;
  p.block = a.block; p.num_blocks = a.num_blocks; p.table_width = a.table_width;
  p.window = a.window; p.first = a.window > 0 ? a.first : 0;
  p.splits = a.splits;
  p.zero_rest = a.zero_rest;
  p.scale_log2 = a.scale * kLog2e;
  p.status = a.status;
  // rows of one copy: a power of two that divides a page
  p.box = 16;
  while (p.box < kCaTile && a.block % (2 * p.box) == 0) p.box *= 2;
  return p;
}

template <int D, bool F8, int R>
int run_cache_few(const CacheFewParams& p, unsigned grid, cudaStream_t stream) {
  using S = CacheFew<D, F8, R>;
  static PerDeviceInt configured;
  if (!configured.cur()) {
    const cudaError_t e = cudaFuncSetAttribute(cache_few_kernel<D, F8, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kTotal);
    if (e != cudaSuccess) return static_cast<int>(e);
    configured.cur() = 1;
  }
  return launch_chained(cache_few_kernel<D, F8, R>, dim3(grid), dim3(S::kThreads), S::kTotal, stream, 0, p);
}

template <int D, bool F8>
int run_cache_few(const CacheFewParams& p, int rows, unsigned grid, cudaStream_t stream) {
  switch (rows) {
    case 4: return run_cache_few<D, F8, 4>(p, grid, stream);
    case 8: return run_cache_few<D, F8, 8>(p, grid, stream);
    case 16: return run_cache_few<D, F8, 16>(p, grid, stream);
    case 32:
      if constexpr (F8) return run_cache_few<D, F8, 32>(p, grid, stream);
      return -9;
    default:
      if constexpr (F8) return run_cache_few<D, F8, 64>(p, grid, stream);
      return -9;
  }
}

int code_map(CUtensorMap* m, const CacheAttnArgs& a, const void* codes, int box, CUtensorMapSwizzle swizzle) {
  return make_tmap_3d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, codes, static_cast<uint64_t>(a.d), static_cast<uint64_t>(a.hk),
                      static_cast<uint64_t>(a.num_blocks) * a.block, static_cast<uint64_t>(a.d), static_cast<uint64_t>(a.hk) * a.d,
                      static_cast<uint32_t>(a.d), 1, static_cast<uint32_t>(box), swizzle, row_fetch(a.d));
}

template <int D>
int launch_join(const CacheFewParams& f, int rows, int ctas, cudaStream_t stream) {
  auto kernel = rows == 4 ? cache_few_join_kernel<D, 4> : rows == 8 ? cache_few_join_kernel<D, 8> : rows == 16 ? cache_few_join_kernel<D, 16>
                : rows == 32 ? cache_few_join_kernel<D, 32> : cache_few_join_kernel<D, 64>;
  return launch_chained(kernel, dim3(f.a.hk, f.a.batch, rows / 4), dim3(128), 0, stream, 0, f, ctas);
}

// One launch over up to kFewSequences sequences; rows of sequences without cu_q begin at first_row.
int launch_cache_few(const CacheAttnArgs& a, int rows, int first_row, cudaStream_t stream) {
  CacheFewParams f = {};
  f.a = cache_params(a);
  CacheAttnParams& p = f.a;
  p.first_row = first_row;
  const int64_t tiles = (static_cast<int64_t>(a.table_width) * a.block + kCaTile - 1) / kCaTile + 1;
  if (tiles * a.hk * a.batch > 0x7FFFFFFFll) return -7;
  const int ctas = sm_count();
  p.po = static_cast<float*>(a.scratch);
  p.pml = p.po + static_cast<int64_t>(ctas) * 4 * rows * a.d;
  f.pre = reinterpret_cast<int*>(p.pml + static_cast<int64_t>(ctas) * 4 * rows * 2);
  const bool f8 = a.k_scale != nullptr;
  p.per_tile = rows / p.group;
  int r = make_tmap_3d(&f.tma_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.q, static_cast<uint64_t>(a.d), static_cast<uint64_t>(a.hq),
                       static_cast<uint64_t>(a.total_q), static_cast<uint64_t>(a.d) * 2, static_cast<uint64_t>(a.q_ld) * 2,
                       static_cast<uint32_t>(f8 ? a.d : 64), static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.per_tile),
                       f8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B);
  if (r != 0) return -10 + r;
  if (f8) {
    if (!al16(a.k_scale) || !al16(a.v_scale)) return -5;
    f.ks = static_cast<const uint8_t*>(a.k_scale); f.vs = static_cast<const uint8_t*>(a.v_scale);
    r = code_map(&f.tma_k, a, a.k, p.box, a.d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
    if (r == 0) r = code_map(&f.tma_v, a, a.v, p.box, CU_TENSOR_MAP_SWIZZLE_NONE);
  } else {
    const int64_t slots = static_cast<int64_t>(a.num_blocks) * a.block;
    r = page_map(&f.tma_k, a, a.k, slots, p.box);
    if (r == 0) r = page_map(&f.tma_v, a, a.v, slots, p.box);
  }
  if (r != 0) return -20 + r;
  // no more CTAs than the table has room for tiles
  const int64_t most = tiles * a.hk * a.batch / kFewLeast;
  const unsigned grid = static_cast<unsigned>(most < 1 ? 1 : most < ctas ? most : ctas);
  if (a.d == 128) r = f8 ? run_cache_few<128, true>(f, rows, grid, stream) : run_cache_few<128, false>(f, rows, grid, stream);
  else r = f8 ? run_cache_few<64, true>(f, rows, grid, stream) : run_cache_few<64, false>(f, rows, grid, stream);
  if (r != 0) return r;
  return a.d == 128 ? launch_join<128>(f, rows, grid, stream) : launch_join<64>(f, rows, grid, stream);
}

// One launch over the sequences of `a`; rows of sequences without cu_q begin at first_row.
int launch_cache_tiles(const CacheAttnArgs& a, int first_row, cudaStream_t stream) {
  const CacheGrid g = cache_grid(a);
  CacheAttnParams p = cache_params(a);
  p.per_tile = g.per_tile;
  int r = make_tmap_3d(&p.tma_q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, a.q, static_cast<uint64_t>(a.d), static_cast<uint64_t>(a.hq),
                       static_cast<uint64_t>(a.total_q), static_cast<uint64_t>(a.d) * 2, static_cast<uint64_t>(a.q_ld) * 2, 64,
                       static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.per_tile));
  if (r != 0) return -10 + r;
  const bool wide = a.k_scale != nullptr;
  p.room = widened_room(a);
  const int64_t slots = wide ? static_cast<int64_t>(a.batch) * p.room : static_cast<int64_t>(a.num_blocks) * a.block;
  if (slots >= (1ll << 31)) return -3;
  if (wide) {
    p.box = kCaTile;
    p.table = nullptr;
  }
  char* wide_k = static_cast<char*>(a.scratch) + part_bytes(a, 0);
  char* wide_v = wide_k + slots * a.hk * a.d * 2;
  r = page_map(&p.tma_k, a, wide ? wide_k : a.k, slots, p.box);
  if (r != 0) return -20 + r;
  r = page_map(&p.tma_v, a, wide ? wide_v : a.v, slots, p.box);
  if (r != 0) return -30 + r;
  p.two = g.two; p.items = g.items * a.splits;
  p.first_row = first_row;
  p.po = static_cast<float*>(a.scratch);
  p.pml = p.po + (a.splits > 1 ? a.total_q * a.hq * a.splits * a.d : 0);
  if (wide) {
    CacheWidenArgs w = {a.k, a.v, a.k_scale, a.v_scale, wide_k, wide_v, a.table, a.lens, a.cu_q, a.table_width, a.block,
                        a.num_blocks, a.hk, p.room, a.max_q, p.window, p.first, a.status};
    const int64_t blocks = (static_cast<int64_t>(p.room) * 2 * a.hk * (a.d / 16) + 255) / 256;
    if (blocks > 0x7FFFFFFFll || a.batch > 65535) return -7;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.batch));
    (a.d == 128 ? cache_widen_kernel<128> : cache_widen_kernel<64>)<<<grid, 256, 0, stream>>>(w);
    r = static_cast<int>(cudaGetLastError());
    if (r != 0) return r;
  }
  const int sms = sm_count();
  const unsigned grid = static_cast<unsigned>(p.items < sms ? p.items : sms);
  r = a.d == 128 ? run_cache_attn<128>(p, grid, stream) : run_cache_attn<64>(p, grid, stream);
  return r != 0 || a.splits == 1 ? r : launch_merge(p, a.d, stream);
}

}  // namespace

int launch_cache_attn(const CacheAttnArgs& a, cudaStream_t stream) {
  if (a.total_q <= 0 || a.batch <= 0) return 0;
  int r = check(a);
  if (r != 0) return r;
  const int few = few_rows(a);
  if (few == 0 && a.splits < 1) return -6;
  if (few == 0 && a.k_scale == nullptr) return a.splits > 1 && a.scratch == nullptr ? -8 : launch_cache_tiles(a, 0, stream);
  const int at_once = few != 0 ? kFewSequences : a.wide_batch;
  if (a.scratch == nullptr || at_once < 1) return -8;
  for (int b = 0; b < a.batch && r == 0; b += at_once) {
    CacheAttnArgs part = a;
    part.batch = a.batch - b < at_once ? a.batch - b : at_once;
    part.table += static_cast<int64_t>(b) * a.table_width;
    part.lens += b;
    if (a.cu_q != nullptr) part.cu_q += b;
    part.zero_rest = a.zero_rest & ((b + part.batch == a.batch ? 1 : 0) | (b == 0 ? 2 : 0));
    r = few != 0 ? launch_cache_few(part, few, b, stream) : launch_cache_tiles(part, b, stream);
  }
  return r;
}

}  // namespace yv
