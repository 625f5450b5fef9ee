// Launchers of the operators of a paged cache (cache.cu): 8-bit keys and values, and attention over pages.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace yv {

// Rows of d numbers, 2 hk of them a token: e4m3 codes [blocks, block, hk, d] and one exponent byte (e8m0) [blocks, hk, block].
struct CacheRowsArgs {
  const void *k = nullptr, *v = nullptr;       // bf16 [tokens, hk * d], pitches below (writing)
  void *ko = nullptr, *vo = nullptr;           // bf16 [tokens, hk * d], contiguous (reading)
  int64_t k_ld = 0, v_ld = 0;
  void *k_codes = nullptr, *v_codes = nullptr;
  void *k_scale = nullptr, *v_scale = nullptr;
  const int* slots = nullptr;                  // [tokens], negative = none
  int64_t tokens = 0, num_slots = 0;
  int hk = 0, d = 0, block = 0;
  uint32_t* status = nullptr;
};
int launch_cache_write_fp8(const CacheRowsArgs& a, cudaStream_t stream);
int launch_cache_read_fp8(const CacheRowsArgs& a, cudaStream_t stream);

struct CacheAttnArgs {
  const void* q = nullptr;                     // bf16 [total_q, hq, d], pitch q_ld
  int64_t q_ld = 0, total_q = 0;
  void* o = nullptr;                           // bf16 [total_q, hq, d], pitch o_ld
  int64_t o_ld = 0;
  const void *k = nullptr, *v = nullptr;       // pages [blocks, block, hk, d]: bf16, or e4m3 codes with k_scale, v_scale
  const void *k_scale = nullptr, *v_scale = nullptr;
  const int* table = nullptr;                  // [batch, table_width]
  const int* lens = nullptr;                   // [batch]
  const int* cu_q = nullptr;                   // [batch + 1], null = one query a sequence
  int batch = 0, max_q = 0, hq = 0, hk = 0, d = 0, block = 0, num_blocks = 0, table_width = 0;
  int window = 0, first = 0;                   // 0 = no window
  float scale = 1.f;
  int splits = 1;                              // key ranges of a query block, see cache_attn_plan
  int zero_rest = 0;                           // rows of o that are cleared: 1 behind the last sequence, 2 in front of the first
  void* scratch = nullptr;                     // as many bytes as the plan says
  int wide_batch = 0;
  uint32_t* status = nullptr;
};
// Decides, from sizes alone (so that a captured call can be replayed), how a call runs: splits (where they are 0) and wide_batch are
// set; returns the bytes of scratch that it takes.
int64_t cache_attn_plan(CacheAttnArgs& a);
int launch_cache_attn(const CacheAttnArgs& a, cudaStream_t stream);

}  // namespace yv
