// Attention over the 8-bit cache for many rows: which launches take these kernels, for new tokens in a line.
#include "ktir_kv8_tile_dev.h"

namespace ktir {

template <int CODE>
static void tile_go(const ktir_kv8_attn_t& d, int64_t slots, hipStream_t st) {
  const dim3 grid((unsigned)(slots * d.cache.heads));
  const int D = (int)d.cache.columns;
  if (D <= 64) hipLaunchKernelGGL((kv8_attn_tile<CODE, 1, 1, 8, false, false>), grid, dim3(512), 0, st, d, KV8Mask{}, (uint32_t)slots, 0, 0, device_error_flag());
  else if (D <= 128) hipLaunchKernelGGL((kv8_attn_tile<CODE, 2, 1, 8, false, false>), grid, dim3(512), 0, st, d, KV8Mask{}, (uint32_t)slots, 0, 0, device_error_flag());
  else hipLaunchKernelGGL((kv8_attn_tile<CODE, 4, 1, 4, false, false>), grid, dim3(256), 0, st, d, KV8Mask{}, (uint32_t)slots, 0, 0, device_error_flag());
}

// Whether a launch takes this kernel, and its tiles of rows for each KV head.  With fewer
// than 128 workgroups the kernel of few rows, which spreads the keys as well, is faster (128
// columns): the last 512 of 4096 tokens (72 tiles) 86 us there and 156 here, the last 700 (88) 120
// and 157, the last 1024 (136) 148 and 157, the last 1400 (176) 202 and 164, 2048 alone (264) 120 and 93,
// 16 sequences of 64 after 1984 (128) 103 and 92, 20 (160) 125 and 90.  With 64 columns 16 sequences (128)
// take 75 and 73, the last 1024 (136) 114 and 123; with 256 this kernel gains later: the last 512 (136)
// 176 and 273, 8 sequences of 300 after 1700 (332) 249 and 275, 32 of 40 after 960 (576) 216 and 171.  And the
// kernel of few rows is where no tile is more than half full: 16 sequences of 20 (80 rows of 256) 50 and 87.
bool kv8_tile_takes(const ktir_kv8_attn_t& d, int64_t* slots) {
  const int64_t grp = d.q_heads / d.cache.heads, TM = d.cache.columns <= 128 ? 256 : 128;
  if (d.max_q * grp <= TM / 2) return false;
  *slots = d.max_q * grp > TM ? d.batch.tokens * grp / TM + d.batch.seqs : d.batch.seqs;
  return *slots * d.cache.heads >= 128;
}

int kv8_tile_launch(const ktir_kv8_attn_t& d, int64_t slots) {
  d.cache.dtype == KTIR_I8 ? tile_go<KTIR_I8>(d, slots, stream_of(d.stream)) : tile_go<KTIR_E4M3>(d, slots, stream_of(d.stream));
  KTIR_HIP_CHECK(hipGetLastError());
  return KTIR_OK;
}

}  // namespace ktir
