// Chunk attention for few packed query rows (paged_chunk_stream.hip), as
// paged_chunk.hip calls it.
#pragma once

#include "common.hpp"

namespace q3 {

// Packed query rows (token, head of the group) of a KV head that it takes at most: the
// columns of one product.  Two column groups for 17-32 rows (one-tile batches, to fit
// the registers) were slower than the staged tiles: 16 x 8 tokens behind 4,000, 32/8
// heads: 77.7 us against 55.5.
constexpr int kChunkStreamRows = 16;

struct ChunkStreamCall {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint16_t* k;
  int64_t k_blk, k_sh, k_slot;
  const uint16_t* v;
  int64_t v_blk, v_sh, v_slot;
  int64_t num_blocks;
  const int32_t* bt;
  int64_t bt_stride, max_rows, max_pages;
  const int32_t* seq_lens;
  const int32_t* row_ids;
  const int32_t* cu;
  uint16_t* o;
  int64_t o_st, o_sh;
  int64_t total;
  int B, Hkv, G, block_size;
  int rows;  // max_chunk * G
  float scale_log2;
};

bool chunk_streams(int B, int64_t rows);
size_t chunk_stream_workspace(int B, int rows);
int launch_chunk_stream(const ChunkStreamCall& c, void* workspace, hipStream_t s, const char* who);

}  // namespace q3
