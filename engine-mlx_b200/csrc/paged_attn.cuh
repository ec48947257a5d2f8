// paged_attn.cuh — what the kernels of emx_sdpa_paged share: the pieces of a
// row's attention and where they are kept.
#pragma once
#include "paged_dev.cuh"

namespace emx {

constexpr float kLog2e = 1.4426950408889634f;

// Pieces of one part (own or shared): first[] by row and q head, more[] by worker.
struct Pieces {
  float* first_o;    // [n_rows * n_q][HD]
  float2* first_ml;  // [n_rows * n_q]
  float* more_o;     // [workers][rows of a tile][HD]
  float2* more_ml;   // [workers][rows of a tile]
};

struct PagedWork {
  PagedAttnArgs a;
  Pieces own, shared;
  int64_t* starts;  // [n_seqs + 1] tiles before each sequence (own part)
  Shares* shares;   // the own part's, for the join
  int own_workers, own_early, own_each;  // (see deal)
  int own_mt, shared_mt;      // rows of a tile
  int own_keys, shared_keys;  // positions of a tile
  // Shares of the shared part (its sizes are known to the host): `shared_per`
  // tiles each, in one line, or (shared_split > 0) shared_split workers to each
  // segment, so that none has tiles of two.
  int shared_per, shared_split;
};

// The shared part of a batch of many rows, on tcgen05 (paged_attn_tc.cu):
// tiles of kTcRows rows and kTcKeys positions, one worker a CTA.
constexpr int kTcRows = 256, kTcKeys = 128;
// Pages that are whole 8-row groups of the tiles' swizzle.
bool paged_shared_tc_takes(const PagedArgs& p);
cudaError_t paged_shared_tc_launch(const PagedWork& w, int num_sms, cudaStream_t st);

}  // namespace emx
