// Verification of drafted tokens: arguments shared by its kernels (drafts.cu) and the C ABI
// (capi_drafts.cu).
#pragma once

#include "common.cuh"

namespace bsb {

// Bytes of a row that one CTA of the first pass takes, and elements.
constexpr int kDraftPieceBytes = 16384;
template <typename T>
__host__ __device__ constexpr int draft_piece() {
  return kDraftPieceBytes / static_cast<int>(sizeof(T));
}
constexpr int kMaxDraftRanks = 8;  // CTAs of a sequence's cluster

struct DraftArgs {
  const void* logits;  // [rows, vocab]
  int64_t logits_stride;
  const int32_t* draft_tokens;  // [rows]; those of sequences' last rows are not looked at
  const int32_t* cu_rows;       // [seqs + 1]
  const float* uniforms;        // [rows]
  const float* temperature;     // [seqs], or null: temperature_all
  float temperature_all;
  const void* draft_probs;  // [rows, vocab] or null
  int64_t probs_stride;
  int32_t num_rows, num_seqs, vocab;
  int32_t pieces, ranks;
  float4* records;  // [rows, pieces]: maximum, sum of exponentials, index of the maximum
  int32_t* tokens;    // [rows]
  int32_t* accepted;  // [seqs]
  uint32_t* status;
};

int launch_verify_drafts(const DraftArgs& a, bool bf16, bool probs_bf16, cudaStream_t stream);

}  // namespace bsb
