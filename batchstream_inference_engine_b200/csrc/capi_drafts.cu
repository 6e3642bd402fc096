// C ABI of the verification of drafted tokens (declared in include/batchstream_b200.h).
// Validation, messages and launch rules as in capi.cu.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdarg>
#include <cstdio>

#include "../../include/batchstream_b200.h"
#include "drafts.cuh"

namespace bsb {
// capi.cu: messages, launch count, SMs of the current device.
void set_last_error(const char* message);
void add_kernel_launches(int n);
int sm_count(int* sms);
}  // namespace bsb

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  bsb::set_last_error(buf);
  return code;
}

#define BS_CHECK(cond, ...)                                \
  do {                                                     \
    if (!(cond)) return fail(BS_ERR_INVALID, __VA_ARGS__); \
  } while (0)

constexpr int64_t kInt32Max = 2147483647ll;

// Pieces of a row: as many as it has when it begins at the end of a 16-byte unit.
int64_t pieces_of(int64_t vocab, int32_t dtype) {
  const int64_t size = dtype == BS_BF16 ? 2 : 4, shift = 16 / size - 1;
  return ((vocab + shift) * size + bsb::kDraftPieceBytes - 1) / bsb::kDraftPieceBytes;
}

int check_sizes(int64_t num_rows, int64_t vocab, int32_t dtype) {
  BS_CHECK(dtype == BS_BF16 || dtype == BS_F32, "logits must be bfloat16 or float32");
  BS_CHECK(num_rows >= 0 && num_rows <= kInt32Max, "num_rows out of range");
  BS_CHECK(vocab > 0, "vocab must be positive");
  if (vocab > (1ll << 30) || num_rows * pieces_of(vocab, dtype) > kInt32Max) {
    return fail(BS_ERR_UNSUPPORTED, "too many rows or tokens");
  }
  return BS_OK;
}

}  // namespace

extern "C" {

int bs_verify_drafts_workspace_bytes(int64_t num_rows, int64_t vocab, int32_t dtype,
                                     uint64_t* bytes_out) {
  BS_CHECK(bytes_out != nullptr, "bytes_out is null");
  if (int rc = check_sizes(num_rows, vocab, dtype)) return rc;
  *bytes_out = static_cast<uint64_t>(num_rows * pieces_of(vocab, dtype)) * sizeof(float4);
  return BS_OK;
}

int bs_verify_drafts(const void* logits, int64_t logits_row_stride, int32_t dtype,
                     int64_t num_rows, int64_t vocab, const int32_t* draft_tokens,
                     const int32_t* cu_rows, int64_t num_seqs, const float* uniforms,
                     const float* temperatures, double temperature, const void* draft_probs,
                     int64_t probs_row_stride, int32_t probs_dtype, int32_t* tokens_out,
                     int32_t* accepted_out, void* workspace, uint64_t workspace_bytes,
                     uint32_t* status, void* stream) {
  if (int rc = check_sizes(num_rows, vocab, dtype)) return rc;
  BS_CHECK(num_seqs >= 0 && num_seqs <= kInt32Max / bsb::kMaxDraftRanks, "num_seqs out of range");
  BS_CHECK(num_rows <= 1 || logits_row_stride >= vocab, "logits rows must hold the vocabulary");
  BS_CHECK(draft_probs == nullptr || probs_dtype == BS_BF16 || probs_dtype == BS_F32,
           "draft_probs must be bfloat16 or float32");
  BS_CHECK(draft_probs == nullptr || num_rows <= 1 || probs_row_stride >= vocab,
           "draft_probs rows must hold the vocabulary");
  const float t = static_cast<float>(temperature);
  BS_CHECK(temperatures != nullptr || (t >= 0.f && t <= 3.4028234e38f),
           "temperature must be finite and not negative");
  if (num_rows == 0 && num_seqs == 0) return BS_OK;
  BS_CHECK(cu_rows && (num_seqs == 0 || accepted_out) &&
               (num_rows == 0 || (logits && draft_tokens && uniforms && tokens_out)),
           "null pointer argument");
  const int64_t need = num_rows * pieces_of(vocab, dtype) * static_cast<int64_t>(sizeof(float4));
  if (need > 0 && (workspace == nullptr || workspace_bytes < static_cast<uint64_t>(need))) {
    return fail(BS_ERR_WORKSPACE, "workspace of %llu bytes is smaller than the %lld needed",
                static_cast<unsigned long long>(workspace_bytes), static_cast<long long>(need));
  }
  BS_CHECK((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0, "workspace must be 16-byte aligned");
  int sms = 0;
  if (int rc = bsb::sm_count(&sms)) return rc;
  bsb::DraftArgs a{};
  a.logits = logits;
  a.logits_stride = logits_row_stride;
  a.draft_tokens = draft_tokens;
  a.cu_rows = cu_rows;
  a.uniforms = uniforms;
  a.temperature = temperatures;
  a.temperature_all = t;
  a.draft_probs = draft_probs;
  a.probs_stride = probs_row_stride;
  a.num_rows = static_cast<int32_t>(num_rows);
  a.num_seqs = static_cast<int32_t>(num_seqs);
  a.vocab = static_cast<int32_t>(vocab);
  a.pieces = static_cast<int32_t>(pieces_of(vocab, dtype));
  // CTAs that draw a sequence's token: one per SM over the batch, 4096 tokens each at least.  us
  // with one a sequence / these / twice as many, of 151936 bf16 logits and draft probabilities,
  // four drafts each: 1 sequence 41 / 21 / 21, 8: 90 / 31 / 31, 32: 100 / 51 / 68, 64: 113 / 80 / 90.
  a.ranks = static_cast<int32_t>(std::max<int64_t>(
      1, std::min({int64_t{bsb::kMaxDraftRanks},
                   num_seqs > 0 ? int64_t{sms} / num_seqs : int64_t{1}, (vocab + 4095) / 4096})));
  a.records = static_cast<float4*>(workspace);
  a.tokens = tokens_out;
  a.accepted = accepted_out;
  a.status = status;
  const int rc = bsb::launch_verify_drafts(a, dtype == BS_BF16, probs_dtype == BS_BF16,
                                           static_cast<cudaStream_t>(stream));
  if (rc != 0) {
    return fail(BS_ERR_CUDA, "verify_drafts launch: %s",
                cudaGetErrorString(static_cast<cudaError_t>(rc)));
  }
  bsb::add_kernel_launches((num_rows > 0 ? 1 : 0) + (num_seqs > 0 ? 1 : 0));
  return BS_OK;
}

}  // extern "C"
