// Internal: the beam-search operators' launch arguments, shared by their kernels and C entry
// points (beams.cu) and the engine's (engine.cu).
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "layout.h"

namespace xg {
namespace beams {

constexpr int32_t kMaxBeams = 64;        // beams of one group
constexpr int32_t kMaxCandidates = 128;  // candidates of one group
constexpr int32_t kMaxVocab = 1 << 20;   // tokens (a candidate's order is beam, then token, in one word)

// Which tokens of a row count: bit v of row r's words, from a table of rows, or, for the
// engine's slots, base[slot] | delta[slot] of each active slot (null pointers and inactive
// slots: every token).
struct RowMasks {
  const uint32_t* words = nullptr;  // [rows][stride]
  int64_t stride = 0;
  const int32_t* slots = nullptr;  // the engine's: slot of each row
  const uint32_t* const* base = nullptr;
  uint32_t* const* delta = nullptr;
  const int32_t* active = nullptr;
  int32_t max_slots = 0;
};

struct SelectArgs {
  const char* logits = nullptr;
  int64_t row_stride = 0;  // elements
  int32_t dtype = 0, groups = 0, beams = 0, vocab = 0, candidates = 0, end_token = -1, renormalize = 1;
  const float* scores = nullptr;
  const uint8_t* finished = nullptr;
  RowMasks masks;
  float* out_scores = nullptr;
  int32_t* out_beams = nullptr;
  int32_t* out_tokens = nullptr;
  uint8_t* out_finished = nullptr;
  char* workspace = nullptr;
  int64_t workspace_bytes = 0;
};

// Checked, then launched on `stream` (status codes and messages as the C ABI's).
int select(const SelectArgs& args, cudaStream_t stream);
int reorder(const XgRowTensor* tensors, int32_t count, const int32_t* parents, int32_t groups, int32_t beams,
            const int32_t* lengths, const int32_t* rows, cudaStream_t stream);

}  // namespace beams
}  // namespace xg
