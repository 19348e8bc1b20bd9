// Sizes of the sampling operators' launches, shared by the checks of sampling_abi.cpp and the
// launchers. Plain C++, so that it can be checked without a GPU.
#pragma once
#include <stdint.h>

namespace ci8 {

constexpr int64_t kMostVocab = 1 << 24, kMostVerified = 1 << 14;
constexpr int kSampleThreads = 256, kRowThreads = 1024;
constexpr int64_t kSamplingWorkspaceBytes = 1 << 20;

// A vocabulary is cut into chunks of a multiple of 1024 tokens, 2048 at least, so that few rows are
// about 1024 workgroups.
struct Chunks {
  int length, count;
};
inline Chunks vocab_chunks(int64_t rows, int64_t vocab) {
  int64_t length = (rows * vocab + 1023) / 1024;
  if (length > vocab) length = vocab;
  if (length < 2048) length = 2048;
  length = (length + 1023) / 1024 * 1024;
  return {int(length), int((vocab + length - 1) / length)};
}

// token_probs: rows from here on take a workgroup each, which needs no workspace.
constexpr int64_t kManyRows = 512;

}  // namespace ci8
