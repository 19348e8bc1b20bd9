// Sizes of the sampling operators' launches, shared by the checks of sampling_abi.cpp and the
// launchers. Plain C++, so that it can be checked without a GPU.
#pragma once
#include <stdint.h>

namespace ci8 {

constexpr int64_t kMostVocab = 1 << 24, kMostVerified = 1 << 14;
constexpr int kSampleThreads = 256, kRowThreads = 1024, kClearThreads = 256;
constexpr int64_t kSamplingWorkspaceBytes = 1 << 20;

// Parts of a row of `length` values.
struct Chunks {
  int length, count;
};

// token_probs: whole multiples of what a workgroup's threads hold at once, as many as fill 256 CUs.
constexpr int kProbsPart = 4096;
inline Chunks probs_parts(int64_t tokens, int64_t vocab) {
  const int64_t steps = (vocab + kProbsPart - 1) / kProbsPart;
  int64_t parts = tokens < 256 ? 256 / tokens : 1;
  if (parts > steps) parts = steps;
  const int64_t each = (steps + parts - 1) / parts;
  return {int(each * kProbsPart), int((steps + each - 1) / each)};
}

// Two kernels: chunks of a row of up to kChunkPacks * 1024 values, 256 of them at least where rows are
// that long, and 256 of a row at most, a thread of the second kernel each. One row of 262208 BF16
// logits 8.6 us in 129 chunks, 29 as a whole row; of 1000000 8.3 and 101.
constexpr int kChunkPacks = 8;
inline Chunks probs_chunks(int64_t tokens, int64_t vocab) {
  const int step = kSampleThreads * 4;
  const int64_t least = (vocab + step * kSampleThreads - 1) / (step * kSampleThreads);
  int64_t packs = tokens * vocab / step / 256;
  if (packs < least) packs = least;
  if (packs > kChunkPacks) packs = kChunkPacks;
  const int64_t length = packs * step;
  return {int(length), int((vocab + length - 1) / length)};
}
// For few rows, and where whole rows of BF16 leave part of a second round of 256 workgroups empty, if the
// sums fit threads and workspace. us, chunks and whole rows, BF16: 1 x 50001 8.1 and 9.5, 52 x 50001 10.0 and
// 13.5, 52 x 152000 13.3 and 24.5, 128 x 152000 26.6 and 34.3, 400 x 50001 30.1 and 37.4; but 256 x 50001 19.4
// and 18.0, 512 x 152000 124 and 110, 52 x 32000 8.8 and 7.8. FP32: 128 x 152000 46 and 58, but 400 x 81000
// 75 and 59. The rule leaves out what later rounds leave empty (BF16 513 x 152000 114 and 128, 520 x 50001 35
// and 42, but 700 x 152000 163 and 159) and that whole FP32 rows past 81920 values are read three times
// (300 x 152000 84 and 119, 256 x 152000 72 and 71): such calls would gain by chunks.
constexpr int64_t kFewVocab = 9 * kProbsPart;
inline bool probs_in_chunks(int64_t tokens, int64_t vocab, const Chunks& c, bool bf16) {
  return vocab >= kFewVocab && (tokens < 192 || (bf16 && tokens > 256 && tokens < 512)) &&
         c.count <= kSampleThreads && tokens * c.count * 8 <= kSamplingWorkspaceBytes;
}

// verify_drafts. With `rounds`, where sums may be needed after each row that fails and twice at the end:
// a workgroup a chunk of 2048 tokens at least, about 1024 of all sequences, whose sums fit the workspace
// for all rounds. Else a wave a chunk, four times as many. One chunk, and one workgroup, where the
// vocabulary is small: us, one and several, 6 rows over 8000 tokens 9.5 and 11.2, 64 x 6 9.9 and 15.9; over
// 16000 10.9 and 10.8, 12.7 and 12.3; over 32000 18.8 and 11.0.
constexpr int kMostRounds = 64 + 2, kMostChunks = 256, kOneChunk = 10000, kPickThreads = 512;
inline Chunks verify_chunks(int64_t seqs, int64_t vocab, bool rounds) {
  if (vocab <= kOneChunk) return {int(vocab), 1};
  int64_t count = (rounds ? 1024 : 4096) / seqs;
  const int64_t fits = kSamplingWorkspaceBytes / 8 / (seqs * kMostRounds);
  if (rounds && count > fits) count = fits;
  if (count > kMostChunks) count = kMostChunks;
  if (count > vocab / (rounds ? 2048 : 512)) count = vocab / (rounds ? 2048 : 512);
  if (count <= 1) return {int(vocab), 1};
  const int64_t length = ((vocab + count - 1) / count + 3) / 4 * 4;
  return {int(length), int((vocab + length - 1) / length)};
}

// Times that a workgroup looks for a sum of another, 0.16 us each, before it computes it: 82 us, about what
// it takes to add up 62 chunks of 2048 tokens (94 us, a workgroup alone; 15 chunks 25, 244 350), so that
// the wait, which ends at once where all workgroups run, costs no more than the sums where some do not.
#ifndef CI8_MOST_POLLS
#define CI8_MOST_POLLS (1 << 9)
#endif
constexpr int kMostPolls = CI8_MOST_POLLS;

}  // namespace ci8
