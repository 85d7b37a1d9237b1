// Launch descriptor of beam search's selection, shared by its kernels and the C-ABI layer.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace va {

constexpr int kBeamsMost = 64;         // beams of a prompt
constexpr int kBeamsCount = 64;        // continuations that a prompt gets
constexpr int kBeamsVocab = 1 << 18;
constexpr int kBeamsRows = 1 << 20;
constexpr int kBeamsCell = 512;        // the smallest cell: 8 numbers per lane of a wave
constexpr int kBeamsCells = 4096;      // cells of a prompt at most
constexpr int kBeamsWaves = 4;         // of a work-group that reads logits
// Work-groups that read logits, and the fewest cells that one reads (two per wave).
constexpr int kBeamsGroups = 2048, kBeamsFewCells = 8;

// How a call's logits are cut: cells of `cell` numbers of a row (the last one may be shorter), `splits`
// work-groups per row. Workspace: the largest number of every cell (rows x cells), then {reference,
// sum of powers of two over it} of every wave (rows x splits x kBeamsWaves), fp32.
struct BeamsLayout {
  int cell, cells, splits;
  int64_t sums, words;  // offset of the waves' pairs; fp32 words in all
};
inline BeamsLayout beams_layout(int64_t rows, int64_t beams, int64_t vocab) {
  BeamsLayout l;
  l.cell = kBeamsCell;
  while (beams * ((vocab + l.cell - 1) / l.cell) > kBeamsCells) l.cell *= 2;
  l.cells = (int)((vocab + l.cell - 1) / l.cell);
  const int64_t most = (l.cells + kBeamsFewCells - 1) / kBeamsFewCells;
  const int64_t wanted = rows > 0 ? (kBeamsGroups + rows - 1) / rows : 1;
  l.splits = (int)(wanted < most ? wanted : most);
  l.sums = (rows * l.cells + 3) / 4 * 4;
  l.words = l.sums + rows * l.splits * kBeamsWaves * 2;
  return l;
}

struct BeamsArgs {
  const void* logits;
  int dtype;
  int64_t row_stride;  // elements
  int groups, beams, vocab;
  const float* scores;
  const uint8_t* ended;  // null: none
  int end_token;
  int count;
  BeamsLayout layout;
  float* workspace;
  float* scores_out;
  int32_t* parents_out;
  int32_t* tokens_out;
  hipStream_t stream;
};

hipError_t launch_select_beams(const BeamsArgs& a);

}  // namespace va
