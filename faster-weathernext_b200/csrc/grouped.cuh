// Launch interface of the products grouped by expert (grouped_fwd.cu, grouped_bwd.cu, grouped.cu), called by grouped_abi.cu.
#pragma once

#include "linear.cuh"

namespace fwn {

constexpr int kGroupsMax = 1023;
constexpr int kGroupMaps = 7, kGroupFirsts = 3;

// Tiles (or runs) of `unit` rows that an expert's rows take; unit 0: one run, whatever they are. Without rows + unit, which may
// pass 2^31: a run of the weights' gradient takes millions of rows where few columns make few tiles.
constexpr int group_tiles(int rows, int unit) { return unit > 0 ? rows / unit + (rows % unit != 0 ? 1 : 0) : 1; }

// What a call's kernels read of the offsets, made on the device by one launch before them: the offsets in order and within
// the tensor, the tiles (or runs) before each expert, the experts' tensor maps, and zeros in the rows of no expert.
struct GroupSetup {
  const int32_t* given;      // [groups + 1]
  int groups;
  int64_t m;                 // rows
  int32_t* offsets;          // [groups + 1]
  int32_t* first[kGroupFirsts];   // [groups + 1] each; or null
  int unit[kGroupFirsts];    // rows of a tile (or run); 0: one run an expert, whatever its rows
  CUtensorMap* maps;         // [n_maps, groups]
  int n_maps;
  void* clear;               // m contiguous rows of clear_row bytes whose rows of no expert become 0; or null
  int64_t clear_row;
};
struct GroupMaps {
  CUtensorMap map[kGroupMaps];    // over all rows: the experts' copies end at their last
};
cudaError_t launch_group_setup(const GroupSetup& s, const GroupMaps& maps, cudaStream_t stream);

// kGroupRows: out = act(a b^T + bias), or (p.pre_grad) x act'(a b^T + bias); kGroupK: out = a^T b.
cudaError_t launch_grouped_forward(int tile, const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items,
                                   int sms, cudaStream_t stream);
cudaError_t launch_grouped_pre_grad(int tile, const CUtensorMap& tb, const LinearParams& p, const GroupParams& g, int64_t items,
                                    int sms, cudaStream_t stream);
cudaError_t launch_grouped_weights(int tile, const CUtensorMap& to, const LinearParams& p, const GroupParams& g, int64_t items,
                                   int sms, cudaStream_t stream);

// m <= kLinearRowsMax rows a of k contiguous values, b [groups, n, k]; rows of no expert become 0.
cudaError_t launch_grouped_rows(const void* a, int64_t lda, const void* b, int64_t ldb, int64_t b_stride, bool wide,
                                const int32_t* given, int groups, const LinearParams& p, cudaStream_t stream);

// x [m, n] (bf16 or float32) rounded to bf16 (cast not null) and, tile by tile of kCastRows rows, its column sums
// (part [tiles, n], not null), rows of an expert only; `most` tiles at most.
constexpr int kCastRows = 256;
cudaError_t launch_grouped_cast(const void* x, bool x_f32, int64_t ldx, int n, void* cast, int64_t ldc, float* part,
                                const GroupParams& g, int64_t most, bool wide, cudaStream_t stream);
// out[e, j] = sum of part's rows first[e] per to first[e + 1] per (at most `most` tiles of `per` rows in all).
cudaError_t launch_grouped_column_sum(const float* part, const int32_t* first, int groups, int64_t most, int per, int n, void* out,
                                      bool out_bf16, cudaStream_t stream);
// out[e] (bf16, [rows, n] contiguous) = sum over the expert's runs of part [runs, rows, ldp].
cudaError_t launch_grouped_run_sum(const float* part, const int32_t* first, int groups, int64_t rows, int n, int64_t ldp,
                                   void* out, cudaStream_t stream);

// The device error words of these files' kernels (read and cleared, after the stream was synchronised).
cudaError_t take_grouped_fwd_error(unsigned int* word);
cudaError_t take_grouped_bwd_error(unsigned int* word);
cudaError_t take_grouped_error(unsigned int* word);

}  // namespace fwn
