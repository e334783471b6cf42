// Parameters and per-type launchers of the selective scan (selective_scan.cu).
#pragma once
#include <string.h>

#include "mixer_common.cuh"

namespace flare {
namespace scan {

constexpr int kTile = 32;  // tokens of a tile, and between two kept states

constexpr int block_channels(int S) { return S == 32 ? 32 : 64; }  // of a block, in either direction

struct ScanParams {
  flare_scan_args_t a;
  int wide;       // rows of x, dt, z, y, dy and their gradients in 16-byte pieces
  int channels;   // of a group
  int blocks_c;   // blocks along a group's channels
  int segments, seg_tokens;  // tokens of a row are cut into segments of whole tiles
  // of every segment: what it leaves behind from zero, then (after the join) what it starts from; the sum of its deltas,
  // -infinity: a document begins in it
  float* carry;      // [B][segments][C][S]
  float* decay;      // [B][segments][C]
  float* partial_bc; // [B][N][G * blocks_c][2 S]
  float* partial_w;  // [B * segments][weight_sums]: dA, dD, dt_bias
};

// (whole 16 bytes)
__host__ __device__ inline int64_t weight_sums(const flare_scan_args_t& a) { return ((int64_t)a.C * (a.S + 2) + 3) / 4 * 4; }

enum Pass { FORWARD, FORWARD_ENDS, BACKWARD, BACKWARD_ENDS, DECODE };

// one of these per element type
template <typename T>
int launch(Pass pass, const ScanParams& p, cudaStream_t stream);

}  // namespace scan
}  // namespace flare
