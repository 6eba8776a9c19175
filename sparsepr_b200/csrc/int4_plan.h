// How the forward product of int4.cu spreads over a GPU: host arithmetic alone, so that
// plans can be enumerated without one.
#pragma once

#include <stdint.h>

#include <algorithm>

#include "../../include/sparsepr_b200.h"

namespace spr {
namespace int4 {

constexpr int most_warps(int nt) { return nt == 1 ? 16 : nt == 2 ? 12 : 8; }  // of a CTA: what shared memory holds
constexpr int kTile = 16;  // weight rows of a product
constexpr int kBlocks = 8;  // blocks of 32 codes in one stage of a warp's ring: 128 bytes of a row
constexpr int kStages = 4;
constexpr int kStageBytes = kTile * kBlocks * 16;
constexpr int kLimbs = 4;

// The weights as the kernels take them.
struct Weights {
  const uint8_t* packed;
  const void* scales;
  const uint8_t* zeros;
  int scale_dtype;
  int64_t n;
  int k, groups, group_blocks, blocks;  // blocks of 32 codes a row, the unused ones of the last group too
};

// Bytes that eight groups' scales and zeros take in a slot.
constexpr int piece_bytes(int scale) { return 8 * (scale ? scale : 4) + 8; }

// Where a launch's warps work: `along` warps of a CTA share a tile, each with
// `warp_chunks` neighbouring chunks of the CTA's slice of the columns; `tiles` such
// teams to a CTA.
struct Shape {
  int along, tiles, warp_chunks;
  int slice_chunks, slices;
  int span, pieces, places;  // chunks of a span, its pieces a row, the places they take
  int slots, slot_bytes;     // a warp's slots of scales and zeros
};

inline int parts_of(int dtype) { return dtype == SPR_BF16 ? 1 : dtype == SPR_F16 ? 2 : 3; }

inline Weights make_weights(const uint8_t* packed, const void* scales, int scale_dtype, const uint8_t* zeros, int64_t n,
                            int64_t k, int group) {
  Weights w{packed, scales, zeros, scale_dtype, n, (int)k, (int)((k + group - 1) / group), group / 32, 0};
  w.blocks = w.groups * w.group_blocks;
  return w;
}

constexpr int kSmem = 225 * 1024;  // of a CTA at most, less what a kernel declares itself

struct ForwardPlan {
  Shape sh;
  bool ints;
  int scale;  // bytes of a scale that is copied ahead, 0: none is
  int parts, pass_rows, passes, nt, gb, grid, smem;
};

// Slots of scales and zeros that a warp needs.  After the chunk at work the warp copies the
// one three ahead, and with a span's first chunk the span's values, into the slot that it
// read `slots` spans before.  All lanes have met since those reads only if they belong
// to an earlier chunk, so the slots - 1 spans between must have three chunks together.
// Four slots always do.  Where warps and slices begin on whole spans (of at least four
// chunks), the last slice's end is the one place that cuts a span short: two slots do if
// that rest has three chunks or none, three if it has two.
inline int span_slots(int scale, int span, int chunks, int slice_chunks, int slices, int warp_chunks) {
  if (!scale) return 2;  // stored by the warp itself, chunk by chunk
  if (warp_chunks % span || slice_chunks % span) return 4;
  const int rest = (chunks - (slices - 1) * slice_chunks) % span;
  return rest == 1 ? 4 : rest == 2 ? 3 : 2;
}

// Rows a pass: what 32 columns of a product hold.  16-bit rows go to the integer
// products while one pass holds them; more of them take fewer columns as bf16 parts.
// The rest weighs, by estimates of the time: slices of the weight's columns (each CTA
// then stages less of x, which leaves room for more warps, but the slices' sums have to
// be joined) against warps on a tile (idle warps at the last round, and sums to join).
inline ForwardPlan plan_forward(int64_t rows, const Weights& w, int dtype, int scale, int64_t sms) {
  ForwardPlan p{};
  p.ints = dtype != SPR_F32 && rows <= 32 / kLimbs;
  p.parts = p.ints ? kLimbs : parts_of(dtype);
  p.pass_rows = (int)std::min<int64_t>(rows, 32 / p.parts);
  p.passes = (int)((rows + p.pass_rows - 1) / p.pass_rows);
  const int cols = p.pass_rows * p.parts;
  p.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  p.gb = w.group_blocks % 8 == 0 ? 8 : w.group_blocks % 4 == 0 ? 4 : w.group_blocks % 2 == 0 ? 2 : 1;
  p.scale = scale;
  Shape& sh = p.sh;
  sh.span = w.group_blocks * ((3 + w.group_blocks) / w.group_blocks);
  sh.pieces = sh.span / w.group_blocks;
  sh.places = p.scale ? sh.pieces | 1 : 1;
  sh.slot_bytes = kTile * sh.places * piece_bytes(p.scale);

  const int chunks = (w.blocks + kBlocks - 1) / kBlocks;
  const int64_t tiles = (w.n + kTile - 1) / kTile;
  const int chunk_bytes = kBlocks * (p.ints ? cols * 32 + p.nt * 32 : cols * 64);
  const int warp_most = kStages * kStageBytes + 4 * sh.slot_bytes + 2 * kTile * p.nt * 8 * 4;
  const int least = std::max(1, (int)(((int64_t)chunks * chunk_bytes + kSmem - 8 * warp_most - 1) /
                                      (kSmem - 8 * warp_most)));  // slices that leave room for eight warps
  double best = 1e30;
  for (int slices = least; slices <= std::min(chunks, 2 * least + 3); ++slices) {
    const int slice_chunks = (chunks + slices - 1) / slices;
    if ((chunks + slice_chunks - 1) / slice_chunks != slices) continue;
    const int64_t work = tiles * p.passes * slices;
    for (int along = 1; along <= 8 && along <= slice_chunks; along *= 2) {
      const int warp_chunks = (slice_chunks + along - 1) / along;
      const int slots = span_slots(p.scale, sh.span, chunks, slice_chunks, slices, warp_chunks);
      const int warp_bytes = kStages * kStageBytes + slots * sh.slot_bytes + 2 * kTile * p.nt * 8 * 4;
      const int fit = std::min(most_warps(p.nt), (kSmem - slice_chunks * chunk_bytes) / warp_bytes);
      const int64_t team_tiles = std::min<int64_t>(fit / along, (work + sms - 1) / sms);
      if (team_tiles < 1) continue;
      // Microseconds: a chunk of a warp (more where many warps share the schedulers), a
      // round's end (with a wait for the tile's other warps), the join.
      const int64_t rounds = (work + team_tiles * sms - 1) / (team_tiles * sms);
      const double chunk = (p.ints ? 0.7 : 0.9) * (1 + 0.25 * (p.nt - 1)) * std::max(1.0, along * team_tiles / 12.0);
      const double time = rounds * (warp_chunks * chunk + (along > 1 ? 0.7 : 0.3)) +
                          (slices > 1 ? 3 + slices * (double)rows * (double)w.n * 8 / 5e6 : 0);
      if (time >= best * 0.98) continue;
      best = time;
      sh.along = along;
      sh.tiles = (int)team_tiles;
      sh.warp_chunks = warp_chunks;
      sh.slice_chunks = slice_chunks;
      sh.slices = slices;
      sh.slots = slots;
      p.smem = along * (int)team_tiles * warp_bytes + slice_chunks * chunk_bytes;
    }
  }
  const int64_t teams = (tiles + sh.tiles - 1) / sh.tiles;
  p.grid = (int)std::min(teams, std::max<int64_t>(1, sms / (p.passes * sh.slices)));
  return p;
}

}  // namespace int4
}  // namespace spr
