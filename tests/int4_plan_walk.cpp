// Enumerates plans of the 4-bit product and walks each warp's sequence of chunks as the
// kernel does.  Prints the number of plans, then a line for each that is wrong.
#include <cstdio>
#include <cstdlib>

#include "int4_plan.h"

using namespace spr::int4;

namespace {

struct Span {
  int64_t tile;
  int chunk;  // the first
  bool operator==(const Span& o) const { return tile == o.tile && chunk == o.chunk; }
};

// The slots of scales of one warp with `tiles` tiles: what is wrong, or null.
const char* walk(const Shape& sh, int from, int to, int tiles) {
  const int lead = from % sh.span;
  Span slot[4];
  int read_at[4];  // the step that last read a slot
  for (int i = 0; i < 4; ++i) slot[i] = {-1, -1}, read_at[i] = -1;
  int64_t copy_tile = 0, at_tile = 0;
  int copy = from, at = from, copy_at = lead, use_at = lead, copy_slot = 0, use_slot = 0, step = 0;
  auto fetch = [&](bool first) -> const char* {
    if (copy_tile >= tiles) return nullptr;
    if (copy == from || copy_at == 0) {
      if (!first && read_at[copy_slot] == step) return "a slot is filled in the step that reads it";
      slot[copy_slot] = {copy_tile, copy};
      copy_slot = copy_slot + 1 == sh.slots ? 0 : copy_slot + 1;
    }
    copy_at = copy_at + 1 == sh.span ? 0 : copy_at + 1;
    if (++copy == to) copy = from, ++copy_tile, copy_at = lead;
    return nullptr;
  };
  for (int i = 0; i < kStages - 1; ++i) fetch(true);
  for (; at_tile < tiles; ++step) {
    const Span want = {at_tile, std::max(from, at - use_at)};
    if (!(slot[use_slot] == want)) return "a slot holds another span than the one at work";
    read_at[use_slot] = step;
    if (const char* bad = fetch(false)) return bad;
    const bool done = ++at == to;
    if (done) at = from, ++at_tile;
    use_at = done ? lead : use_at + 1 == sh.span ? 0 : use_at + 1;
    if (done || use_at == 0) use_slot = use_slot + 1 == sh.slots ? 0 : use_slot + 1;
  }
  return nullptr;
}

const char* check(const ForwardPlan& p, const Weights& w, int64_t rows) {
  const Shape& sh = p.sh;
  const int chunks = (w.blocks + kBlocks - 1) / kBlocks;
  if (sh.along < 1 || sh.tiles < 1 || sh.slices < 1 || p.grid < 1) return "no work is given out";
  if (sh.along * sh.tiles > most_warps(p.nt) || (sh.along > 1 && sh.tiles > 15)) return "too many warps or barriers";
  const int warp = kStages * kStageBytes + sh.slots * sh.slot_bytes + 2 * kTile * p.nt * 8 * 4;
  const int x = kBlocks * (p.ints ? p.pass_rows * p.parts * 32 + p.nt * 32 : p.pass_rows * p.parts * 64);
  if (p.smem < sh.along * sh.tiles * warp + sh.slice_chunks * x || p.smem > kSmem) return "shared memory";
  if ((int64_t)p.passes * p.pass_rows < rows || p.pass_rows * p.parts > p.nt * 8) return "rows are left out";
  if (sh.slots < 1 || sh.slots > 4) return "slots";
  int next = 0;
  for (int z = 0; z < sh.slices; ++z) {
    const int c0 = z * sh.slice_chunks, c1 = std::min(chunks, c0 + sh.slice_chunks);
    if (c0 != next || c1 <= c0) return "a slice's columns";
    next = c0;
    for (int wk = 0; wk < sh.along; ++wk) {
      const int from = c0 + wk * sh.warp_chunks, to = std::min(c1, from + sh.warp_chunks);
      if (from >= to) continue;
      if (from != next) return "a warp's columns";
      next = to;
      if (p.scale)
        if (const char* bad = walk(sh, from, to, 6)) return bad;
    }
    if (next != c1) return "columns are left out";
  }
  return next == chunks ? nullptr : "columns are left out";
}

uint64_t state = 88172645463325252ull;
int64_t draw(int64_t lo, int64_t hi) {
  state ^= state << 13, state ^= state >> 7, state ^= state << 17;
  return lo + (int64_t)(state % (uint64_t)(hi - lo + 1));
}

int64_t plans = 0, wrong = 0;
void one(int64_t rows, int64_t n, int64_t k, int group, int dtype, int64_t sms) {
  const Weights w = make_weights(nullptr, nullptr, 0, nullptr, n, k, group);
  // As the launch decides whether scales can be copied ahead, for every alignment and type.
  const bool whole = w.groups % 8 == 0 && (kBlocks % w.group_blocks == 0 || w.group_blocks % kBlocks == 0);
  for (int scale : {0, 2, 4}) {
    if (scale && !whole) continue;
    ++plans;
    const char* bad = check(plan_forward(rows, w, dtype, scale, sms), w, rows);
    if (bad && ++wrong <= 20)
      printf("rows %lld n %lld k %lld group %d dtype %d scale bytes %d SMs %lld: %s\n", (long long)rows, (long long)n,
             (long long)k, group, dtype, scale, (long long)sms, bad);
  }
}

}  // namespace

int main() {
  const int groups[] = {32, 64, 96, 128, 160, 256, 512, 1024, 16384};
  // Every remainder of the chunks, several slices, few and many tiles a warp.
  for (int dtype : {SPR_F32, SPR_BF16, SPR_F16})
    for (int64_t rows : {1, 2, 3, 4, 8, 9, 23, 70})
      for (int64_t n : {40, 15360, 61440, 245760})
        for (int64_t k = 32; k <= 16384; k += k < 1024 ? 32 : 256)
          for (int group : {32, 64, 128, 256}) one(rows, n, k, group, dtype, 148);
  for (int i = 0; i < 150000; ++i) {
    const int64_t k = draw(0, 3) ? draw(1, 16384) : draw(1, 1 << 20);
    one(draw(0, 3) ? draw(1, 32) : draw(1, 65535), draw(0, 1) ? draw(1, 300000) : draw(1, 5000), k, groups[draw(0, 8)],
        (int)draw(0, 2), draw(0, 3) ? 148 : draw(1, 160));
  }
  for (int64_t k : {1ll << 20, (1ll << 24) + 5, (1ll << 27) - 256, 1ll << 27})
    for (int group : {32, 128, 1 << 20})
      for (int64_t rows : {1, 8, 32, 65535})
        for (int dtype : {SPR_F32, SPR_BF16, SPR_F16}) one(rows, 7, k, group, dtype, 148);
  printf("%lld plans, %lld wrong\n", (long long)plans, (long long)wrong);
  return wrong != 0;
}
