// Product of a few rows with 4-bit weights under group scales, and its gradient
// with respect to the rows (layout and formula at spr_int4_linear in the header).
//   y[r][n] = sum_g scale[n][g] * sum_{k in g} x[r][k]*(code[n][k] - zero[n][g]) + bias[n]
//   dx[r][k] = sum_n (dy[r][n]*scale[n][g]) * (code[n][k] - zero[n][g])
// What bounds both is the codes' bytes: HBM gives an SM 23 bytes, 46 codes, a cycle,
// so a 16 x 32 block of codes has 44 instruction slots of the SM's four schedulers
// for everything.  Hence tensor-core products whose operand is a few instructions
// from the packed codes:
// * 16-bit x: integer products (m16n8k32).  The codes are the bytes w & 0x0f0f0f0f and
//   (w >> 4) & 0x0f0f0f0f; x is a 31-bit integer relative to its row's largest
//   magnitude (of the CTA's columns), in four signed bytes, each a column of the
//   product.  An inner sum is an exact integer.  A value far below the largest is
//   rounded at 2^-30 of it: beside the largest's own term less than an fp32 sum
//   rounds, and where that term is 0 small values still have bf16's 8 bits down to
//   2^-22 of it; below 2^-31 it is lost.
// * fp32 x, and more rows than the integer columns hold: bf16 products (m16n8k16).  A
//   code is the exact integer code - zero, and x is cut into as many bf16 parts as
//   its significand needs (bf16 1, fp16 2, fp32 3; exact), each a column.
// Measured on B200 (copy bandwidth 6.56 TB/s) under a sustained load, 245,760 x 5120
// codes: two bf16 rows, groups of 128 133 us (75% of the copy's bytes a second), one row,
// groups of 64 150 us (70%); the schedulers issue in 55% to 60% of all cycles, waiting
// for one another's products.  122,880 x 5120 codes: 9, 16 and 32 bf16 rows, groups of
// 128, 129, 145 and 301 us; one, two and three fp32 rows (three parts each), groups of 64,
// 109, 115 and 149 us.  The gradient has more to do a code (pairs of weight rows are
// formed, and the other operand for each group): two rows, groups of 128 200 us; 30,720 x
// 5120 four rows 75 us.
// The 5th-generation tensor instructions would take 128 weight rows a tile, from shared or
// tensor memory: the codes, once unpacked, would have to be written there, two to four
// times the bytes that were copied in.  Whether larger tiles win back those instructions
// was not measured.
#include <math.h>

#include <initializer_list>

#include "common.cuh"
#include "int4_plan.h"

namespace spr {

using namespace int4;

namespace {

__device__ __forceinline__ float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == SPR_F32) return __ldg((const float*)p + i);
  if (dtype == SPR_BF16) return to_f32(((const __nv_bfloat16*)p)[i]);
  return to_f32(((const __half*)p)[i]);
}

__device__ __forceinline__ void store_f32(void* p, int dtype, int64_t i, float v) {
  if (dtype == SPR_F32) ((float*)p)[i] = v;
  else if (dtype == SPR_BF16) ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
  else ((__half*)p)[i] = __float2half_rn(v);
}

// Part `part` of v in bf16 (the value's upper 8 significant bits, the next 8, the
// last 8), as the high half of a word.  What is not finite is in part 0 alone.
__device__ __forceinline__ uint32_t bf16_part(float v, int part) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u) return part ? 0u : (u & 0x007fffffu ? 0x7fff0000u : u);
  const float a = __uint_as_float(u & 0xffff0000u), rest = v - a;
  if (part == 0) return __float_as_uint(a);
  const float b = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
  return part == 1 ? __float_as_uint(b) : __float_as_uint(rest - b) & 0xffff0000u;
}
__device__ __forceinline__ uint32_t bf16_pair(uint32_t low, uint32_t high) { return __byte_perm(low, high, 0x7632); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_int(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes i and i + 4 of a word as bf16 integers 128 + code, less `zero` = 128 + zero
// in both halves: exact.
template <int I>
__device__ __forceinline__ uint32_t codes(uint32_t word, uint32_t zero) {
  uint32_t v;
  asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(v) : "r"(word >> (4 * I)));  // (a & b) | c
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v),
                                   *reinterpret_cast<const __nv_bfloat162*>(&zero));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// The rows as the kernels take them.
struct Rows {
  const void* x;
  int64_t stride;
  int dtype, parts, all, pass;  // columns a row, rows, rows a launch's pass takes
};

// A warp's ring holds the codes of 16 weight rows by 256 columns a stage.  16-byte
// piece j of row r lies at j ^ (r's low bits reversed): lanes that read one, two or
// four words of neighbouring rows at once meet different banks.
__device__ __forceinline__ int turn(int row) { return (row & 1) << 2 | (row & 2) | (row >> 2 & 1); }
__device__ __forceinline__ int piece(int row, int j) { return row * 128 + ((j ^ turn(row)) << 4); }

template <int U>
__device__ __forceinline__ void load_words(const char* p, uint32_t (&w)[U]) {
  if constexpr (U == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (U == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// Scales and zeros of a warp's weight rows.  Where a row's lie in whole aligned pieces
// of eight groups (kScale, their bytes), those of a span of at least four chunks are
// copied with the span's first chunk: neighbouring lanes take neighbouring pieces, so
// that a row's are few memory requests.  Otherwise (kScale 0) the values of each
// chunk's segments (GB blocks, within one group) are loaded one chunk ahead into
// registers.  A slot holds a span; a row's pieces take an odd number of places, which
// keeps the rows in different banks.
template <int GB>
struct Values {
  static constexpr int kSegments = kBlocks / GB, kRegs = kSegments > 1 ? kSegments / 2 : 1;
  float scale[kRegs];
  uint8_t zero[kRegs];
  __device__ __forceinline__ void load(const Weights& w, int64_t row_at, int chunk, int lane) {
    // row_at: the first group of weight row lane & 15
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int g = min((chunk * kSegments + 2 * i + (lane >> 4)) * GB / w.group_blocks, w.groups - 1);
      scale[i] = load_as_f32(w.scales, w.scale_dtype, row_at + g);
      zero[i] = w.zeros ? __ldg(w.zeros + row_at + g) : 8;
    }
  }
  __device__ __forceinline__ void store(char* slot, int lane) const {  // as one piece a row, fp32
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int at = (lane & 15) * 8 + 2 * i + (lane >> 4);
      reinterpret_cast<float*>(slot)[at] = scale[i];
      reinterpret_cast<uint8_t*>(slot + kTile * 32)[at] = zero[i];
    }
  }
};

// Eight values of x from column k, zeros past the end.
__device__ __forceinline__ void load_x(const Rows& in, bool wide, int64_t at, int k, int k_end, float (&v)[8]) {
  if (wide && k + 8 <= k_end) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>((const char*)in.x + at * 2));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t h = (&u.x)[e >> 1] >> (16 * (e & 1)) & 0xffffu;
      v[e] = in.dtype == SPR_BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < k_end ? load_as_f32(in.x, in.dtype, at + e) : 0.f;
  }
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1,%2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ bool finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }

// The slice's x in shared memory in the order in which codes come apart.  A unit is
// U blocks, whose 4*U words go to the four lanes of a weight row U at a time: word j
// of lane t is word t*U + j of the unit.
// bf16: [block][column][lane] the pairs (k, k+4), (k+1, k+5), (k+2, k+6), (k+3, k+7)
// of the lane's word.  Integers: the bytes (k, k+2, k+4, k+6), (k+1, k+3, k+5, k+7).
template <int U>
__device__ __forceinline__ int x_place(int b, int word, int cols, int col) {
  const int at = (b % U) * 4 + word;  // within the unit
  return ((b / U * U + at % U) * cols + col) * 4 + at / U;
}

template <int U>
__device__ __forceinline__ void stage_bf16(const Weights& w, const Rows& in, int row0, int rows, int b0, int nb, float down,
                                           bool wide, uint4* xs) {
  const int cols = rows * in.parts;
  for (int i = threadIdx.x; i < nb * rows * 4; i += blockDim.x) {
    const int word = i & 3, b = (i >> 2) % nb, r = (i >> 2) / nb, k = (b0 + b) * 32 + word * 8;
    float v[8];
    load_x(in, wide, (int64_t)(row0 + r) * in.stride + k, k, w.k, v);
    for (int p = 0; p < in.parts; ++p) {
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = bf16_part(v[e] * down, p);
      xs[x_place<U>(b, word, cols, r * in.parts + p)] =
          make_uint4(bf16_pair(h[0], h[4]), bf16_pair(h[1], h[5]), bf16_pair(h[2], h[6]), bf16_pair(h[3], h[7]));
    }
  }
}

// Each row's largest magnitude of the slice's x, and whether any is not finite.
__device__ __forceinline__ void scan_x(const Weights& w, const Rows& in, int row0, int rows, int b0, int nb, bool wide,
                                       uint32_t* largest, int* bad) {
  const int words = nb * 4;
  if (threadIdx.x < 32) {
    largest[threadIdx.x] = 0;
    bad[threadIdx.x] = 0;
  }
  __syncthreads();
  for (int r = 0; r < rows; ++r) {
    uint32_t most = 0, any = 0;
    for (int i = threadIdx.x; i < words; i += blockDim.x) {
      const int k = b0 * 32 + i * 8;
      float v[8];
      load_x(in, wide, (int64_t)(row0 + r) * in.stride + k, k, w.k, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t u = __float_as_uint(v[e]) & 0x7fffffffu;
        any |= u >= 0x7f800000u;
        most = max(most, u >= 0x7f800000u ? 0u : u);
      }
    }
    most = __reduce_max_sync(0xffffffffu, most);
    any = __reduce_or_sync(0xffffffffu, any);
    if ((threadIdx.x & 31) == 0) {
      if (any) bad[r] = 1;
      if (most > largest[r]) atomicMax(&largest[r], most);
    }
  }
  __syncthreads();
}

// Integers q = round(x * 2^p) of at most 2^30 in magnitude, as signed bytes d0 +
// 256 d1 + 65536 d2 + 2^24 d3: the bytes of q + 0x80808080 less 128 each.  sums[segment's
// first block][column]: the bytes of a segment added up.  What is not finite (bad[r]) counts
// as 0.  back[r]: 2^-p as two factors.
template <int U, int GB>
__device__ __forceinline__ void stage_int(const Weights& w, const Rows& in, int row0, int rows, int b0, int nb, bool wide,
                                          uint2* xs, int* sums, int sum_cols, const uint32_t* largest, float2* back,
                                          const int* bad) {
  const int cols = rows * kLimbs, words = nb * 4;
  for (int r = 0; r < rows; ++r) {
    const int p = 29 - ((int)(largest[r] >> 23) - 127), half = p / 2;  // -98 .. 156: two factors, each exact
    if (threadIdx.x == 0) back[r] = make_float2(__int_as_float((127 - half) << 23), __int_as_float((127 - p + half) << 23));
    const float f0 = __int_as_float((127 + half) << 23), f1 = __int_as_float((127 + p - half) << 23);
    const bool check = bad[r];
    for (int first = 0; first < words; first += blockDim.x) {
      const int i = first + threadIdx.x, b = i >> 2, word = i & 3, k = b0 * 32 + i * 8;
      uint32_t u[8];
      if (i < words) {
        float v[8];
        load_x(in, wide, (int64_t)(row0 + r) * in.stride + k, k, w.k, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (check && !finite(v[e])) v[e] = 0.f;
          u[e] = 0x80808080u + (uint32_t)__float2int_rn(v[e] * f0 * f1);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = 0x80808080u;
      }
#pragma unroll
      for (int l = 0; l < kLimbs; ++l) {
        constexpr uint32_t pick[kLimbs] = {0x40, 0x51, 0x62, 0x73};
        const uint32_t d0 = __byte_perm(__byte_perm(u[0], u[2], pick[l]), __byte_perm(u[4], u[6], pick[l]), 0x5410) ^
                            0x80808080u;
        const uint32_t d1 = __byte_perm(__byte_perm(u[1], u[3], pick[l]), __byte_perm(u[5], u[7], pick[l]), 0x5410) ^
                            0x80808080u;
        int total = __dp4a((int)d0, 0x01010101, __dp4a((int)d1, 0x01010101, 0));
#pragma unroll
        for (int o = 1; o < 4 * GB; o *= 2) total += __shfl_xor_sync(0xffffffffu, total, o);  // a segment's words
        if (i < words) {
          xs[x_place<U>(b, word, cols, r * kLimbs + l)] = make_uint2(d0, d1);
          if (i % (4 * GB) == 0) sums[b * sum_cols + r * kLimbs + l] = total;
        }
      }
    }
  }
}

// y for up to NT*8 columns (a row's parts or bytes each one): warp products of 16 weight
// rows by 32 columns of the weight a step.  Each warp copies its own codes three
// chunks (6 KB) ahead and needs no other warp until its tile ends, so that an SM has
// about 100 KB in flight; the CTA's slice of x is laid out in shared memory once.
template <int NT, int GB, bool kInt, int kScale>
__global__ void __launch_bounds__(most_warps(NT) * 32, 1)
int4_linear_kernel(const Weights w, const Shape sh, const Rows in, float down, float up, const void* bias, void* y,
                   float* partial) {
  constexpr int U = GB < 4 ? GB : 4, kUnits = GB / U;  // a unit's blocks, a segment's units
  extern __shared__ __align__(128) char smem[];
  __shared__ uint32_t largest[32];
  __shared__ int bad[32];
  __shared__ float2 back[32];  // two powers of two: from a row's integers to its values
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;  // warp: the same in all lanes
  const int warps = sh.along * sh.tiles;
  const int row0 = blockIdx.y * in.pass, rows = min(in.pass, in.all - row0), cols = rows * in.parts;
  const int c0 = blockIdx.z * sh.slice_chunks;
  const int c1 = min((w.blocks + kBlocks - 1) / kBlocks, c0 + sh.slice_chunks);
  const int b0 = c0 * kBlocks, nb = min(w.blocks, c1 * kBlocks) - b0;  // the slice's blocks
  char* ring = smem + warp * kStages * kStageBytes;
  char* slots = smem + warps * kStages * kStageBytes + warp * sh.slots * sh.slot_bytes;
  float* red = reinterpret_cast<float*>(smem + warps * (kStages * kStageBytes + sh.slots * sh.slot_bytes));
  char* xs = reinterpret_cast<char*>(red + 2 * warps * kTile * NT * 8);
  int* sums = reinterpret_cast<int*>(xs + nb * cols * 32);  // integers only

  const int wt = warp / sh.along, wk = warp % sh.along;
  const int tiles = (int)((w.n + kTile - 1) / kTile), tile_step = gridDim.x * sh.tiles;
  const int from_chunk = c0 + wk * sh.warp_chunks, to_chunk = min(c1, from_chunk + sh.warp_chunks);
  const int64_t pitch = (int64_t)w.blocks * 16;
  // Two places in the warp's sequence of chunks: being copied, being computed (and
  // without kScale a third: its scales being loaded).  A warp without chunks passes
  // over each tile once.
  struct Place {
    int tile, chunk;
  };
  auto next = [&](Place& p) {
    if (++p.chunk < to_chunk) return false;
    p.chunk = from_chunk;
    p.tile += tile_step;
    return true;
  };
  const Place start = {(int)(blockIdx.x * sh.tiles + wt), from_chunk};
  Place copy = start, at = start, load = start;

  // A span's chunks lie between multiples of its length; the first of a tile may start within.
  const int lead = kScale ? from_chunk % sh.span : 0;
  const int span_chunks = GB < 8 ? GB : w.group_blocks;  // of a piece
  const uint8_t* from = nullptr;  // the tile's first row, in the chunk to copy
  uint32_t row_at[kTile / 4];     // the lane's 16 bytes of rows lane/8 + 4i
  // A lane's pieces of a span: piece_row[j] of the tile, pieces side by side in neighbouring
  // lanes.  Byte offsets from the tile's first row, for scales of one byte.
  constexpr int kPieces = GB < 4 ? 4 / GB : 1, kCopies = (kTile * kPieces + 31) / 32;
  uint32_t piece_at[kCopies];
  auto aim_scales = [&](int last) {
#pragma unroll
    for (int j = 0; j < kCopies; ++j)
      piece_at[j] = (uint32_t)min((lane + 32 * j) / kPieces, last) * (uint32_t)w.groups + (lane + 32 * j) % kPieces * 8;
  };
  auto aim = [&]() {
    const int64_t n = (int64_t)copy.tile * kTile;
    from = w.packed + n * pitch + from_chunk * (kBlocks * 16);
    const int last = (int)min((int64_t)kTile, w.n - n) - 1;  // past the last row: that one again
#pragma unroll
    for (int i = 0; i < kTile / 4; ++i)
      row_at[i] = (uint32_t)min(i * 4 + (lane >> 3), last) * (uint32_t)pitch + (lane & 7) * 16;
    if constexpr (kScale != 0) aim_scales(last);
  };
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring), slot_at = (uint32_t)__cvta_generic_to_shared(slots);
  uint32_t to[kTile / 4];
#pragma unroll
  for (int i = 0; i < kTile / 4; ++i) to[i] = ring_at + piece(i * 4 + (lane >> 3), lane & 7);
  if (copy.tile < tiles) aim();
  int copy_slot = 0, use_slot = 0, copy_at = lead, use_at = lead;  // chunks from the span's start
  auto copy_scales = [&]() {
    const uint32_t dst = slot_at + copy_slot * sh.slot_bytes, dst_zero = dst + kTile * sh.places * 8 * kScale;
    copy_slot = copy_slot + 1 == sh.slots ? 0 : copy_slot + 1;
    const int first = (copy.chunk - copy_at) / span_chunks;  // piece: eight groups, of group_blocks chunks
    const char* scales = (const char*)w.scales + ((int64_t)copy.tile * kTile * w.groups + first * 8) * kScale;
    const uint8_t* zeros = w.zeros + (int64_t)copy.tile * kTile * w.groups + first * 8;
#pragma unroll
    for (int j = 0; j < kCopies; ++j) {
      const int p = (lane + 32 * j) % kPieces, place = (lane + 32 * j) / kPieces * sh.places + p;
      if ((kTile * kPieces < 32 && lane >= kTile * kPieces) || (first + p) * 8 >= w.groups) continue;
#pragma unroll
      for (int h = 0; h < kScale / 2; ++h)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + place * 8 * kScale + h * 16),
                     "l"(scales + piece_at[j] * (uint32_t)kScale + h * 16)
                     : "memory");
      if (w.zeros)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst_zero + place * 8), "l"(zeros + piece_at[j])
                     : "memory");
    }
  };
  auto fetch = [&](int stage) {
    if (copy.tile < tiles) {
      if (copy.chunk * kBlocks + (lane & 7) < w.blocks && copy.chunk < to_chunk)
#pragma unroll
        for (int i = 0; i < kTile / 4; ++i)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to[i] + stage * kStageBytes), "l"(from + row_at[i])
                       : "memory");
      if (kScale && (copy.chunk == from_chunk || copy_at == 0) && copy.chunk < to_chunk) copy_scales();
      from += kBlocks * 16;
      copy_at = copy_at + 1 == sh.span ? 0 : copy_at + 1;
      if (next(copy)) {
        if (copy.tile < tiles) aim();
        copy_at = lead;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // x first: behind the rings' first copies its loads would wait for 100 KB an SM.
  const bool wide = in.dtype != SPR_F32 && in.stride % 8 == 0 && reinterpret_cast<uintptr_t>(in.x) % 16 == 0;
  if constexpr (kInt) scan_x(w, in, row0, rows, b0, nb, wide, largest, bad);
  else stage_bf16<U>(w, in, row0, rows, b0, nb, down, wide, reinterpret_cast<uint4*>(xs));
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  Values<GB> values;
  int64_t load_at = 0;
  if constexpr (!kScale) {
    load_at = min((int64_t)load.tile * kTile + (lane & 15), w.n - 1) * w.groups;
    if (load.tile < tiles) values.load(w, load_at, load.chunk, lane);
  }

  if constexpr (kInt)
    stage_int<U, GB>(w, in, row0, rows, b0, nb, wide, reinterpret_cast<uint2*>(xs), sums, NT * 8, largest, back, bad);
  __syncthreads();

  uint64_t acc[NT][2] = {};  // pairs of neighbouring columns, rows r8 and r8 + 8
  int stage = 0, odd = 0;
  const int t = lane & 3, r8 = lane >> 2;
  const char* lane_words = ring + r8 * 128;
  int col_at[NT];  // a lane past the last column reads that one; its sums are not used
#pragma unroll
  for (int q = 0; q < NT; ++q) col_at[q] = (min(q * 8 + r8, cols - 1) * 4 + t) * (kInt ? 8 : 16);
  const int block_bytes = cols * (kInt ? 32 : 64);
  while (at.tile < tiles) {
    if constexpr (!kScale) {
      values.store(slots + use_slot * sh.slot_bytes, lane);
      if (next(load)) load_at = min((int64_t)load.tile * kTile + (lane & 15), w.n - 1) * w.groups;
      if (load.tile < tiles) values.load(w, load_at, load.chunk, lane);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    const int first = at.chunk * kBlocks, here = at.chunk < to_chunk ? min(kBlocks, w.blocks - first) : 0;
    const char* words = lane_words + stage * kStageBytes;
    const char* xb = xs + (first - b0) * block_bytes;
    const int* sb = sums + (first - b0) * (NT * 8) + 2 * t;
    // The lane's rows' scales and zeros, from the chunk's first segment's group on.
    constexpr int kBytes = kScale ? kScale : 4;
    const char* slot = slots + use_slot * sh.slot_bytes;
    const int places = kScale ? sh.places : 1;
    const int group0 = !kScale ? 0 : GB < 8 ? use_at * (8 / GB) : use_at * kBlocks / w.group_blocks;
    const char* sp = slot + (r8 * places * 8 + group0) * kBytes;
    const uint8_t* zp = reinterpret_cast<const uint8_t*>(slot) + kTile * places * 8 * kBytes + r8 * places * 8 + group0;
    float2 m0, m1;
    float c[NT][4];
    int ci[NT][4];
#pragma unroll
    for (int u = 0; u < kBlocks / U; ++u) {
      if (u * U >= here) break;
      if (u % kUnits == 0) {
        const int g = u / kUnits;
        if constexpr (kScale == 2) {
          const uint16_t h0 = reinterpret_cast<const uint16_t*>(sp)[g];
          const uint16_t h1 = reinterpret_cast<const uint16_t*>(sp + places * 128)[g];
          const bool bf = w.scale_dtype == SPR_BF16;
          m0.x = bf ? __uint_as_float((uint32_t)h0 << 16) : __half2float(__ushort_as_half(h0));
          m1.x = bf ? __uint_as_float((uint32_t)h1 << 16) : __half2float(__ushort_as_half(h1));
        } else {
          m0.x = reinterpret_cast<const float*>(sp)[g];
          m1.x = reinterpret_cast<const float*>(sp + places * 256)[g];
        }
        int z0 = 8, z1 = 8;
        if (!kScale || w.zeros) {
          z0 = zp[g];
          z1 = zp[places * 64 + g];
        }
        if constexpr (!kInt) {
          m0.y = __int_as_float(0x43004300 + 0x00010001 * z0);
          m1.y = __int_as_float(0x43004300 + 0x00010001 * z1);
        }
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          if constexpr (kInt) {  // sums of x*(code - zero), as the low bits of 1.5*2^23
            const int2 xsum = *reinterpret_cast<const int2*>(sb + u * U * NT * 8 + q * 8);
            ci[q][0] = 0x4b400000 - z0 * xsum.x;
            ci[q][1] = 0x4b400000 - z0 * xsum.y;
            ci[q][2] = 0x4b400000 - z1 * xsum.x;
            ci[q][3] = 0x4b400000 - z1 * xsum.y;
          } else {
            c[q][0] = c[q][1] = c[q][2] = c[q][3] = 0.f;
          }
        }
      }
      // U words of the lane's share of the unit, of rows r8 and r8 + 8.
      uint32_t w0[U], w1[U];
      const char* from0 = words + (((u * U + t * U / 4) ^ turn(r8)) << 4) + (t * U % 4) * 4;
      load_words<U>(from0, w0);
      load_words<U>(from0 + 1024, w1);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const char* xj = xb + (u * U + j) * block_bytes;
        if constexpr (kInt) {
          const uint32_t a0 = w0[j] & 0x0f0f0f0fu, a1 = w1[j] & 0x0f0f0f0fu;
          const uint32_t a2 = w0[j] >> 4 & 0x0f0f0f0fu, a3 = w1[j] >> 4 & 0x0f0f0f0fu;
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            const uint2 v = *reinterpret_cast<const uint2*>(xj + col_at[q]);
            mma_int(ci[q], a0, a1, a2, a3, v.x, v.y);
          }
        } else {
          const uint32_t z0 = __float_as_uint(m0.y), z1 = __float_as_uint(m1.y);
          const uint32_t a0 = codes<0>(w0[j], z0), a1 = codes<0>(w1[j], z1);
          const uint32_t a2 = codes<1>(w0[j], z0), a3 = codes<1>(w1[j], z1);
          const uint32_t d0 = codes<2>(w0[j], z0), d1 = codes<2>(w1[j], z1);
          const uint32_t d2 = codes<3>(w0[j], z0), d3 = codes<3>(w1[j], z1);
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            const uint4 v = *reinterpret_cast<const uint4*>(xj + col_at[q]);
            mma_bf16(c[q], a0, a1, a2, a3, v.x, v.y);
            mma_bf16(c[q], d0, d1, d2, d3, v.z, v.w);
          }
        }
      }
      if (u % kUnits == kUnits - 1) {
#pragma unroll
        for (int q = 0; q < NT; ++q)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint64_t v = kInt ? pair(__int_as_float(ci[q][2 * i]), __int_as_float(ci[q][2 * i + 1]))
                              : pair(c[q][2 * i], c[q][2 * i + 1]);
            if (kInt) v = add2(v, pair(-12582912.f, -12582912.f));
            const float m = i ? m1.x : m0.x;
            acc[q][i] = fma2(v, pair(m, m), acc[q][i]);
          }
      }
    }
    // The stage that this fetch fills was read in the round before.
    fetch(stage == 0 ? kStages - 1 : stage - 1);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    const int tile = at.tile;
    const bool done = next(at);
    use_at = done ? lead : use_at + 1 == sh.span ? 0 : use_at + 1;
    if (!kScale || done || use_at == 0) use_slot = use_slot + 1 == sh.slots ? 0 : use_slot + 1;
    if (!done) continue;
    // The tile is done: join the warps' sums and a row's columns.
    float* mine = red + ((odd * sh.tiles + wt) * sh.along + wk) * kTile * NT * 8;
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      *reinterpret_cast<uint64_t*>(mine + r8 * NT * 8 + q * 8 + 2 * t) = acc[q][0];
      *reinterpret_cast<uint64_t*>(mine + (r8 + 8) * NT * 8 + q * 8 + 2 * t) = acc[q][1];
      acc[q][0] = acc[q][1] = 0;
    }
    if (sh.along > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + wt), "r"(sh.along * 32) : "memory");
    else __syncwarp();
    const float* part = red + (odd * sh.tiles + wt) * sh.along * kTile * NT * 8;
    for (int i = wk * 32 + lane; i < kTile * rows; i += sh.along * 32) {
      const int row = i % kTile, r = i / kTile;
      const int64_t n = (int64_t)tile * kTile + row;
      if (n >= w.n) continue;
      // A row's parts, or its bytes' sums: each of these is brought to its place by powers of
      // two before they meet, since 2^30 times the result may leave fp32.
      float v = 0.f, unit = 1.f;
      for (int p = 0; p < in.parts; ++p) {
        float a = 0.f;
        for (int q = 0; q < sh.along; ++q) a += part[(q * kTile + row) * NT * 8 + r * in.parts + p];
        if constexpr (kInt) {
          a = a * back[r].x * unit * back[r].y;
          unit *= 256.f;
        }
        v += a;
      }
      if constexpr (kInt) {
        if (bad[r])  // infinities and NaN of the row, one by one
          for (int k = b0 * 32; k < min(w.k, (b0 + nb) * 32); ++k) {
            const float xv = load_as_f32(in.x, in.dtype, (int64_t)(row0 + r) * in.stride + k);
            if (finite(xv)) continue;
            const int64_t g = n * w.groups + k / (w.group_blocks * 32);
            const int code = w.packed[n * pitch + k / 2] >> (k & 1) * 4 & 15;
            v += xv * ((float)(code - (w.zeros ? w.zeros[g] : 8)) * load_as_f32(w.scales, w.scale_dtype, g));
          }
      } else {
        v *= up;
      }
      if (partial) partial[((int64_t)blockIdx.z * in.all + row0 + r) * w.n + n] = v;
      else store_f32(y, in.dtype, (row0 + r) * w.n + n, bias ? v + load_as_f32(bias, in.dtype, n) : v);
    }
    odd ^= 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Joins slices (or walks) of `size` sums.  Where they are many (blockDim.y 8), 32 sums
// by 8 threads, each every eighth slice in its order.
__global__ void __launch_bounds__(256)
int4_join_kernel(const float* partial, int slices, int64_t size, int64_t n, const void* bias, void* y, int dtype) {
  __shared__ float part[8][32];
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  float v = 0.f;
  if (i < size)
#pragma unroll 4
    for (int s = threadIdx.y; s < slices; s += blockDim.y) v += partial[s * size + i];
  if (blockDim.y > 1) {
    part[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y == 0)
#pragma unroll
      for (int q = 1; q < 8; ++q) v += part[q][threadIdx.x];
  }
  if (threadIdx.y == 0 && i < size) store_f32(y, dtype, i, bias ? v + load_as_f32(bias, dtype, i % n) : v);
}

void join_slices(const float* partial, int slices, int64_t size, int64_t n, const void* bias, void* y, int dtype,
                 cudaStream_t st) {
  const dim3 block = slices > 8 ? dim3(32, 8) : dim3(256, 1);
  int4_join_kernel<<<(unsigned)((size + block.x - 1) / block.x), block, 0, st>>>(partial, slices, size, n, bias, y, dtype);
}

// The gradient.  A warp takes 128 columns of the weight (a chunk) and walks down its
// rows; the eight warps of a CTA take neighbouring chunks of the same rows, or rows
// beside each other.  Products of 16 rows of parts (dy*scale of a row of dy, cut into
// two or three bf16 parts: the first operand, formed once for 16 weight rows and a
// group) by 16 weight rows by 8 columns: the codes are the second operand, pairs of
// weight rows in a register.  A column of a product is a word of eight codes (or, for
// groups of 32, one of four words and its even or odd codes), so that a product's
// columns lie in one group.  Each walk's sums go to the workspace and are joined in a
// fixed order.
// The scales and zeros of the next band of weight rows are copied into shared memory
// meanwhile (in whole pieces of eight groups, where they lie so); each thread widens
// what it has copied itself.
constexpr int kGradWarps = 8;
constexpr int kGradRows = 32;    // weight rows of a stage
constexpr int kGradBlocks = 4;   // blocks of 32 codes a row of a stage: 64 bytes
constexpr int kGradStage = kGradRows * kGradBlocks * 16;
constexpr int kGradThreads = kGradWarps * 32;
static_assert(kStages == 4, "the waits for a band's pieces count the ring's stages");

// Two rows to 128 bytes; pieces turned so that rows 0, 2, 4, 6 (or 1, 3, 5, 7) and two
// neighbouring pieces meet all banks.
__device__ __forceinline__ int grad_piece(int row, int j) {
  return (row >> 1) * 128 + ((((row & 1) << 2 | j) ^ ((row >> 1 & 3) << 1)) << 4);
}

struct GradShape {
  int chunks, along;        // chunks of a row; warps of a CTA on neighbouring chunks
  int beside;               // and on walks beside each other: 1, 2 or 4
  int band;                 // weight rows, of all the CTA's walks, in shared memory at a time
  int walk;                 // weight rows of one walk, a multiple of its share of a band
  int groups;               // of a CTA's chunks, at most
  int scale, pieces;        // bytes of a scale that is copied ahead (0: none is); a row's pieces of eight
  int pass, rows;           // rows of dy in a pass, and of all passes
};

// HALVES: eights of a product's 16 rows that are used (1 with MT 1 and few rows).
template <int MT, int HALVES, int G, int PARTS>
__global__ void __launch_bounds__(kGradThreads, MT == 1 ? 2 : 1)
int4_linear_grad_kernel(const Weights w, const GradShape sh, const void* dy, int64_t dy_stride, int dtype,
                        float* partial) {
  extern __shared__ __align__(128) char smem[];
  constexpr int kTileRows = HALVES * 8 / PARTS, kRowsMax = MT * kTileRows;  // rows of dy in a product, in all
  constexpr int kEights = MT * HALVES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, beside = sh.beside;
  const int row0 = blockIdx.z * sh.pass, rows = min(sh.pass, sh.rows - row0);
  const int chunk0 = blockIdx.x * sh.along;
  const int all = sh.band, band = all / beside, bands = sh.walk / band;  // band: a walk's rows of it
  float2* meta = reinterpret_cast<float2*>(smem + kGradWarps * kStages * kGradStage);  // [band row][group]
  float* dys = reinterpret_cast<float*>(meta + all * sh.groups);                        // [row of dy][band row]
  char* raw = reinterpret_cast<char*>(dys + all * kRowsMax);  // [band row][piece] of scales, then of zeros
  const int group0 = chunk0 * kGradBlocks / w.group_blocks, piece0 = group0 / 8;
  const uint32_t raw_at = (uint32_t)__cvta_generic_to_shared(raw), raw_zero = all * sh.pieces * 8 * sh.scale;
  // The weight row of a band row, -1 past the end of its walk.
  auto weight_row = [&](int b, int br) {
    const int64_t walk0 = ((int64_t)blockIdx.y * beside + br / band) * sh.walk, n = walk0 + b * band + br % band;
    return n < min(w.n, walk0 + sh.walk) ? n : (int64_t)-1;
  };
  auto copy_raw = [&](int b) {
    if (sh.scale)
      for (int i = threadIdx.x; i < all * sh.pieces; i += kGradThreads) {
        const int br = i / sh.pieces, p = min(piece0 + i % sh.pieces, w.groups / 8 - 1);
        const int64_t n = weight_row(b, br), g = (n < 0 ? w.n - 1 : n) * w.groups + p * 8;
        for (int h = 0; h < sh.scale / 2; ++h)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(raw_at + i * 8 * sh.scale + h * 16),
                       "l"((const char*)w.scales + g * sh.scale + h * 16)
                       : "memory");
        if (w.zeros)
          asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(raw_at + raw_zero + i * 8), "l"(w.zeros + g)
                       : "memory");
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  constexpr int kDyRegs = (kRowsMax + 1) / 2;  // of 128 band rows
  float dy_next[kDyRegs];
  auto load_dy = [&](int b) {
#pragma unroll
    for (int j = 0; j < kDyRegs; ++j) {
      const int i = threadIdx.x + j * kGradThreads, br = i % all, r = i / all;
      const int64_t n = r < rows ? weight_row(b, br) : -1;
      dy_next[j] = n < 0 ? 0.f : load_as_f32(dy, dtype, (int64_t)(row0 + r) * dy_stride + n);
    }
  };
  // The band's values in the form that the products take; whether any is so large (or
  // not finite) that a product may leave fp32.
  auto widen = [&](int b) {
    bool large = false;
    auto put = [&](int br, int g, float v, uint32_t z) {
      if (g < 0 || g >= sh.groups) return;
      meta[br * sh.groups + g] = make_float2(v, __uint_as_float(0x4300u + z));
      large |= !(fabsf(v) < 0x1p60f);
    };
    if (sh.scale) {
      for (int i = threadIdx.x; i < all * sh.pieces; i += kGradThreads) {
        const int br = i / sh.pieces, g = (piece0 + i % sh.pieces) * 8 - group0;
        const bool in = weight_row(b, br) >= 0;
        const uint2 z8 = w.zeros ? *reinterpret_cast<const uint2*>(raw + raw_zero + i * 8)
                                 : make_uint2(0x08080808u, 0x08080808u);
        const char* from = raw + i * 8 * sh.scale;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float v;
          if (sh.scale == 4) {
            v = reinterpret_cast<const float*>(from)[e];
          } else {
            const uint16_t h = reinterpret_cast<const uint16_t*>(from)[e];
            v = w.scale_dtype == SPR_BF16 ? __uint_as_float((uint32_t)h << 16) : __half2float(__ushort_as_half(h));
          }
          put(br, g + e, in ? v : 0.f, (e < 4 ? z8.x >> 8 * e : z8.y >> 8 * (e - 4)) & 0xffu);
        }
      }
    } else {
#pragma unroll 4
      for (int i = threadIdx.x; i < all * sh.groups; i += kGradThreads) {
        const int br = i / sh.groups, g = i % sh.groups;
        const int64_t n = weight_row(b, br), at = n * w.groups + group0 + g;
        const bool in = n >= 0 && group0 + g < w.groups;
        put(br, g, in ? load_as_f32(w.scales, w.scale_dtype, at) : 0.f, in && w.zeros ? __ldg(w.zeros + at) : 8u);
      }
    }
#pragma unroll
    for (int j = 0; j < kDyRegs; ++j) {
      const int i = threadIdx.x + j * kGradThreads;
      if (i < all * kRowsMax) dys[i] = dy_next[j];
      large |= !(fabsf(dy_next[j]) < 0x1p60f);
    }
    return large;
  };

  const int chunk = chunk0 + warp % sh.along, walk_id = blockIdx.y * beside + warp / sh.along;
  const int64_t n0 = (int64_t)walk_id * sh.walk, n1 = min(w.n, n0 + sh.walk);
  const bool mine = chunk < sh.chunks && warp < sh.along * beside && n0 < n1;
  const int steps = mine ? (int)(n1 - n0 + kGradRows - 1) / kGradRows : 0;
  char* ring = smem + warp * kStages * kGradStage;
  const int64_t pitch = (int64_t)w.blocks * 16;

  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  uint32_t to[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) to[i] = ring_at + grad_piece(8 * i + (lane >> 2), lane & 3);
  const bool has_piece = mine && chunk * kGradBlocks + (lane & 3) < w.blocks;
  const uint8_t* from = w.packed + (n0 + (lane >> 2)) * pitch + (int64_t)chunk * (kGradBlocks * 16) + (lane & 3) * 16;
  int fetched = 0;
  auto fetch = [&](int stage) {
    if (fetched < steps && has_piece)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (n0 + fetched * kGradRows + 8 * i + (lane >> 2) < w.n)  // past the end: whatever the stage holds, times 0
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to[i] + stage * kGradStage),
                       "l"(from + i * 8 * pitch)
                       : "memory");
      }
    from += kGradRows * pitch;
    ++fetched;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  copy_raw(0);
  load_dy(0);
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);

  const int t = lane & 3, c8 = lane >> 2;
  constexpr int kTiles = kGradBlocks * 4;  // products' columns: 8 of the chunk's 128 each
  float acc[MT][kTiles][4] = {};
  // The lane's rows of parts, one of each eight: its row of dy and which bits of a value
  // the parts before its own hold.
  int dy_row[kEights];
  uint32_t cut0[kEights], cut1[kEights];
#pragma unroll
  for (int m = 0; m < kEights; ++m) {
    const int rr = m % HALVES * 8 + c8, r = m / HALVES * kTileRows + rr / PARTS;
    const bool in = rr < kTileRows * PARTS && r < rows;
    dy_row[m] = in ? r * all : -1;
    cut0[m] = rr % PARTS > 0 ? 0xffff0000u : 0u;
    cut1[m] = rr % PARTS > 1 ? 0xffff0000u : 0u;
  }
  // Words of rows 2t (+1) and pieces: grad_piece of row 16h + 2t + 8q + o, piece 2b + ... is
  // (8h + 4q + t)*128 + place[o][b].
  int place[2][2];
#pragma unroll
  for (int o = 0; o < 2; ++o)
#pragma unroll
    for (int b = 0; b < 2; ++b)
      place[o][b] = t * 128 + (((o * 4 + 2 * b) ^ (2 * t)) + (G == 1 ? 0 : c8 >> 2)) * 16 + (c8 & 3) * 4;
  const int first_block = chunk * kGradBlocks;
  int stage = 0, step = 0;
  for (int b = 0; b < bands; ++b) {
    // The band's pieces were copied before the ring's last `band / kGradRows` stages (at
    // first its first three).
    if (b == 0 || band >= 3 * kGradRows) asm volatile("cp.async.wait_group 3;" ::: "memory");
    else if (band == 2 * kGradRows) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();  // the last readers of the band before are done
    const bool large = widen(b);
    if (b + 1 < bands) {
      copy_raw(b + 1);
      load_dy(b + 1);
    }
    const bool any_wild = __syncthreads_or(large);
    const float* dband = dys;
    for (int at = 0; at < band; at += kGradRows, ++step) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      __syncwarp();
      if (step >= steps) {  // past the walk's end: the groups of copies go on being counted
        asm volatile("cp.async.commit_group;" ::: "memory");
        continue;
      }
      const char* codes_at = ring + stage * kGradStage;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int base = warp / sh.along * band + at + half * 16 + 2 * t;  // band row of the lane's first weight row
        float2 d[kEights][2];
#pragma unroll
        for (int m = 0; m < kEights; ++m)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            d[m][q] = dy_row[m] < 0 ? make_float2(0.f, 0.f)
                                    : *reinterpret_cast<const float2*>(dband + dy_row[m] + base + 8 * q);
        const float2* mp = meta + base * sh.groups;
#pragma unroll
        for (int gi = 0; gi < kGradBlocks / G; ++gi) {
          const int block = first_block + gi * G;
          if (block >= w.blocks) break;
          const int g = (G < 4 ? block / G : block / w.group_blocks) - group0;
          const int gg = G < 4 && w.group_blocks != G ? block / w.group_blocks - group0 : g;
          const float2 s[4] = {mp[gg], mp[gg + sh.groups], mp[gg + 8 * sh.groups], mp[gg + 9 * sh.groups]};
          const uint32_t z01 = __byte_perm(__float_as_uint(s[0].y), __float_as_uint(s[1].y), 0x5410);
          const uint32_t z23 = __byte_perm(__float_as_uint(s[2].y), __float_as_uint(s[3].y), 0x5410);
          uint32_t a[MT * 2][2];
#pragma unroll
          for (int m = 0; m < MT * 2; ++m)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              if (m % 2 >= HALVES) {
                a[m][q] = 0;
                continue;
              }
              const int e = m / 2 * HALVES + m % 2;
              float v[2] = {d[e][q].x * s[2 * q].x, d[e][q].y * s[2 * q + 1].x};
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float all = v[i];
                v[i] -= __uint_as_float(__float_as_uint(v[i]) & cut0[e]);
                if (PARTS == 3) v[i] -= __uint_as_float(__float_as_uint(v[i]) & cut1[e]);
                if (any_wild && !finite(all)) v[i] = cut0[e] ? 0.f : all;  // in the first part alone
              }
              a[m][q] = bf16_pair(__float_as_uint(v[0]), __float_as_uint(v[1]));
            }
          if constexpr (G == 1) {
            const int odd = (c8 >> 2) * 4;
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[i] = *reinterpret_cast<const uint32_t*>(codes_at + (8 * half + 4 * (i >> 1)) * 128 +
                                                        (place[i & 1][gi >> 1] ^ (gi & 1) * 16)) >>
                     odd;
            const uint32_t l0 = __byte_perm(v[0], v[1], 0x5410), h0 = __byte_perm(v[0], v[1], 0x7632);
            const uint32_t l1 = __byte_perm(v[2], v[3], 0x5410), h1 = __byte_perm(v[2], v[3], 0x7632);
            const uint32_t b0[4] = {codes<0>(l0, z01), codes<2>(l0, z01), codes<0>(h0, z01), codes<2>(h0, z01)};
            const uint32_t b1[4] = {codes<0>(l1, z23), codes<2>(l1, z23), codes<0>(h1, z23), codes<2>(h1, z23)};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
              for (int m = 0; m < MT; ++m)
                mma_bf16(acc[m][gi * 4 + j], a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], b0[j], b1[j]);
          } else {
#pragma unroll
            for (int u = 0; u < G / 2; ++u) {
              const int b64 = gi * G / 2 + u;  // 64 columns
              uint32_t v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                v[i] = *reinterpret_cast<const uint32_t*>(codes_at + (8 * half + 4 * (i >> 1)) * 128 +
                                                          place[i & 1][b64]);
              const uint32_t l0 = __byte_perm(v[0], v[1], 0x5410), h0 = __byte_perm(v[0], v[1], 0x7632);
              const uint32_t l1 = __byte_perm(v[2], v[3], 0x5410), h1 = __byte_perm(v[2], v[3], 0x7632);
              const uint32_t b0[8] = {codes<0>(l0, z01), codes<1>(l0, z01), codes<2>(l0, z01), codes<3>(l0, z01),
                                      codes<0>(h0, z01), codes<1>(h0, z01), codes<2>(h0, z01), codes<3>(h0, z01)};
              const uint32_t b1[8] = {codes<0>(l1, z23), codes<1>(l1, z23), codes<2>(l1, z23), codes<3>(l1, z23),
                                      codes<0>(h1, z23), codes<1>(h1, z23), codes<2>(h1, z23), codes<3>(h1, z23)};
#pragma unroll
              for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int m = 0; m < MT; ++m)
                  mma_bf16(acc[m][b64 * 8 + j], a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], b0[j],
                           b1[j]);
            }
          }
        }
      }
      // The stage that this fetch fills was read in the round before.
      fetch(stage == 0 ? kStages - 1 : stage - 1);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
  if (!mine) return;
  // The warp's ring takes a product's sums in the order of the columns; a row's parts
  // are added in their order.
  float* out = reinterpret_cast<float*>(ring);  // [16][128]
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int j = 0; j < kTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = 2 * t + (i & 1);
        const int k = G == 1 ? j / 4 * 32 + (col & 3) * 8 + j % 4 * 2 + (col >> 2) : j / 8 * 64 + col * 8 + j % 8;
        out[(c8 + (i >> 1) * 8) * 128 + k] = acc[m][j][i];
      }
    __syncwarp();
    for (int r = m * kTileRows; r < min(rows, (m + 1) * kTileRows); ++r)
      for (int i = lane; i < 128; i += 32) {
        const int k = chunk * 128 + i;
        float v = 0.f;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) v += out[((r - m * kTileRows) * PARTS + p) * 128 + i];
        if (k < w.k) partial[((int64_t)walk_id * sh.rows + row0 + r) * w.k + k] = v;
      }
    __syncwarp();
  }
}

// Sizes that the kernels' indices hold, as check_int4 names them.  A launch takes kLaunchRows
// rows (a grid's passes), more of them are cut into launches that share the workspace.
constexpr int64_t kMostOut = 0x7fffffffLL, kMostRows = 0x7fffffffLL, kMostIn = 1 << 27, kLaunchRows = 65535;
constexpr int kMostGroup = 1 << 20;
bool sizes_fit(int64_t rows, int64_t n, int64_t k, int group) {
  return rows > 0 && rows <= kMostRows && n > 0 && n <= kMostOut && k > 0 && k <= kMostIn && group >= 32 &&
         group % 32 == 0 && group <= kMostGroup;
}

int check_int4(const char* what, int64_t stride, int dtype, int64_t rows, int64_t n, int64_t k, int64_t row_len,
               int group, const void* packed, int scale_dtype) {
  if (rows < 0 || n < 0 || k < 1)
    return fail(SPR_ERR_SHAPE, "%s: rows=%lld n=%lld k=%lld", what, (long long)rows, (long long)n, (long long)k);
  if (rows > kMostRows || n > kMostOut || k > kMostIn)
    return fail(SPR_ERR_SHAPE, "%s: rows=%lld n=%lld k=%lld too large", what, (long long)rows, (long long)n,
                (long long)k);
  if (group < 32 || group % 32 || group > kMostGroup)
    return fail(SPR_ERR_SHAPE, "%s: group=%d must be a multiple of 32", what, group);
  if (rows > 1 && stride < row_len) return fail(SPR_ERR_SHAPE, "%s: row stride %lld", what, (long long)stride);
  for (int d : {dtype, scale_dtype})
    if (d != SPR_F32 && d != SPR_BF16 && d != SPR_F16) return fail(SPR_ERR_DTYPE, "%s: unsupported dtype %d", what, d);
  if (!aligned(packed, 16)) return fail(SPR_ERR_ALIGN, "%s: packed codes must be 16-byte aligned", what);
  return SPR_OK;
}

int sm_count() {
  static thread_local int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return sms[dev];
}

// Whether the rows, results, scales and the workspace begin on their elements.
int check_pointers(const char* what, int dtype, std::initializer_list<const void*> of_dtype, const void* scales,
                   int scale_dtype, const void* workspace) {
  bool ok = aligned(scales, dtype_bytes(scale_dtype)) && aligned(workspace, 4);
  for (const void* p : of_dtype) ok &= aligned(p, dtype_bytes(dtype));
  return ok ? SPR_OK : fail(SPR_ERR_ALIGN, "%s: an operand is not aligned to its elements", what);
}

// Bytes of a scale that can be copied ahead: pieces of eight, whole and aligned, and
// groups that a chunk does not straddle; else 0.
int scale_ahead(const Weights& w) {
  const bool whole = w.groups % 8 == 0 && (kBlocks % w.group_blocks == 0 || w.group_blocks % kBlocks == 0);
  return whole && aligned(w.scales, 16) && aligned(w.zeros, 8) ? dtype_bytes(w.scale_dtype) : 0;
}

template <int NT, int GB, bool kInt, int kScale>
int launch_forward(const ForwardPlan& p, const Weights& w, const void* x, int64_t x_stride, int dtype, int rows,
                   const void* bias, void* y, float* partial, cudaStream_t st) {
  auto kern = int4_linear_kernel<NT, GB, kInt, kScale>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
    return check_launch("int4 linear");
  // A bf16 product's inner sum of up to 15*32*GB values of x stays below the largest
  // fp32 number: x is taken times a power of two and the scale divided by it.
  int e = 4;
  while ((1 << (e - 4)) < GB * 32) ++e;
  const Rows in{x, x_stride, dtype, p.parts, rows, p.pass_rows};
  kern<<<dim3(p.grid, p.passes, p.sh.slices), p.sh.along * p.sh.tiles * 32, p.smem, st>>>(
      w, p.sh, in, kInt ? 1.f : ldexpf(1.f, -e), kInt ? 1.f : ldexpf(1.f, e), partial ? nullptr : bias, y, partial);
  if (partial) {
    const int64_t size = (int64_t)rows * w.n;
    join_slices(partial, p.sh.slices, size, w.n, bias, y, dtype, st);
  }
  return check_launch("int4 linear");
}

// Calls f(Int<NT>{}, Int<GB>{}, Int<integers>{}, Int<scale>{}) for a plan.
template <int N>
struct Int {
  static constexpr int value = N;
};
template <typename F>
int by_plan(const ForwardPlan& p, F f) {
  auto by_group = [&](auto nt) {
    auto by_kind = [&](auto gb) {
      auto by_scale = [&](auto ints) {
        return p.scale == 2 ? f(nt, gb, ints, Int<2>{}) : p.scale == 4 ? f(nt, gb, ints, Int<4>{}) : f(nt, gb, ints, Int<0>{});
      };
      return p.ints ? by_scale(Int<1>{}) : by_scale(Int<0>{});
    };
    return p.gb == 8 ? by_kind(Int<8>{}) : p.gb == 4 ? by_kind(Int<4>{}) : p.gb == 2 ? by_kind(Int<2>{}) : by_kind(Int<1>{});
  };
  return p.nt == 1 ? by_group(Int<1>{}) : p.nt == 2 ? by_group(Int<2>{}) : by_group(Int<4>{});
}

struct GradPlan {
  GradShape sh;
  int mt, halves, g, parts, walks, passes, smem;
  dim3 grid;
};

// Two parts hold the product of two bf16 numbers exactly, three what fp32 holds.  Walks:
// as many as fill the GPU, of at least 128 weight rows.
GradPlan plan_grad(int64_t rows, const Weights& w, int dtype) {
  GradPlan p{};
  p.parts = dtype == SPR_BF16 && w.scale_dtype == SPR_BF16 ? 2 : 3;
  p.halves = rows * p.parts <= 8 ? 1 : 2;
  const int tile_rows = p.halves * 8 / p.parts;
  p.mt = rows > tile_rows ? 2 : 1;
  p.g = w.group_blocks % 4 == 0 ? 4 : w.group_blocks % 2 == 0 ? 2 : 1;
  p.sh.rows = (int)rows;
  p.sh.pass = (int)std::min<int64_t>(rows, p.mt * tile_rows);
  p.passes = (int)((rows + p.sh.pass - 1) / p.sh.pass);
  p.sh.chunks = (w.blocks + kGradBlocks - 1) / kGradBlocks;
  p.sh.along = p.sh.chunks >= 8 ? 8 : p.sh.chunks >= 4 ? 4 : 2;
  p.sh.beside = kGradWarps / p.sh.along;
  p.sh.groups = (p.sh.along * kGradBlocks - 1) / w.group_blocks + 2;
  p.sh.band = p.sh.groups > 20 && p.sh.beside <= 2 ? 64 : 128;
  p.sh.scale = w.groups % 8 == 0 && aligned(w.scales, 16) && aligned(w.zeros, 8) ? dtype_bytes(w.scale_dtype) : 0;
  p.sh.pieces = (p.sh.groups + 6) / 8 + 1;
  const int beside = p.sh.beside, across = (p.sh.chunks + p.sh.along - 1) / p.sh.along;
  const int band = p.sh.band / beside;
  const int64_t ctas = (int64_t)sm_count() * (p.mt == 1 ? 2 : 1);
  int64_t walks = std::max<int64_t>(1, ctas / (across * p.passes)) * beside;
  walks = std::max<int64_t>(1, std::min(walks, w.n / 128));
  p.sh.walk = (int)(((w.n + walks - 1) / walks + band - 1) / band * band);
  p.walks = (int)((w.n + p.sh.walk - 1) / p.sh.walk);
  p.smem = kGradWarps * kStages * kGradStage +
           p.sh.band * (p.sh.groups * 8 + p.mt * tile_rows * 4 + (p.sh.scale ? p.sh.pieces * (8 * p.sh.scale + 8) : 0));
  p.grid = dim3(across, (p.walks + beside - 1) / beside, p.passes);
  return p;
}

template <int MT, int HALVES, int G, int PARTS>
int launch_grad(const GradPlan& p, const Weights& w, const void* dy, int64_t dy_stride, int dtype, float* partial,
                cudaStream_t st) {
  auto kern = int4_linear_grad_kernel<MT, HALVES, G, PARTS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
    return check_launch("int4 linear grad");
  kern<<<p.grid, kGradThreads, p.smem, st>>>(w, p.sh, dy, dy_stride, dtype, partial);
  return check_launch("int4 linear grad");
}

int linear_rows(const Weights& w, const void* x, int64_t x_stride, int dtype, int64_t rows, const void* bias, void* y,
                void* workspace, size_t workspace_bytes, cudaStream_t st) {
  const ForwardPlan p = plan_forward(rows, w, dtype, scale_ahead(w), sm_count());
  const size_t need = p.sh.slices > 1 ? (size_t)p.sh.slices * rows * w.n * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return fail(SPR_ERR_WORKSPACE, "int4 linear: workspace %zu < %zu bytes", workspace_bytes, need);
  float* partial = need ? (float*)workspace : nullptr;
  return by_plan(p, [&](auto nt, auto gb, auto ints, auto scale) {
    return launch_forward<decltype(nt)::value, decltype(gb)::value, decltype(ints)::value != 0, decltype(scale)::value>(
        p, w, x, x_stride, dtype, (int)rows, bias, y, partial, st);
  });
}

int grad_rows(const Weights& w, int group, const void* dy, int64_t dy_stride, int dtype, int64_t rows, void* dx,
              void* workspace, size_t workspace_bytes, cudaStream_t st) {
  int walks = 0;
  if (w.n) {
    const GradPlan p = plan_grad(rows, w, dtype);
    const size_t need = spr_int4_linear_grad_workspace_bytes(rows, w.n, w.k, group, dtype);
    if (!workspace || workspace_bytes < need)
      return fail(SPR_ERR_WORKSPACE, "int4 linear grad: workspace %zu < %zu bytes", workspace_bytes, need);
    auto by_group = [&](auto mt, auto halves, auto parts) {
      constexpr int MT = decltype(mt)::value, H = decltype(halves)::value, PARTS = decltype(parts)::value;
      float* out = (float*)workspace;
      return p.g == 4   ? launch_grad<MT, H, 4, PARTS>(p, w, dy, dy_stride, dtype, out, st)
             : p.g == 2 ? launch_grad<MT, H, 2, PARTS>(p, w, dy, dy_stride, dtype, out, st)
                        : launch_grad<MT, H, 1, PARTS>(p, w, dy, dy_stride, dtype, out, st);
    };
    auto by_rows = [&](auto parts) {
      return p.halves == 1 ? by_group(Int<1>{}, Int<1>{}, parts)
             : p.mt == 1   ? by_group(Int<1>{}, Int<2>{}, parts)
                           : by_group(Int<2>{}, Int<2>{}, parts);
    };
    if (int rc = p.parts == 2 ? by_rows(Int<2>{}) : by_rows(Int<3>{})) return rc;
    walks = p.walks;
  }
  join_slices((const float*)workspace, walks, rows * w.k, w.k, nullptr, dx, dtype, st);
  return check_launch("int4 linear grad");
}

}  // namespace

}  // namespace spr

using namespace spr;

extern "C" size_t spr_int4_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int group, int dtype) {
  if (!sizes_fit(rows, n, k, group)) return 0;
  rows = std::min(rows, kLaunchRows);
  const Weights w = make_weights(nullptr, nullptr, 0, nullptr, n, k, group);
  size_t most = 0;
  for (int scale : {0, 2, 4}) {  // whatever the scales' type and alignment will be
    const ForwardPlan p = plan_forward(rows, w, dtype, scale, sm_count());
    if (p.sh.slices > 1) most = std::max(most, (size_t)p.sh.slices * rows * n * sizeof(float));
  }
  return most;
}

extern "C" int spr_int4_linear(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t n, int64_t k,
                               int group, const uint8_t* packed, const void* scales, int scale_dtype,
                               const uint8_t* zeros, const void* bias, void* y, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (int rc = check_int4("int4 linear", x_stride, dtype, rows, n, k, k, group, packed, scale_dtype)) return rc;
  if (rows == 0 || n == 0) return SPR_OK;
  if (!x || !packed || !scales || !y) return fail(SPR_ERR_ARG, "int4 linear: null operand");
  if (int rc = check_pointers("int4 linear", dtype, {x, bias, y}, scales, scale_dtype, workspace)) return rc;
  const Weights w = make_weights(packed, scales, scale_dtype, zeros, n, k, group);
  const int e = dtype_bytes(dtype);
  for (int64_t r = 0; r < rows; r += kLaunchRows)
    if (int rc = linear_rows(w, (const char*)x + r * x_stride * e, x_stride, dtype, std::min(rows - r, kLaunchRows), bias,
                             (char*)y + r * n * e, workspace, workspace_bytes, (cudaStream_t)stream))
      return rc;
  return SPR_OK;
}

extern "C" size_t spr_int4_linear_grad_workspace_bytes(int64_t rows, int64_t n, int64_t k, int group, int dtype) {
  if (!sizes_fit(rows, n, k, group)) return 0;
  rows = std::min(rows, kLaunchRows);
  size_t most = 0;
  for (int scale_dtype : {SPR_F32, SPR_BF16}) {
    const GradPlan p = plan_grad(rows, make_weights(nullptr, nullptr, scale_dtype, nullptr, n, k, group), dtype);
    most = std::max(most, (size_t)p.walks * rows * k * sizeof(float));
  }
  return most;
}

extern "C" int spr_int4_linear_grad(const void* dy, int64_t dy_stride, int dtype, int64_t rows, int64_t n, int64_t k,
                                    int group, const uint8_t* packed, const void* scales, int scale_dtype,
                                    const uint8_t* zeros, void* dx, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  if (int rc = check_int4("int4 linear grad", dy_stride, dtype, rows, n, k, n, group, packed, scale_dtype)) return rc;
  if (rows == 0) return SPR_OK;
  if (!dx || (n && (!dy || !packed || !scales))) return fail(SPR_ERR_ARG, "int4 linear grad: null operand");
  if (int rc = check_pointers("int4 linear grad", dtype, {dy, dx}, scales, scale_dtype, workspace)) return rc;
  const Weights w = make_weights(packed, scales, scale_dtype, zeros, n, k, group);
  const int e = dtype_bytes(dtype);
  for (int64_t r = 0; r < rows; r += kLaunchRows)
    if (int rc = grad_rows(w, group, (const char*)dy + r * dy_stride * e, dy_stride, dtype, std::min(rows - r, kLaunchRows),
                           (char*)dx + r * k * e, workspace, workspace_bytes, (cudaStream_t)stream))
      return rc;
  return SPR_OK;
}
