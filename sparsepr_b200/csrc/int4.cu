// Product of a few rows with 4-bit weights under group scales, and its gradient
// with respect to the rows (layout and formula at spr_int4_linear in the header).
//   y[r][n] = sum_g scale[n][g] * sum_{k in g} x[r][k]*(code[n][k] - zero[n][g]) + bias[n]
//   dx[r][k] = sum_n (dy[r][n]*scale[n][g]) * (code[n][k] - zero[n][g])
// What bounds both is the codes' bytes (an SM takes 23 bytes, 46 codes, a cycle from
// HBM), so the arithmetic on a code has to stay within two or three instructions.
// Tensor-core products (m16n8k16, bf16 with fp32 sums) take a code as the exact bf16
// integer code - zero: three instructions make two of them.  The other operand is
// split into as many bf16 parts as its significand needs (bf16 1, fp16 2, fp32 3, by
// cutting off, which is exact), each part a row or column of its own in the same
// product, so that nothing is rounded before the fp32 sums.  With at most 32 rows
// the 5th-generation tensor instructions would idle on 128-row tiles, and their
// operands would have to pass through shared memory once more after unpacking.
#include <math.h>

#include "common.cuh"

namespace spr {

namespace {

constexpr int kWarps = 8;        // of a CTA, at most
constexpr int kTile = 16;        // weight rows of a product
constexpr int kChunk = 256;      // codes of a row in one stage of a warp's ring: 128 bytes
constexpr int kBlocks = kChunk / 32;
constexpr int kStages = 4;
constexpr int kStageBytes = kTile * kChunk / 2;

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

__device__ __forceinline__ void copy16_async(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
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

// The operands as the kernels take them.
struct Weights {
  const uint8_t* packed;
  const void* scales;
  const uint8_t* zeros;
  int scale_dtype;
  int64_t n;
  int k, groups, group_blocks, blocks;  // blocks of 32 codes a row, the unused ones of the last group too
};

// A warp's ring holds the codes of 16 weight rows by 256 columns a stage.  16-byte
// piece j of row r lies at j ^ (r & 7): what eight lanes groups read at once falls
// into different banks.
__device__ __forceinline__ int piece(int row, int j) { return row * 128 + ((j ^ (row & 7)) << 4); }

__device__ __forceinline__ void fetch_codes(const Weights& w, int64_t tile, int chunk, char* stage, int lane) {
  const int j = lane & 7;
  if (chunk * kBlocks + j < w.blocks) {
#pragma unroll
    for (int i = 0; i < kTile / 4; ++i) {
      const int row = i * 4 + (lane >> 3);
      const int64_t n = min(tile * kTile + row, w.n - 1);
      copy16_async(stage + piece(row, j), w.packed + (n * w.blocks + chunk * kBlocks + j) * 16);
    }
  }
}

// Scale and 128 + zero (bf16, in both halves) of a stage's rows and groups: loaded one
// stage ahead into registers, then put where the warp's lanes find them.
template <int kRegs>
struct Meta {
  float scale[kRegs];
  uint32_t zero[kRegs];
  __device__ __forceinline__ void load(const Weights& w, int64_t tile, int chunk, int lane, float up) {
    const int64_t n = min(tile * kTile + (lane & 15), w.n - 1);
    const int g0 = chunk * kBlocks / w.group_blocks;
#pragma unroll
    for (int i = 0; i < kRegs; ++i) {
      const int g = min(g0 + 2 * i + (lane >> 4), w.groups - 1);
      scale[i] = load_as_f32(w.scales, w.scale_dtype, n * w.groups + g) * up;
      zero[i] = 0x43004300u + 0x00010001u * (w.zeros ? (uint32_t)__ldg(w.zeros + n * w.groups + g) : 8u);
    }
  }
  __device__ __forceinline__ void store(float2* meta, int lane) const {
#pragma unroll
    for (int i = 0; i < kRegs; ++i) meta[i * 32 + lane] = make_float2(scale[i], __uint_as_float(zero[i]));
  }
};
constexpr int kMetaRegs(int gb) { return gb == 1 ? 4 : gb == 4 ? 1 : 2; }  // groups a stage touches, in pairs

// Where a launch's warps work: `along` warps of a CTA share a tile, each with every
// `along`-th chunk of the CTA's slice of the columns; `tiles` such teams to a CTA.
struct Shape {
  int along, tiles;
  int slice_chunks, slices;
};

// y for up to NT*8 columns (a row's parts each one): warp products of 16 weight rows
// by 32 columns of the weight a step, the x parts staged in shared memory in the order
// in which a word's codes come apart (k, k+4), (k+1, k+5), ...
template <int NT, int GB>
__global__ void __launch_bounds__(kWarps * 32, 2)
int4_linear_kernel(const Weights w, const Shape sh, const void* x, int64_t x_stride, int dtype, int parts, int all_rows,
                   int pass_rows, float down, float up, const void* bias, void* y, float* partial) {
  constexpr int kRegs = kMetaRegs(GB);
  extern __shared__ __align__(128) char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = sh.along * sh.tiles;
  const int row0 = blockIdx.y * pass_rows, rows = min(pass_rows, all_rows - row0), cols = rows * parts;
  const int c0 = blockIdx.z * sh.slice_chunks;
  const int c1 = min((w.blocks + kBlocks - 1) / kBlocks, c0 + sh.slice_chunks);
  const int b0 = c0 * kBlocks, nb = min(w.blocks, c1 * kBlocks) - b0;  // the slice's blocks
  char* ring = smem + warp * kStages * kStageBytes;
  float2* meta = reinterpret_cast<float2*>(smem + warps * kStages * kStageBytes) + warp * 2 * 32 * kRegs;
  float* red = reinterpret_cast<float*>(smem + warps * (kStages * kStageBytes + 2 * 32 * kRegs * 8));
  uint4* xs = reinterpret_cast<uint4*>(red + 2 * warps * kTile * NT * 8);  // [block][column][word of the block]

  const int wt = warp / sh.along, wk = warp % sh.along;
  const int64_t tiles = (w.n + kTile - 1) / kTile, tile_step = (int64_t)gridDim.x * sh.tiles;
  // Three places in the warp's sequence of stages: being copied, its scales being
  // loaded, being computed.
  struct Place {
    int64_t tile;
    int chunk;
  };
  auto next = [&](Place& p) {
    p.chunk += sh.along;
    if (p.chunk >= c1) {
      p.chunk = c0 + wk;
      p.tile += tile_step;
    }
  };
  const Place start = {(int64_t)blockIdx.x * sh.tiles + wt, c0 + wk};
  Place copy = start, load = start, at = start;
  auto fetch = [&](int stage) {
    if (copy.tile < tiles) {
      fetch_codes(w, copy.tile, copy.chunk, ring + stage * kStageBytes, lane);
      next(copy);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  Meta<kRegs> mt;
  if (load.tile < tiles) mt.load(w, load.tile, load.chunk, lane, up);

  const int esize = dtype == SPR_F32 ? 4 : 2;
  const bool wide = esize == 2 && x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0;
  for (int i = threadIdx.x; i < nb * rows * 4; i += blockDim.x) {
    const int word = i & 3, r = (i >> 2) % rows, b = (i >> 2) / rows;
    const int k = (b0 + b) * 32 + word * 8;
    const int64_t at_x = (int64_t)(row0 + r) * x_stride + k;
    float v[8];
    if (wide && k + 8 <= w.k) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>((const char*)x + at_x * 2));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t h = (&u.x)[e >> 1] >> (16 * (e & 1)) & 0xffffu;
        v[e] = dtype == SPR_BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < w.k ? load_as_f32(x, dtype, at_x + e) : 0.f;
    }
    for (int p = 0; p < parts; ++p) {
      uint32_t h[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = bf16_part(v[e] * down, p);
      xs[(b * cols + r * parts + p) * 4 + word] =
          make_uint4(bf16_pair(h[0], h[4]), bf16_pair(h[1], h[5]), bf16_pair(h[2], h[6]), bf16_pair(h[3], h[7]));
    }
  }
  mt.store(meta, lane);
  __syncthreads();
  next(load);

  float acc[NT][4] = {};
  int stage = 0, buffer = 0, odd = 0;
  const int t = lane & 3, r8 = lane >> 2;
  const char* codes_at = ring + r8 * 128 + t * 4;
  while (at.tile < tiles) {
    if (load.tile < tiles) mt.load(w, load.tile, load.chunk, lane, up);
    next(load);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncwarp();
    const int first = at.chunk * kBlocks, here = min(kBlocks, w.blocks - first);
    const char* words = codes_at + stage * kStageBytes;
    const float2* mp = meta + buffer * 32 * kRegs + r8;
    float c[NT][4];
    float2 m0, m1;
    int left = 0, g = 0;  // of a group's blocks, without GB
    if (GB == 0) left = w.group_blocks - first % w.group_blocks;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
      if (b < here) {
        const bool begins = GB ? b % (GB ? GB : 1) == 0 : b == 0 || left == w.group_blocks;
        if (begins) {
          const int gi = GB ? b / (GB ? GB : 1) : g;
          m0 = mp[gi * 16];
          m1 = mp[gi * 16 + 8];
#pragma unroll
          for (int q = 0; q < NT; ++q) c[q][0] = c[q][1] = c[q][2] = c[q][3] = 0.f;
        }
        const int at16 = (b ^ r8) << 4;
        const uint32_t u0 = *reinterpret_cast<const uint32_t*>(words + at16);
        const uint32_t u1 = *reinterpret_cast<const uint32_t*>(words + at16 + 1024);
        const uint32_t z0 = __float_as_uint(m0.y), z1 = __float_as_uint(m1.y);
        const uint32_t a0 = codes<0>(u0, z0), a1 = codes<0>(u1, z1), a2 = codes<1>(u0, z0), a3 = codes<1>(u1, z1);
        const uint32_t d0 = codes<2>(u0, z0), d1 = codes<2>(u1, z1), d2 = codes<3>(u0, z0), d3 = codes<3>(u1, z1);
        const uint4* xb = xs + ((first - b0 + b) * cols) * 4 + t;
#pragma unroll
        for (int q = 0; q < NT; ++q) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (q * 8 + r8 < cols) v = xb[(q * 8 + r8) * 4];
          mma_bf16(c[q], a0, a1, a2, a3, v.x, v.y);
          mma_bf16(c[q], d0, d1, d2, d3, v.z, v.w);
        }
        const bool ends = b == here - 1 || (GB ? b % (GB ? GB : 1) == (GB ? GB : 1) - 1 : left == 1);
        if (ends) {
#pragma unroll
          for (int q = 0; q < NT; ++q) {
            acc[q][0] = fmaf(c[q][0], m0.x, acc[q][0]);
            acc[q][1] = fmaf(c[q][1], m0.x, acc[q][1]);
            acc[q][2] = fmaf(c[q][2], m1.x, acc[q][2]);
            acc[q][3] = fmaf(c[q][3], m1.x, acc[q][3]);
          }
        }
        if (GB == 0 && --left == 0) {
          left = w.group_blocks;
          ++g;
        }
      }
    }
    // The stage that this fetch fills was read in the round before.
    fetch(stage == 0 ? kStages - 1 : stage - 1);
    stage = stage + 1 == kStages ? 0 : stage + 1;
    buffer ^= 1;
    mt.store(meta + buffer * 32 * kRegs, lane);
    const int64_t tile = at.tile;
    next(at);
    if (at.tile == tile) {
      __syncwarp();
      continue;
    }
    // The tile is done: join the warps' sums and the parts.
    float* mine = red + ((odd * sh.tiles + wt) * sh.along + wk) * kTile * NT * 8;
#pragma unroll
    for (int q = 0; q < NT; ++q) {
      *reinterpret_cast<float2*>(mine + r8 * NT * 8 + q * 8 + 2 * t) = make_float2(acc[q][0], acc[q][1]);
      *reinterpret_cast<float2*>(mine + (r8 + 8) * NT * 8 + q * 8 + 2 * t) = make_float2(acc[q][2], acc[q][3]);
      acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0.f;
    }
    if (sh.along > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + wt), "r"(sh.along * 32) : "memory");
    else __syncwarp();
    const float* sums = red + (odd * sh.tiles + wt) * sh.along * kTile * NT * 8;
    for (int i = wk * 32 + lane; i < kTile * rows; i += sh.along * 32) {
      const int row = i % kTile, r = i / kTile;
      const int64_t n = tile * kTile + row;
      if (n >= w.n) continue;
      float v = 0.f;
      for (int q = 0; q < sh.along; ++q)
        for (int p = 0; p < parts; ++p) v += sums[(q * kTile + row) * NT * 8 + r * parts + p];
      if (partial) partial[((int64_t)blockIdx.z * all_rows + row0 + r) * w.n + n] = v;
      else store_f32(y, dtype, (row0 + r) * w.n + n, bias ? v + load_as_f32(bias, dtype, n) : v);
    }
    odd ^= 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Joins the slices in their order.
__global__ void __launch_bounds__(256)
int4_join_kernel(const float* partial, int slices, int64_t size, int64_t n, const void* bias, void* y, int dtype) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= size) return;
  float v = 0.f;
  for (int s = 0; s < slices; ++s) v += partial[s * size + i];
  store_f32(y, dtype, i, bias ? v + load_as_f32(bias, dtype, i % n) : v);
}

// One warp per word column (eight k); a lane takes weight rows.
__global__ void __launch_bounds__(256)
int4_linear_grad_kernel(const void* dy, int64_t dy_stride, int dtype, int64_t rows, int64_t n, int64_t k, int group,
                        const uint32_t* packed, const void* scales, int scale_dtype, const uint8_t* zeros, void* dx) {
  const int64_t groups = (k + group - 1) / group, words = groups * group / 8;
  const int64_t w = (int64_t)blockIdx.x * (256 / 32) + (threadIdx.x >> 5);
  if (w >= words) return;
  const int lane = threadIdx.x & 31;
  const int64_t g = w * 8 / group, r = blockIdx.y;
  float acc[8] = {};
  for (int64_t col = lane; col < n; col += 32) {
    const uint32_t word = packed[col * words + w];
    const float z = zeros ? (float)zeros[col * groups + g] : 8.f;
    const float d = load_as_f32(dy, dtype, r * dy_stride + col) * load_as_f32(scales, scale_dtype, col * groups + g);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(d, (float)((word >> (4 * j)) & 15) - z, acc[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if (lane == 0 && w * 8 + j < k) store_f32(dx, dtype, r * k + w * 8 + j, acc[j]);
  }
}

int check_int4(const char* what, int64_t stride, int dtype, int64_t rows, int64_t n, int64_t k, int64_t row_len,
               int group, const void* packed, int scale_dtype) {
  if (rows < 0 || n < 0 || k < 1)
    return fail(SPR_ERR_SHAPE, "%s: rows=%lld n=%lld k=%lld", what, (long long)rows, (long long)n, (long long)k);
  if (rows > 65535 || n > 0x7fffffffLL || k > 0x7fffffffLL - (1 << 20))
    return fail(SPR_ERR_SHAPE, "%s: rows=%lld n=%lld k=%lld too large", what, (long long)rows, (long long)n,
                (long long)k);
  if (group < 32 || group % 32 || group > (1 << 20))
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

int parts_of(int dtype) { return dtype == SPR_BF16 ? 1 : dtype == SPR_F16 ? 2 : 3; }

Weights make_weights(const uint8_t* packed, const void* scales, int scale_dtype, const uint8_t* zeros, int64_t n,
                     int64_t k, int group) {
  Weights w{packed, scales, zeros, scale_dtype, n, (int)k, (int)((k + group - 1) / group), group / 32, 0};
  w.blocks = w.groups * w.group_blocks;
  return w;
}

struct ForwardPlan {
  Shape sh;
  int pass_rows, passes, nt, gb, grid, smem;
};

// Rows a pass: what 32 columns of a product hold.  The columns of the weight are cut
// into slices where the staged rows would take more than 64 KB a CTA, and where
// fewer than two tiles a SM would leave SMs without work.
ForwardPlan plan_forward(int64_t rows, const Weights& w, int dtype) {
  ForwardPlan p{};
  const int parts = parts_of(dtype);
  p.pass_rows = (int)std::min<int64_t>(rows, 32 / parts);
  p.passes = (int)((rows + p.pass_rows - 1) / p.pass_rows);
  const int cols = p.pass_rows * parts;
  p.nt = cols <= 8 ? 1 : cols <= 16 ? 2 : 4;
  p.gb = w.group_blocks == 1 || w.group_blocks == 2 || w.group_blocks == 4 ? w.group_blocks : 0;
  const int chunks = (w.blocks + kBlocks - 1) / kBlocks;
  const int64_t tiles = (w.n + kTile - 1) / kTile;
  const int chunk_bytes = kBlocks * cols * 64;
  const int64_t sms = sm_count();
  int slices = std::max(1, (int)(((int64_t)chunks * chunk_bytes + 65535) / 65536));
  if (tiles * p.passes < sms) slices = std::max<int64_t>(slices, std::min<int64_t>(chunks / 4, sms / (tiles * p.passes)));
  p.sh.slice_chunks = (chunks + slices - 1) / slices;
  p.sh.slices = (chunks + p.sh.slice_chunks - 1) / p.sh.slice_chunks;
  // Warps on a tile: the number that shares its chunks most evenly.
  int along = 1;
  for (int a = 2; a <= std::min(kWarps, p.sh.slice_chunks); ++a) {
    const int steps_a = (p.sh.slice_chunks + a - 1) / a, steps = (p.sh.slice_chunks + along - 1) / along;
    if (steps_a * a * 8 <= p.sh.slice_chunks * 9 || steps_a * a <= steps * along) along = a;
  }
  p.sh.along = along;
  const int64_t work = tiles * p.passes * p.sh.slices;
  p.sh.tiles = (int)std::max<int64_t>(1, std::min<int64_t>(kWarps / along, work / (2 * sms)));
  const int warps = along * p.sh.tiles;
  p.smem = warps * (kStages * kStageBytes + 2 * 32 * kMetaRegs(p.gb) * 8 + 2 * kTile * p.nt * 8 * 4) +
           p.sh.slice_chunks * chunk_bytes;
  const int64_t teams = (tiles + p.sh.tiles - 1) / p.sh.tiles;
  const int64_t fit = std::max(1, std::min(227 * 1024 / (p.smem + 1024), 16 / warps));  // 128 registers a thread
  p.grid = (int)std::min(teams, std::max<int64_t>(1, sms * fit / (p.passes * p.sh.slices)));
  return p;
}

template <int NT, int GB>
int launch_forward(const ForwardPlan& p, const Weights& w, const void* x, int64_t x_stride, int dtype, int rows,
                   const void* bias, void* y, float* partial, cudaStream_t st) {
  auto kern = int4_linear_kernel<NT, GB>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024) != cudaSuccess)
    return check_launch("int4 linear");
  // A group's inner sum of up to 15*group values of x stays below the largest fp32
  // number: x is taken times a power of two and the scale divided by it.
  int e = 4;
  while ((1 << (e - 4)) < w.group_blocks * 32) ++e;
  const dim3 grid(p.grid, p.passes, p.sh.slices);
  kern<<<grid, p.sh.along * p.sh.tiles * 32, p.smem, st>>>(w, p.sh, x, x_stride, dtype, parts_of(dtype), rows,
                                                           p.pass_rows, ldexpf(1.f, -e), ldexpf(1.f, e),
                                                           partial ? nullptr : bias, y, partial);
  if (partial) {
    const int64_t size = (int64_t)rows * w.n;
    int4_join_kernel<<<(unsigned)((size + 255) / 256), 256, 0, st>>>(partial, p.sh.slices, size, w.n, bias, y, dtype);
  }
  return check_launch("int4 linear");
}

template <int NT>
int launch_forward_by_group(const ForwardPlan& p, const Weights& w, const void* x, int64_t x_stride, int dtype, int rows,
                            const void* bias, void* y, float* partial, cudaStream_t st) {
  if (p.gb == 1) return launch_forward<NT, 1>(p, w, x, x_stride, dtype, rows, bias, y, partial, st);
  if (p.gb == 2) return launch_forward<NT, 2>(p, w, x, x_stride, dtype, rows, bias, y, partial, st);
  if (p.gb == 4) return launch_forward<NT, 4>(p, w, x, x_stride, dtype, rows, bias, y, partial, st);
  return launch_forward<NT, 0>(p, w, x, x_stride, dtype, rows, bias, y, partial, st);
}

}  // namespace

}  // namespace spr

using namespace spr;

extern "C" size_t spr_int4_linear_workspace_bytes(int64_t rows, int64_t n, int64_t k, int group, int dtype) {
  if (rows <= 0 || n <= 0 || k <= 0 || group < 32) return 0;
  const ForwardPlan p = plan_forward(rows, make_weights(nullptr, nullptr, 0, nullptr, n, k, group), dtype);
  return p.sh.slices > 1 ? (size_t)p.sh.slices * rows * n * sizeof(float) : 0;
}

extern "C" int spr_int4_linear(const void* x, int64_t x_stride, int dtype, int64_t rows, int64_t n, int64_t k,
                               int group, const uint8_t* packed, const void* scales, int scale_dtype,
                               const uint8_t* zeros, const void* bias, void* y, void* workspace,
                               size_t workspace_bytes, void* stream) {
  if (int rc = check_int4("int4 linear", x_stride, dtype, rows, n, k, k, group, packed, scale_dtype)) return rc;
  if (rows == 0 || n == 0) return SPR_OK;
  if (!x || !packed || !scales || !y) return fail(SPR_ERR_ARG, "int4 linear: null operand");
  const Weights w = make_weights(packed, scales, scale_dtype, zeros, n, k, group);
  const ForwardPlan p = plan_forward(rows, w, dtype);
  const size_t need = p.sh.slices > 1 ? (size_t)p.sh.slices * rows * n * sizeof(float) : 0;
  if (need && (!workspace || workspace_bytes < need))
    return fail(SPR_ERR_WORKSPACE, "int4 linear: workspace %zu < %zu bytes", workspace_bytes, need);
  float* partial = need ? (float*)workspace : nullptr;
  cudaStream_t st = (cudaStream_t)stream;
  if (p.nt == 1) return launch_forward_by_group<1>(p, w, x, x_stride, dtype, (int)rows, bias, y, partial, st);
  if (p.nt == 2) return launch_forward_by_group<2>(p, w, x, x_stride, dtype, (int)rows, bias, y, partial, st);
  return launch_forward_by_group<4>(p, w, x, x_stride, dtype, (int)rows, bias, y, partial, st);
}

extern "C" size_t spr_int4_linear_grad_workspace_bytes(int64_t, int64_t, int64_t, int, int) { return 0; }

extern "C" int spr_int4_linear_grad(const void* dy, int64_t dy_stride, int dtype, int64_t rows, int64_t n, int64_t k,
                                    int group, const uint8_t* packed, const void* scales, int scale_dtype,
                                    const uint8_t* zeros, void* dx, void* workspace, size_t workspace_bytes,
                                    void* stream) {
  (void)workspace;
  (void)workspace_bytes;
  if (int rc = check_int4("int4 linear grad", dy_stride, dtype, rows, n, k, n, group, packed, scale_dtype)) return rc;
  if (rows == 0) return SPR_OK;
  if (!dx || (n && (!dy || !packed || !scales))) return fail(SPR_ERR_ARG, "int4 linear grad: null operand");
  const int64_t words = (k + group - 1) / group * group / 8;
  const dim3 grid((unsigned)((words + 256 / 32 - 1) / (256 / 32)), (unsigned)rows);
  int4_linear_grad_kernel<<<grid, 256, 0, (cudaStream_t)stream>>>(dy, dy_stride, dtype, rows, n, k, group,
                                                                       (const uint32_t*)packed, scales, scale_dtype,
                                                                       zeros, dx);
  return check_launch("int4 linear grad");
}
