// Modulated layer norm with an optional gated residual in front of it, forward
// and backward (the operands are described at SprAdaln in the header):
//   z = x + gate*y,  n = (z - mean z) * rstd,  h = n*w + shift,  w = offset + scale
//   u = dh*w,  g = dz + rstd*(u - mean u - n*mean(u*n)),  dx = g,  dy = g*gate
//   dshift = sum dh,  dscale = sum dh*n,  dgate = sum g*y   over the rows of a group
// Statistics and sums are fp32, and each result is rounded once.  A row is read once
// and written once a pass, 2 to 4 fp32 operations a byte, so HBM bounds every pass of
// more than a few hundred rows; below that the launch does.  Bandwidths in this
// file are of B200's measured copy, 6.56 TB/s, under a sustained load.
#include <atomic>
#include <tuple>
#include <type_traits>

#include "common.cuh"

namespace spr {

namespace {

constexpr int kMaxChannels = 16384;

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// Element vectors: 16 bytes of T (V elements) where the width, the strides and the
// pointers allow it, single elements otherwise.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// Two fp32 operations in one instruction, each rounded by itself.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1,%2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t p) {
  float2 f;
  asm("mov.b64 {%0,%1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
  return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// V fp32 values as pairs; a single element leaves the second half 0.
template <int V>
struct Vals {
  static constexpr int kPairs = (V + 1) / 2;
  uint64_t q[kPairs];
  __device__ __forceinline__ void fill(float v) {
#pragma unroll
    for (int i = 0; i < kPairs; ++i) q[i] = pair(v, V == 1 ? 0.f : v);
  }
};
template <int V>
__device__ __forceinline__ uint64_t both(float v) { return pair(v, V == 1 ? 0.f : v); }

template <typename T>
__device__ __forceinline__ uint64_t widen(uint32_t u);  // two 16-bit values
template <>
__device__ __forceinline__ uint64_t widen<__nv_bfloat16>(uint32_t u) {
  return pair(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
template <>
__device__ __forceinline__ uint64_t widen<__half>(uint32_t u) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
  return pair(f.x, f.y);
}
template <typename T>
__device__ __forceinline__ uint32_t narrow(uint64_t p);
template <>
__device__ __forceinline__ uint32_t narrow<__nv_bfloat16>(uint64_t p) {
  const float2 f = halves(p);
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t narrow<__half>(uint64_t p) {
  const float2 f = halves(p);
  const __half2 h = __floats2half2_rn(f.x, f.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The elements of 16 bytes of T, at q[0 .. kVec<T>/2).
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& u, uint64_t* q) {
  if constexpr (sizeof(T) == 4) {
    q[0] = pair(__uint_as_float(u.x), __uint_as_float(u.y));
    q[1] = pair(__uint_as_float(u.z), __uint_as_float(u.w));
  } else {
    q[0] = widen<T>(u.x);
    q[1] = widen<T>(u.y);
    q[2] = widen<T>(u.z);
    q[3] = widen<T>(u.w);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const uint64_t* q) {
  if constexpr (sizeof(T) == 4) {
    const float2 a = halves(q[0]), b = halves(q[1]);
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  } else {
    return make_uint4(narrow<T>(q[0]), narrow<T>(q[1]), narrow<T>(q[2]), narrow<T>(q[3]));
  }
}

// Rows pass the L1 by; vectors that many rows read stay in it.
template <typename T, int V>
__device__ __forceinline__ void load_row(const T* p, Vals<V>& f) {
  if constexpr (V == 1) {
    f.q[0] = pair(to_f32(__ldg(p)), 0.f);
  } else {
    uint4 u;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                 : "l"(p));
    unpack16<T>(u, f.q);
  }
}
template <typename MT, int V>
__device__ __forceinline__ void load_vector(const MT* p, Vals<V>& f) {
  if constexpr (V == 1) {
    f.q[0] = pair(to_f32(__ldg(p)), 0.f);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += kVec<MT>) unpack16<MT>(__ldg(reinterpret_cast<const uint4*>(p + i)), f.q + i / 2);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_row(T* p, const Vals<V>& f) {
  if constexpr (V == 1) {
    p[0] = from_f32<T>(halves(f.q[0]).x);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += kVec<T>) *reinterpret_cast<uint4*>(p + i) = pack16<T>(f.q + i / 2);
  }
}

// A row belongs to a team of threads: a power of two of lanes up to 32 (several
// teams to a warp, no barrier), or a whole CTA of several warps.
__device__ __forceinline__ float team_sum(float v, int team) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < team) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t team_sum2(uint64_t v, int team) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < team) v = add2(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Two sums over a CTA's warps with one barrier.  Two buffers in turn: a warp that
// writes the next row's pair does not meet readers of this row's.  `red` starts
// as zeros, so an odd number of warps reads a zero pair.
__device__ __forceinline__ uint64_t join_warps(const ulonglong2* red, int warps) {
  uint64_t a = 0, b = 0;
#pragma unroll 4
  for (int w = 0; w < (warps + 1) / 2; ++w) {
    const ulonglong2 e = red[w];
    a = add2(a, e.x);
    b = add2(b, e.y);
  }
  return add2(a, b);
}
__device__ __forceinline__ uint64_t warps_sum2(uint64_t v, ulonglong2* red, int warps) {
  if ((threadIdx.x & 31) == 0) reinterpret_cast<uint64_t*>(red)[threadIdx.x >> 5] = v;
  __syncthreads();
  return join_warps(red, warps);
}

// The residual stream: product and sum rounded to fp32 one after the other, so
// that z is what the two separate operations store (the paired forms were joined
// to one rounding by the compiler).
template <typename T, int V>
__device__ __forceinline__ void residual(Vals<V>& x, const Vals<V>& y, const Vals<V>& gate) {
#pragma unroll
  for (int i = 0; i < Vals<V>::kPairs; ++i) {
    const float2 a = halves(x.q[i]), b = halves(y.q[i]), g = halves(gate.q[i]);
    x.q[i] = pair(__fadd_rn(a.x, __fmul_rn(g.x, b.x)), __fadd_rn(a.y, __fmul_rn(g.y, b.y)));
    if constexpr (sizeof(T) == 2) x.q[i] = widen<T>(narrow<T>(x.q[i]));
  }
}

struct RowId {
  int64_t b, t;
};
__device__ __forceinline__ RowId row_id(const SprAdaln& op, int64_t row) {
  if (op.batch == 1) return {0, row};
  const uint32_t b = (uint32_t)row / (uint32_t)op.tokens;  // batch*tokens < 2^31
  return {b, row - (int64_t)b * op.tokens};
}

template <typename MT, int V>
__device__ __forceinline__ void load_factor(const SprAdaln& op, const RowId& id, int v, Vals<V>& w) {
  if (op.scale) {
    load_vector<MT, V>((const MT*)op.scale + id.b * op.scale_sb + id.t * op.scale_st + v * V, w);
    const uint64_t offset = both<V>(op.scale_offset);
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i) w.q[i] = add2(w.q[i], offset);
  } else {
    w.fill(1.f);
  }
}
template <typename MT, int V>
__device__ __forceinline__ void load_gate(const SprAdaln& op, const RowId& id, int v, Vals<V>& w) {
  if (op.gate) load_vector<MT, V>((const MT*)op.gate + id.b * op.gate_sb + id.t * op.gate_st + v * V, w);
  else w.fill(1.f);
}

// The rows that share one vector: row r of group g is g*group_step + r*row_step.
// A group's rows are cut into `chunks` runs; run s of group g writes its column
// sums to partial[g][s] (or, with one run, the gradients themselves).
struct Groups {
  int64_t count, rows, group_step, row_step;
  int chunks;
  int64_t chunk_rows;
};

__device__ __forceinline__ void copy16_async(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}

// Mean and 1/sqrt(var + eps) of a row that a team holds.  The variance is taken about
// the warp's own mean and the warps' values are joined by
//   M2 = sum_w M2_w + n_w (mean_w - mean)^2,
// so that a row costs one barrier and loses nothing to an offset.
template <int V, int P>
__device__ __forceinline__ float2 row_stats(const Vals<V> (&z)[P], int lane, int team, int nvec, float inv_c, float eps,
                                            float4* red) {
  const int first = lane & ~31, width = min(team, 32);  // the warp's vectors in its team
  int n = 0;
  uint64_t acc[2] = {0, 0};
#pragma unroll
  for (int p = 0; p < P; ++p) {
    n += min(max(nvec - first - p * team, 0), width) * V;
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i) acc[i & 1] = add2(acc[i & 1], z[p].q[i]);
  }
  float2 h = halves(add2(acc[0], acc[1]));
  const float sum = team_sum(h.x + h.y, team);
  float mean = sum * __frcp_rn((float)n);
  const uint64_t minus = both<V>(-mean);
  acc[0] = acc[1] = 0;
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (lane + p * team < nvec)
#pragma unroll
      for (int i = 0; i < Vals<V>::kPairs; ++i) {
        const uint64_t d = add2(z[p].q[i], minus);
        acc[i & 1] = fma2(d, d, acc[i & 1]);
      }
  h = halves(add2(acc[0], acc[1]));
  float m2 = team_sum(h.x + h.y, team);
  if (team > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float4(sum, mean, m2, (float)n);
    __syncthreads();
    const int w = threadIdx.x & 31;
    const float4 part = w < team / 32 ? red[w] : make_float4(0.f, 0.f, 0.f, 0.f);
    mean = team_sum(part.x, 32) * inv_c;
    const float d = part.y - mean;
    m2 = team_sum(fmaf(d * d, part.w, part.z), 32);
  }
  return make_float2(mean, rsqrtf(m2 * inv_c + eps));
}

// One row per team, kept in registers: few rows, any width and alignment, and the
// widest rows with a vector each.  Four rows of 5120 take 3 us, all of it latency.  Nothing
// is copied ahead, and a CTA ends with its rows: 10,000 x 12,288 bf16 138 us (54% of
// bandwidth).
template <typename T, typename MT, int V, int P, bool kRes>
__global__ void __launch_bounds__(1024) adaln_forward_kernel(const SprAdaln op, int team) {
  __shared__ float4 red[32];
  const int c = op.channels, nvec = c / V;
  const int lane = threadIdx.x % team;
  const int64_t rows = op.batch * op.tokens;
  const int64_t want = (int64_t)blockIdx.x * (blockDim.x / team) + threadIdx.x / team;
  const bool valid = want < rows;
  const int64_t row = valid ? want : rows - 1;  // a team past the end repeats the last row and stores nothing
  const RowId id = row_id(op, row);
  const T* x = (const T*)op.x + id.b * op.x_sb + id.t * op.x_st;
  Vals<V> z[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int v = lane + p * team;
    if (v < nvec) load_row<T, V>(x + v * V, z[p]);
    else z[p].fill(0.f);
  }
  if constexpr (kRes) {
    const T* y = (const T*)op.y + id.b * op.y_sb + id.t * op.y_st;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int v = lane + p * team;
      if (v < nvec) {
        Vals<V> yv, gv;
        load_row<T, V>(y + v * V, yv);
        load_gate<MT, V>(op, id, v, gv);
        residual<T, V>(z[p], yv, gv);
        if (valid) store_row<T, V>((T*)op.z + row * c + v * V, z[p]);
      }
    }
  }
  const float2 ms = row_stats<V, P>(z, lane, team, nvec, __frcp_rn((float)c), op.eps, red);
  const float mean = ms.x, rstd = ms.y;
  if (!valid) return;
  const uint64_t minus = both<V>(-mean);
  const uint64_t r2 = both<V>(rstd);
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int v = lane + p * team;
    if (v >= nvec) continue;
    Vals<V> w, b;
    load_factor<MT, V>(op, id, v, w);
    if (op.shift) load_vector<MT, V>((const MT*)op.shift + id.b * op.shift_sb + id.t * op.shift_st + v * V, b);
    else b.fill(0.f);
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i) z[p].q[i] = fma2(mul2(add2(z[p].q[i], minus), r2), w.q[i], b.q[i]);
    store_row<T, V>((T*)op.h + row * c + v * V, z[p]);
  }
  if (lane == 0 && op.mean) {
    op.mean[row] = mean;
    op.rstd[row] = rstd;
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// The sum over lanes 0..15 (a CTA's warps, one a lane) in all of them.
__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, 16);
  return v;
}

// Where a run's rows lie: the first row and the step to the next, for rows that are
// equally spaced in every operand.
struct Run {
  int64_t row0, step;
  int rows;
  RowId first, group;
  __device__ __forceinline__ Run(const SprAdaln& op, const Groups& gp, int64_t unit) {
    const int64_t g = unit / gp.chunks, r0 = unit % gp.chunks * gp.chunk_rows;
    row0 = g * gp.group_step + r0 * gp.row_step;
    step = gp.row_step;
    rows = (int)(min(gp.rows, r0 + gp.chunk_rows) - r0);
    first = row_id(op, row0);
    group = row_id(op, g * gp.group_step);
  }
  __device__ __forceinline__ const char* at(const void* base, int64_t sb, int64_t st, int e) const {
    return (const char*)base + (first.b * sb + first.t * st) * e + threadIdx.x * 16;
  }
};

// Vectors of a row's own (scale, shift, gate) in a ring beside the rows: of M bytes an
// element, kM 16-byte pieces for a vector of the row's elements.
template <typename T, typename MT>
constexpr int row_pieces = kVec<T> * (int)sizeof(MT) / 16;
enum Vector { kScaleVector, kShiftVector, kGateVector };
template <typename T, typename MT, int P, bool kRow, Vector... kWhich>
struct RowVectors {
  static constexpr int kM = row_pieces<T, MT>, kVectors = sizeof...(kWhich);
  const char* at[kVectors];
  int64_t step[kVectors];
  __device__ __forceinline__ RowVectors(const SprAdaln& op, const Run& run) {
    if constexpr (kRow) {
      constexpr Vector which[kVectors] = {kWhich...};
      const void* base[3] = {op.scale, op.shift, op.gate};
      const int64_t sb[3] = {op.scale_sb, op.shift_sb, op.gate_sb}, st[3] = {op.scale_st, op.shift_st, op.gate_st};
#pragma unroll
      for (int j = 0; j < kVectors; ++j) {
        const int k = which[j];
        at[j] = base[k] ? (const char*)base[k] + (run.first.b * sb[k] + run.first.t * st[k]) * (int)sizeof(MT) +
                              threadIdx.x * kM * 16
                        : nullptr;
        step[j] = st[k] * (int)sizeof(MT);
      }
    }
  }
  template <typename Mine>
  __device__ __forceinline__ void copy(uint4* to, int team, Mine mine) {
#pragma unroll
    for (int j = 0; j < kVectors; ++j) {
      if (!at[j]) continue;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (mine(p))
#pragma unroll
          for (int h = 0; h < kM; ++h)
            copy16_async(to + ((j * kM + h) * P + p) * team, at[j] + (p * team * kM + h) * 16);
      at[j] += step[j];
    }
  }
  // Vector j of the row in a slot, `offset` added, or `missing` without it.
  __device__ __forceinline__ void read(const uint4* slot, int team, int p, int j, float offset, float missing,
                                       Vals<kVec<T>>& f) const {
    if (!at[j]) {
      f.fill(missing);
      return;
    }
#pragma unroll
    for (int h = 0; h < kM; ++h) unpack16<MT>(slot[((j * kM + h) * P + p) * team], f.q + h * kVec<MT> / 2);
    if (j == 0)
#pragma unroll
      for (int i = 0; i < Vals<kVec<T>>::kPairs; ++i) f.q[i] = add2(f.q[i], pair(offset, offset));
  }
};
template <typename T, typename MT, int P, bool kRow, bool kRes>
using ForwardVectors = std::conditional_t<kRes, RowVectors<T, MT, P, kRow, kScaleVector, kShiftVector, kGateVector>,
                                          RowVectors<T, MT, P, kRow, kScaleVector, kShiftVector>>;
template <typename T, typename MT, int P, bool kRow, bool kRes>
using BackwardVectors = std::conditional_t<kRes, RowVectors<T, MT, P, kRow, kScaleVector, kGateVector>,
                                           RowVectors<T, MT, P, kRow, kScaleVector>>;

// Long groups of wide rows that share their vectors: CTAs that stay on their SM walk
// runs of rows with the vectors in registers, P 16-byte vectors a thread.  Each
// thread copies its own vectors of the next kStages - 1 rows into shared memory:
// the copies need no barrier and stay in flight across the one that joins a row's
// statistics.  kFull: every thread has all of its P vectors.  kRow: each row has
// vectors of its own, which are streamed as the rows are.
// 75,600 x 5120 bf16: 249 us (95%), gated with fp32 vectors 490 us (96%); 60,000 x 2048
// fp32 gated 317 us (94%); 40,000 x 1536 bf16 gated with vectors for every row 136 us (97%).
template <typename T, typename MT, int P, bool kRes, bool kFull, bool kRow, int kThreads, int kMin, int kStages>
__global__ void __launch_bounds__(kThreads, kMin) adaln_forward_stream_kernel(const SprAdaln op, const Groups gp) {
  constexpr int V = kVec<T>, kIn = kRes ? 2 : 1, e = sizeof(T);
  constexpr int kM = kRow ? row_pieces<T, MT> : 0, kAll = kIn + kM * (kRes ? 3 : 2);
  __shared__ float2 red[2][16];
  extern __shared__ uint4 ring[];  // [stage][operand][P][thread]
  const int c = op.channels, nvec = c / V, team = blockDim.x, lane = threadIdx.x, warps = team / 32;
  const Run run(op, gp, blockIdx.x);
  auto mine = [&](int p) { return kFull || lane + p * team < nvec; };
  // This warp's elements, and those of warp `lane` for the join.
  auto elements = [&](int w) {
    int n = 0;
#pragma unroll
    for (int p = 0; p < P; ++p) n += min(max(nvec - 32 * w - p * team, 0), 32) * V;
    return (float)n;
  };
  const int who = lane & 15;
  const float n_who = who < warps ? elements(who) : 0.f;
  const float inv_who = n_who > 0.f ? __frcp_rn(n_who) : 0.f;
  const float inv_n = __frcp_rn(elements(lane >> 5)), inv_c = __frcp_rn((float)c);
  if (lane < 32) red[lane >> 4][lane & 15] = make_float2(0.f, 0.f);
  __syncthreads();
  const char* x = run.at(op.x, op.x_sb, op.x_st, e);
  const char* y = kRes ? run.at(op.y, op.y_sb, op.y_st, e) : nullptr;
  const int64_t x_step = (run.step == 1 ? op.x_st : op.x_sb) * e, y_step = (run.step == 1 ? op.y_st : op.y_sb) * e;
  ForwardVectors<T, MT, P, kRow, kRes> vec(op, run);
  int fetched = 0;
  auto fetch = [&](int stage) {
    if (fetched++ < run.rows) {
      uint4* to = ring + stage * (kAll * P) * team + lane;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (mine(p)) {
          copy16_async(to + p * team, x + p * team * 16);
          if constexpr (kRes) copy16_async(to + (P + p) * team, y + p * team * 16);
        }
      x += x_step;
      if constexpr (kRes) y += y_step;
      if constexpr (kRow) vec.copy(to + kIn * P * team, team, [&](int p) { return mine(p); });
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  constexpr int kHeld = kRow ? 1 : P;
  Vals<V> w[kHeld], b[kHeld], gate[kHeld];
#pragma unroll
  for (int p = 0; p < (kRow ? 0 : P); ++p) {
    const int v = lane + p * team;
    if (!mine(p)) continue;
    load_factor<MT, V>(op, run.group, v, w[p]);
    if (op.shift)
      load_vector<MT, V>((const MT*)op.shift + run.group.b * op.shift_sb + run.group.t * op.shift_st + v * V, b[p]);
    else b[p].fill(0.f);
    if constexpr (kRes) load_gate<MT, V>(op, run.group, v, gate[p]);
  }
  int stage = 0;
  char* z_out = (char*)op.z + (run.row0 * c * e + lane * 16);
  char* h_out = (char*)op.h + (run.row0 * c * e + lane * 16);
  const int64_t out_step = run.step * c * e;
  for (int r = 0; r < run.rows; ++r) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    const uint4* slot = ring + stage * (kAll * P) * team + lane;
    Vals<V> z[P];
    uint64_t acc[2] = {0, 0};
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (!mine(p)) continue;
      unpack16<T>(slot[p * team], z[p].q);
      if constexpr (kRes) {
        Vals<V> yv;
        unpack16<T>(slot[(P + p) * team], yv.q);
        if constexpr (kRow) vec.read(slot + kIn * P * team, team, p, 2, 0.f, 1.f, gate[0]);
        residual<T, V>(z[p], yv, gate[kRow ? 0 : p]);
        *reinterpret_cast<uint4*>(z_out + p * team * 16) = pack16<T>(z[p].q);
      }
#pragma unroll
      for (int i = 0; i < V / 2; ++i) acc[i & 1] = add2(acc[i & 1], z[p].q[i]);
    }
    // The slot that this fetch fills was read in the round before.
    fetch(stage == 0 ? kStages - 1 : stage - 1);
    float2 h = halves(add2(acc[0], acc[1]));
    const float sum = warp_sum(h.x + h.y);
    const float near = -sum * inv_n;
    acc[0] = acc[1] = 0;
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (mine(p))
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const uint64_t d = add2(z[p].q[i], pair(near, near));
          acc[i & 1] = fma2(d, d, acc[i & 1]);
        }
    h = halves(add2(acc[0], acc[1]));
    float m2 = warp_sum(h.x + h.y);
    if ((lane & 31) == 0) red[r & 1][lane >> 5] = make_float2(sum, m2);
    __syncthreads();
    // M2 = sum_w M2_w + n_w (mean_w - mean)^2, a warp's values in each of 16 lanes.
    const float2 part = red[r & 1][who];
    const float mean = sum16(part.x) * inv_c;
    const float off = fmaf(part.x, inv_who, -mean);
    const float rstd = rsqrtf(sum16(fmaf(off * off, n_who, part.y)) * inv_c + op.eps);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (!mine(p)) continue;
      constexpr int kHold = kRow ? 0 : 1;
      if constexpr (kRow) {
        vec.read(slot + kIn * P * team, team, p, 0, op.scale_offset, 1.f, w[0]);
        vec.read(slot + kIn * P * team, team, p, 1, 0.f, 0.f, b[0]);
      }
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        z[p].q[i] = fma2(mul2(add2(z[p].q[i], pair(-mean, -mean)), pair(rstd, rstd)), w[p * kHold].q[i], b[p * kHold].q[i]);
      *reinterpret_cast<uint4*>(h_out + p * team * 16) = pack16<T>(z[p].q);
    }
    if (lane == 0 && op.mean) {
      op.mean[run.row0 + r * run.step] = mean;
      op.rstd[run.row0 + r * run.step] = rstd;
    }
    if constexpr (kRes) z_out += out_step;
    h_out += out_step;
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Rows that 16-byte vectors do not fit (odd widths, odd strides or offsets), in long
// groups: a CTA that stays on its SM copies the aligned 16-byte pieces which hold a
// row into shared memory, some rows ahead.  A warp takes 32*P neighbouring columns, a
// thread every 32nd of them: its columns, and its part of the vectors, are the same
// in every row, at constant distances.  The first piece may begin before the row
// (inside the allocation: these begin on multiples of 16 bytes); the last is cut at its
// end and zeros fill the place up, so that only stores and the variance look at the
// width, in the last warp.  One barrier a row: it joins the row's sums, shows every
// thread the next row, and lets the row before be overwritten.
// Bound by instructions, a load, a conversion and a store for every element: 30,000 x 1003
// fp32 47 us (78% of bandwidth), gated 92 us (80%); 16-bit elements are twice as many
// for the bytes: 30,000 x 1537 bf16 66 us (43%), gated 117 us (48%).
template <int P>
__device__ __forceinline__ int first_column() { return (threadIdx.x & ~31) * P + (threadIdx.x & 31); }
// Bytes that a row of at most `c` elements takes in a slot.
__host__ __device__ constexpr int window_bytes(int c, int e) { return (c * e + 15 + 15) / 16 * 16; }
struct Window {
  const char* at;  // the next row to copy; null: none is
  int64_t step;
  int row_bytes, place_bytes, off;
  uint32_t phase;  // where the row at work begins in its first piece
  __device__ __forceinline__ Window() : at(nullptr), step(0), row_bytes(0), place_bytes(0), off(0), phase(0) {}
  __device__ __forceinline__ Window(const Run& run, const void* base, int64_t sb, int64_t st, int e, int c, int off)
      : at(base ? (const char*)base + (run.first.b * sb + run.first.t * st) * e : nullptr),
        step((run.step == 1 ? st : sb) * e), row_bytes(c * e), place_bytes(window_bytes(c, e)), off(off), phase((uint32_t)(uintptr_t)at & 15) {}
  __device__ __forceinline__ void copy(char* slot) {
    if (!at) return;
    const int shift = (int)((uintptr_t)at & 15), bytes = shift + row_bytes;
    for (int i = threadIdx.x * 16; i < place_bytes; i += blockDim.x * 16) {
      const int some = min(max(bytes - i, 0), 16);  // the rest of the 16 is zeros
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       (uint32_t)__cvta_generic_to_shared(slot + off + i)),
                   "l"(at - shift + (some ? i : 0)), "r"(some)
                   : "memory");
    }
    at += step;
  }
  __device__ __forceinline__ void advance() { phase = (phase + (uint32_t)step) & 15; }
  // The thread's elements of the row in a slot, zeros past the end.
  template <typename U, int P>
  __device__ __forceinline__ void read(const char* slot, Vals<P>& f) const {
    const U* p = reinterpret_cast<const U*>(slot + off + phase) + first_column<P>();
#pragma unroll
    for (int i = 0; i < P / 2; ++i) f.q[i] = pair(to_f32(p[64 * i]), to_f32(p[64 * i + 32]));
  }
};

template <int P>
__device__ __forceinline__ bool whole_warp(int c) { return ((threadIdx.x & ~31) + 32) * P <= c; }
// The thread's elements of a vector or a row in memory.
template <typename U, int P>
__device__ __forceinline__ void load_columns(const U* p, int c, Vals<P>& f) {
  const int first = first_column<P>();
  p += first;
#pragma unroll
  for (int i = 0; i < P / 2; ++i)
    f.q[i] = pair(first + 64 * i < c ? to_f32(__ldg(p + 64 * i)) : 0.f,
                  first + 64 * i + 32 < c ? to_f32(__ldg(p + 64 * i + 32)) : 0.f);
}
template <typename U, int P>
__device__ __forceinline__ void store_columns(U* p, int c, const Vals<P>& f) {
  const int first = first_column<P>();
  p += first;
  const bool all = whole_warp<P>(c);
#pragma unroll
  for (int i = 0; i < P / 2; ++i) {
    const float2 v = halves(f.q[i]);
    if (all || first + 64 * i < c) p[64 * i] = from_f32<U>(v.x);
    if (all || first + 64 * i + 32 < c) p[64 * i + 32] = from_f32<U>(v.y);
  }
}
// Zeros in the whole ring, for the places behind the rows.
__device__ __forceinline__ void clear_ring(uint4* ring, int bytes) {
  for (int i = threadIdx.x; i < bytes / 16; i += blockDim.x) ring[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
}
template <int P>
__device__ __forceinline__ void add_offset(Vals<P>& w, float offset) {
#pragma unroll
  for (int i = 0; i < P / 2; ++i) w.q[i] = add2(w.q[i], pair(offset, offset));
}
__device__ __forceinline__ void wait_for_next_row(int stages) {
  if (stages == 4) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, typename MT, int P, bool kRes, bool kRow, int kThreads>
__global__ void __launch_bounds__(kThreads, 1)
adaln_forward_any_kernel(const SprAdaln op, const Groups gp, int stages, int slot_bytes) {
  __shared__ float2 red[2][16];
  extern __shared__ uint4 ring[];
  const int c = op.channels, team = blockDim.x, lane = threadIdx.x, warps = team / 32, e = sizeof(T), me = sizeof(MT);
  const Run run(op, gp, blockIdx.x);
  const int row_place = window_bytes(team * P, e), vec_place = window_bytes(team * P, me);
  Window x(run, op.x, op.x_sb, op.x_st, e, c, 0), y, scale, shift, gate;
  if constexpr (kRes) y = Window(run, op.y, op.y_sb, op.y_st, e, c, row_place);
  if constexpr (kRow) {
    constexpr int rows = kRes ? 2 : 1;
    scale = Window(run, op.scale, op.scale_sb, op.scale_st, me, c, rows * row_place);
    shift = Window(run, op.shift, op.shift_sb, op.shift_st, me, c, rows * row_place + vec_place);
    if constexpr (kRes) gate = Window(run, op.gate, op.gate_sb, op.gate_st, me, c, rows * row_place + 2 * vec_place);
  }
  auto elements = [&](int w) { return (float)min(max(c - 32 * P * w, 0), 32 * P); };
  const int who = lane & 15, first = first_column<P>();
  const bool whole = whole_warp<P>(c);
  const float n_who = who < warps ? elements(who) : 0.f;
  const float inv_who = n_who > 0.f ? __frcp_rn(n_who) : 0.f;
  const float inv_n = __frcp_rn(elements(lane >> 5)), inv_c = __frcp_rn((float)c);
  if (lane < 32) red[lane >> 4][lane & 15] = make_float2(0.f, 0.f);
  int fetched = 0;
  auto fetch = [&](int stage) {
    if (fetched++ < run.rows) {
      char* slot = reinterpret_cast<char*>(ring) + stage * slot_bytes;
      x.copy(slot);
      if constexpr (kRes) y.copy(slot);
      if constexpr (kRow) {
        scale.copy(slot);
        shift.copy(slot);
        if constexpr (kRes) gate.copy(slot);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  clear_ring(ring, stages * slot_bytes);
  for (int i = 0; i < stages - 1; ++i) fetch(i);
  Vals<P> w, b, g;
  w.fill(1.f);
  b.fill(0.f);
  g.fill(1.f);
  if constexpr (!kRow) {
    const RowId& id = run.group;
    if (op.scale) {
      load_columns<MT, P>((const MT*)op.scale + id.b * op.scale_sb + id.t * op.scale_st, c, w);
      add_offset<P>(w, op.scale_offset);
    }
    if (op.shift) load_columns<MT, P>((const MT*)op.shift + id.b * op.shift_sb + id.t * op.shift_st, c, b);
    if (kRes && op.gate) load_columns<MT, P>((const MT*)op.gate + id.b * op.gate_sb + id.t * op.gate_st, c, g);
  }
  if (stages == 4) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 1;" ::: "memory");
  __syncthreads();
  int stage = 0;
  for (int r = 0; r < run.rows; ++r) {
    const char* slot = reinterpret_cast<const char*>(ring) + stage * slot_bytes;
    const int64_t row = run.row0 + r * run.step;
    Vals<P> z;
    x.read<T, P>(slot, z);
    if constexpr (kRes) {
      Vals<P> yv;
      y.read<T, P>(slot, yv);
      if (kRow && gate.at) gate.read<MT, P>(slot, g);
      residual<T, P>(z, yv, g);
      store_columns<T, P>((T*)op.z + row * c, c, z);
    }
    uint64_t acc[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < P / 2; ++i) acc[i & 1] = add2(acc[i & 1], z.q[i]);
    float2 h = halves(add2(acc[0], acc[1]));
    const float sum = warp_sum(h.x + h.y);
    const float near = -sum * inv_n;
    acc[0] = acc[1] = 0;
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      uint64_t d = add2(z.q[i], pair(near, near));
      if (!whole) {
        const float2 f = halves(d);
        d = pair(first + 64 * i < c ? f.x : 0.f, first + 64 * i + 32 < c ? f.y : 0.f);
      }
      acc[i & 1] = fma2(d, d, acc[i & 1]);
    }
    h = halves(add2(acc[0], acc[1]));
    const float m2 = warp_sum(h.x + h.y);
    if ((lane & 31) == 0) red[r & 1][lane >> 5] = make_float2(sum, m2);
    wait_for_next_row(stages);
    __syncthreads();
    fetch(stage == 0 ? stages - 1 : stage - 1);
    // M2 = sum_w M2_w + n_w (mean_w - mean)^2, a warp's values in each of 16 lanes.
    const float2 part = red[r & 1][who];
    const float mean = sum16(part.x) * inv_c;
    const float off = fmaf(part.x, inv_who, -mean);
    const float rstd = rsqrtf(sum16(fmaf(off * off, n_who, part.y)) * inv_c + op.eps);
    if constexpr (kRow) {
      if (scale.at) {
        scale.read<MT, P>(slot, w);
        add_offset<P>(w, op.scale_offset);
      }
      if (shift.at) shift.read<MT, P>(slot, b);
    }
#pragma unroll
    for (int i = 0; i < P / 2; ++i)
      z.q[i] = fma2(mul2(add2(z.q[i], pair(-mean, -mean)), pair(rstd, rstd)), w.q[i], b.q[i]);
    store_columns<T, P>((T*)op.h + row * c, c, z);
    if (lane == 0 && op.mean) {
      op.mean[row] = mean;
      op.rstd[row] = rstd;
    }
    x.advance();
    y.advance();
    scale.advance();
    shift.advance();
    gate.advance();
    stage = stage + 1 == stages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// The row arithmetic that both backward kernels share: n = (z - mean)*rstd, u = dh*w
// and a lane's sums before the reduction, the gradients after it.
template <int V, int P>
struct Sums {
  Vals<V> shift[P], scale[P], gate[P];  // column sums

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      shift[p].fill(0.f);
      scale[p].fill(0.f);
      gate[p].fill(0.f);
    }
  }
  __device__ __forceinline__ void first(int p, const Vals<V>& z, const Vals<V>& dh, const Vals<V>& w, uint64_t minus,
                                        uint64_t rstd, Vals<V>& n, Vals<V>& u, uint64_t& s0, uint64_t& s1) {
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i) {
      n.q[i] = mul2(add2(z.q[i], minus), rstd);
      u.q[i] = mul2(dh.q[i], w.q[i]);
      s0 = add2(s0, u.q[i]);
      s1 = fma2(u.q[i], n.q[i], s1);
      shift[p].q[i] = add2(shift[p].q[i], dh.q[i]);
      scale[p].q[i] = fma2(dh.q[i], n.q[i], scale[p].q[i]);
    }
  }
  // dgate += g*y, dy = g*gate
  __device__ __forceinline__ void branch(int p, const Vals<V>& g, const Vals<V>& y, Vals<V>& dy) {
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i) {
      gate[p].q[i] = fma2(g.q[i], y.q[i], gate[p].q[i]);
      dy.q[i] = mul2(g.q[i], dy.q[i]);
    }
  }
};
// rstd*(u - m0 - n*m1) + dz
template <int V>
__device__ __forceinline__ void second(const Vals<V>& n, const Vals<V>& u, uint64_t minus_m0, uint64_t minus_m1,
                                       uint64_t rstd, const Vals<V>& dz, Vals<V>& g) {
#pragma unroll
  for (int i = 0; i < Vals<V>::kPairs; ++i)
    g.q[i] = fma2(fma2(n.q[i], minus_m1, add2(u.q[i], minus_m0)), rstd, dz.q[i]);
}

template <typename MT, int V>
__device__ __forceinline__ void store_sums(const SprAdalnGrad& gr, const Groups& gp, int64_t unit, int c, int v,
                                           float* partial, const Vals<V>& shift, const Vals<V>& scale,
                                           const Vals<V>& gate) {
  if (gp.chunks == 1) {
    const int64_t at = unit * c + v * V;
    if (gr.dshift) store_row<MT, V>((MT*)gr.dshift + at, shift);
    if (gr.dscale) store_row<MT, V>((MT*)gr.dscale + at, scale);
    if (gr.dgate) store_row<MT, V>((MT*)gr.dgate + at, gate);
  } else {
    float* p = partial + unit * 3 * c + v * V;
    if (gr.dshift) store_row<float, V>(p, shift);
    if (gr.dscale) store_row<float, V>(p + c, scale);
    if (gr.dgate) store_row<float, V>(p + 2 * c, gate);
  }
}

// Any width: a CTA takes one run of a group, its teams every other row of it, and
// joins the teams' column sums at the end; with `own` each team takes a run by
// itself (groups of few rows, such as a vector for every token).  75,600 x 64 bf16 17 us
// (26% of bandwidth).  Launches of up to 1,024 threads leave a thread 64 registers, too few
// for its column sums and two operands from two vectors a thread on: the widest rows keep
// them in local memory (10,000 x 12,288 bf16 493 us, 23%; gated 1,909 us, 12%).
template <typename T, typename MT, int V, int P, bool kRes>
__global__ void __launch_bounds__(1024) adaln_backward_kernel(const SprAdaln op, const SprAdalnGrad gr,
                                                              const Groups gp, int team, int own, float* partial) {
  __shared__ ulonglong2 red[2][16];
  extern __shared__ float joined[];
  const int c = op.channels, nvec = c / V;
  const int lane = threadIdx.x % team, sub = threadIdx.x / team, teams = blockDim.x / team;
  const int64_t units = gp.count * gp.chunks;
  const int64_t unit = own ? (int64_t)blockIdx.x * teams + sub : blockIdx.x;
  const bool busy = unit < units;
  const int64_t g = busy ? unit / gp.chunks : 0, s = busy ? unit % gp.chunks : 0;
  const int64_t r0 = s * gp.chunk_rows, r1 = busy ? min(gp.rows, r0 + gp.chunk_rows) : r0;
  const int64_t step = own ? 1 : teams, base = own ? r0 : r0 + sub;
  // Every team runs as many rounds as the longest, so that shuffles and barriers meet.
  const int64_t rounds = own ? gp.chunk_rows : (r1 - r0 + teams - 1) / teams;
  const float inv_c = 1.f / c;
  const RowId gid = row_id(op, g * gp.group_step);
  if (threadIdx.x < 64) (&red[0][0].x)[threadIdx.x] = 0;
  if (team > 32) __syncthreads();
  Vals<V> n[P], u[P];
  Sums<V, P> st;
  st.clear();
  for (int64_t i = 0; i < rounds; ++i) {
    const int64_t r = base + i * step;
    const bool valid = r < r1;
    const int64_t row = g * gp.group_step + (valid ? r : r0) * gp.row_step;
    const RowId id = row_id(op, row);
    const uint64_t minus = both<V>(-op.mean[row]), rstd = both<V>(op.rstd[row]);
    uint64_t s0 = 0, s1 = 0;
    if (valid)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int v = lane + p * team;
        if (v >= nvec) continue;
        Vals<V> z, dh, w;
        load_row<T, V>((const T*)op.x + id.b * op.x_sb + id.t * op.x_st + v * V, z);
        load_row<T, V>((const T*)gr.dh + id.b * gr.dh_sb + id.t * gr.dh_st + v * V, dh);
        load_factor<MT, V>(op, gid, v, w);
        st.first(p, z, dh, w, minus, rstd, n[p], u[p], s0, s1);
      }
    const float2 a = halves(s0), b = halves(s1);
    uint64_t sums = team_sum2(pair(a.x + a.y, b.x + b.y), team);
    if (team > 32) sums = warps_sum2(sums, red[i & 1], team / 32);
    const float2 m = halves(sums);
    const uint64_t m0 = both<V>(-m.x * inv_c), m1 = both<V>(-m.y * inv_c);
    if (valid)
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int v = lane + p * team;
        if (v >= nvec) continue;
        Vals<V> dz, gx;
        if (kRes && gr.dz) load_row<T, V>((const T*)gr.dz + id.b * gr.dz_sb + id.t * gr.dz_st + v * V, dz);
        else dz.fill(0.f);
        second<V>(n[p], u[p], m0, m1, rstd, dz, gx);
        if constexpr (kRes) {
          Vals<V> y, dy;
          load_row<T, V>((const T*)op.y + id.b * op.y_sb + id.t * op.y_st + v * V, y);
          load_gate<MT, V>(op, gid, v, dy);
          st.branch(p, gx, y, dy);
          store_row<T, V>((T*)gr.dy + row * c + v * V, dy);
        }
        store_row<T, V>((T*)gr.dx + row * c + v * V, gx);
      }
  }
  if (!gr.dshift && !gr.dscale && !gr.dgate) return;
  if (!own && teams > 1) {
    // Several teams are at most a warp wide each: kCtaThreads*V*P columns among them.
    float* mine = joined + sub * 3 * c;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int v = lane + p * team;
      if (v < nvec)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 a = halves(st.shift[p].q[e / 2]), b = halves(st.scale[p].q[e / 2]),
                       d = halves(st.gate[p].q[e / 2]);
          mine[v * V + e] = e % 2 ? a.y : a.x;
          mine[c + v * V + e] = e % 2 ? b.y : b.x;
          mine[2 * c + v * V + e] = e % 2 ? d.y : d.x;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 3 * c; i += blockDim.x) {
      float v = 0.f;
      for (int q = 0; q < teams; ++q) v += joined[q * 3 * c + i];
      void* outs[3] = {gr.dshift, gr.dscale, gr.dgate};
      if (!outs[i / c]) continue;
      if (gp.chunks == 1) ((MT*)outs[i / c])[unit * c + i % c] = from_f32<MT>(v);
      else partial[unit * 3 * c + i] = v;
    }
    return;
  }
  if (busy)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int v = lane + p * team;
      if (v < nvec) store_sums<MT, V>(gr, gp, unit, c, v, partial, st.shift[p], st.scale[p], st.gate[p]);
    }
}

// Long groups of wide rows: CTAs that stay on their SM walk runs of rows with the
// vectors and their column sums in registers, P 16-byte vectors a thread.  Each
// thread copies its own vectors of the next kStages - 1 rounds into shared memory,
// so the copies need no barrier and stay in flight across the one that joins a
// round's sums.  A round is R rows, which share the latency of shuffles and barrier.
// kAgain: n and u are formed again after the barrier instead of held across it
// (512 threads have 128 registers each; held, they spill).  kRow: each row has vectors
// of its own; they are streamed as the rows are, and so are their gradients.
// 75,600 x 5120 bf16: 372 us (95%), gated with fp32 vectors 740 us (96%), both with the join;
// 40,000 x 1536 bf16 gated with vectors for every row 210 us (98%).
constexpr int kStatRows = 256;  // rows whose statistics are in shared memory at a time
template <typename T, typename MT, int P, bool kRes, bool kFull, bool kRow, bool kAgain, int R, int kThreads, int kStages>
__global__ void __launch_bounds__(kThreads, 1)
adaln_backward_stream_kernel(const SprAdaln op, const SprAdalnGrad gr, const Groups gp, float* partial) {
  constexpr int V = kVec<T>, kIn = kRes ? 4 : 2, e = sizeof(T);
  constexpr int kM = kRow ? row_pieces<T, MT> : 0, kAll = kIn + kM * (kRes ? 2 : 1);
  __shared__ uint64_t red[2][R][16];
  __shared__ float stats[2][kStatRows];
  extern __shared__ uint4 ring[];  // [stage][row][operand][P][thread]
  const int c = op.channels, nvec = c / V, team = blockDim.x, lane = threadIdx.x;
  const Run run(op, gp, blockIdx.x);
  auto mine = [&](int p) { return kFull || lane + p * team < nvec; };
  const float inv_c = 1.f / c;
  for (int i = lane; i < 32 * R; i += team) (&red[0][0][0])[i] = 0;
  Sums<V, kRow ? 1 : P> st;
  st.clear();
  constexpr int kHeld = kAgain ? 1 : P, kOwn = kRow ? 1 : P;
  Vals<V> n[R][kHeld], u[R][kHeld], w[kOwn], gate[kOwn];
#pragma unroll
  for (int p = 0; p < (kRow ? 0 : P); ++p)
    if (mine(p)) {
      load_factor<MT, V>(op, run.group, lane + p * team, w[p]);
      if constexpr (kRes) load_gate<MT, V>(op, run.group, lane + p * team, gate[p]);
    }
  const bool has_dz = kRes && gr.dz != nullptr;
  const char* in[4] = {run.at(op.x, op.x_sb, op.x_st, e), run.at(gr.dh, gr.dh_sb, gr.dh_st, e),
                       kRes ? run.at(op.y, op.y_sb, op.y_st, e) : nullptr,
                       has_dz ? run.at(gr.dz, gr.dz_sb, gr.dz_st, e) : nullptr};
  const bool along = run.step == 1;
  const int64_t step[4] = {(along ? op.x_st : op.x_sb) * e, (along ? gr.dh_st : gr.dh_sb) * e,
                           (along ? op.y_st : op.y_sb) * e, (along ? gr.dz_st : gr.dz_sb) * e};
  BackwardVectors<T, MT, P, kRow, kRes> vec(op, run);
  int fetched = 0;
  auto fetch = [&](int stage) {
#pragma unroll
    for (int q = 0; q < R; ++q)
      if (fetched++ < run.rows) {
        uint4* to = ring + (stage * R + q) * (kAll * P) * team + lane;
        if constexpr (kRow) vec.copy(to + kIn * P * team, team, [&](int p) { return mine(p); });
#pragma unroll
        for (int k = 0; k < kIn; ++k) {
          if (k == 3 && !has_dz) continue;
#pragma unroll
          for (int p = 0; p < P; ++p)
            if (mine(p)) copy16_async(to + (k * P + p) * team, in[k] + p * team * 16);
          in[k] += step[k];
        }
      }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  int stage = 0;
  char* dx = (char*)gr.dx + (run.row0 * c * e + lane * 16);
  char* dy = (char*)gr.dy + (run.row0 * c * e + lane * 16);
  const int64_t out_step = run.step * c * e;
  for (int r = 0, odd = 0; r < run.rows; r += R, odd ^= 1) {
    const int at = r % kStatRows;
    if (at == 0) {
      __syncthreads();  // the last readers of the statistics are done
      for (int i = lane; i < min(kStatRows, run.rows - r); i += team) {
        stats[0][i] = -op.mean[run.row0 + (r + i) * run.step];
        stats[1][i] = op.rstd[run.row0 + (r + i) * run.step];
      }
      __syncthreads();
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    const uint4* slot = ring + stage * R * (kAll * P) * team + lane;
    uint64_t sums[R];
#pragma unroll
    for (int q = 0; q < R; ++q) {
      uint64_t s0 = 0, s1 = 0;
      if (R == 1 || r + q < run.rows) {
        const uint64_t minus = both<V>(stats[0][at + q]), rs = both<V>(stats[1][at + q]);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          if (!mine(p)) continue;
          Vals<V> z, dh;
          unpack16<T>(slot[((q * kAll + 0) * P + p) * team], z.q);
          unpack16<T>(slot[((q * kAll + 1) * P + p) * team], dh.q);
          if constexpr (kRow) {
            vec.read(slot + (q * kAll + kIn) * P * team, team, p, 0, op.scale_offset, 1.f, w[0]);
            st.clear();  // a row's own: written below, not added up
          }
          st.first(kRow ? 0 : p, z, dh, w[kRow ? 0 : p], minus, rs, n[q][kAgain ? 0 : p], u[q][kAgain ? 0 : p], s0, s1);
          if constexpr (kRow) {
            const int64_t at_c = (run.row0 + r + q) * c + (lane + p * team) * V;
            if (gr.dshift) store_row<MT, V>((MT*)gr.dshift + at_c, st.shift[0]);
            if (gr.dscale) store_row<MT, V>((MT*)gr.dscale + at_c, st.scale[0]);
          }
        }
      }
      const float2 a = halves(s0), b = halves(s1);
      sums[q] = pair(a.x + a.y, b.x + b.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int q = 0; q < R; ++q) sums[q] = add2(sums[q], __shfl_xor_sync(0xffffffffu, sums[q], o));
    // The slots that this fetch fills were read in the round before.
    fetch(stage == 0 ? kStages - 1 : stage - 1);
    if ((lane & 31) == 0)
#pragma unroll
      for (int q = 0; q < R; ++q) red[odd][q][lane >> 5] = sums[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < R; ++q) sums[q] = red[odd][q][lane & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
      for (int q = 0; q < R; ++q) sums[q] = add2(sums[q], __shfl_xor_sync(0xffffffffu, sums[q], o, 16));
#pragma unroll
    for (int q = 0; q < R; ++q) {
      if (R > 1 && r + q >= run.rows) continue;
      const float2 m = halves(sums[q]);
      const uint64_t m0 = both<V>(-m.x * inv_c), m1 = both<V>(-m.y * inv_c), rs = both<V>(stats[1][at + q]);
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (!mine(p)) continue;
        Vals<V> gx, dz;
        if (has_dz) unpack16<T>(slot[((q * kAll + 3) * P + p) * team], dz.q);
        else dz.fill(0.f);
        if constexpr (kAgain) {
          Vals<V> z, dh;
          unpack16<T>(slot[((q * kAll + 0) * P + p) * team], z.q);
          unpack16<T>(slot[((q * kAll + 1) * P + p) * team], dh.q);
          const uint64_t minus = both<V>(stats[0][at + q]);
          if constexpr (kRow) vec.read(slot + (q * kAll + kIn) * P * team, team, p, 0, op.scale_offset, 1.f, w[0]);
#pragma unroll
          for (int i = 0; i < V / 2; ++i) {
            n[q][0].q[i] = mul2(add2(z.q[i], minus), rs);
            u[q][0].q[i] = mul2(dh.q[i], w[kRow ? 0 : p].q[i]);
          }
        }
        second<V>(n[q][kAgain ? 0 : p], u[q][kAgain ? 0 : p], m0, m1, rs, dz, gx);
        if constexpr (kRes) {
          Vals<V> y, gy = gate[kRow ? 0 : p];
          unpack16<T>(slot[((q * kAll + 2) * P + p) * team], y.q);
          if constexpr (kRow) {
            vec.read(slot + (q * kAll + kIn) * P * team, team, p, 1, 0.f, 1.f, gy);
            st.gate[0].fill(0.f);
          }
          st.branch(kRow ? 0 : p, gx, y, gy);
          if constexpr (kRow)
            if (gr.dgate) store_row<MT, V>((MT*)gr.dgate + (run.row0 + r + q) * c + (lane + p * team) * V, st.gate[0]);
          *reinterpret_cast<uint4*>(dy + p * team * 16) = pack16<T>(gy.q);
        }
        *reinterpret_cast<uint4*>(dx + p * team * 16) = pack16<T>(gx.q);
      }
      dx += out_step;
      if constexpr (kRes) dy += out_step;
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if constexpr (!kRow)
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int v = lane + p * team;
      if (mine(p)) store_sums<MT, V>(gr, gp, blockIdx.x, c, v, partial, st.shift[p], st.scale[p], st.gate[p]);
    }
}

// The backward pass of rows that 16-byte vectors do not fit, as the forward pass takes
// them: 30,000 x 1537 bf16 84 us (50% of bandwidth), gated 171 us (49%), 30,000 x 1003 fp32
// gated 142 us (77%).
template <typename T, typename MT, int P, bool kRes, bool kRow, int kThreads>
__global__ void __launch_bounds__(kThreads, 1)
adaln_backward_any_kernel(const SprAdaln op, const SprAdalnGrad gr, const Groups gp, int stages, int slot_bytes,
                          float* partial) {
  __shared__ uint64_t red[2][16];
  extern __shared__ uint4 ring[];
  const int c = op.channels, team = blockDim.x, lane = threadIdx.x, e = sizeof(T), me = sizeof(MT);
  const Run run(op, gp, blockIdx.x);
  const int row_place = window_bytes(team * P, e), vec_place = window_bytes(team * P, me);
  Window x(run, op.x, op.x_sb, op.x_st, e, c, 0), dh(run, gr.dh, gr.dh_sb, gr.dh_st, e, c, row_place), y, dz, scale,
      gate;
  if constexpr (kRes) {
    y = Window(run, op.y, op.y_sb, op.y_st, e, c, 2 * row_place);
    dz = Window(run, gr.dz, gr.dz_sb, gr.dz_st, e, c, 3 * row_place);
  }
  if constexpr (kRow) {
    constexpr int rows = kRes ? 4 : 2;
    scale = Window(run, op.scale, op.scale_sb, op.scale_st, me, c, rows * row_place);
    if constexpr (kRes) gate = Window(run, op.gate, op.gate_sb, op.gate_st, me, c, rows * row_place + vec_place);
  }
  const float inv_c = 1.f / c;
  if (lane < 32) (&red[0][0])[lane] = 0;
  int fetched = 0;
  auto fetch = [&](int stage) {
    if (fetched++ < run.rows) {
      char* slot = reinterpret_cast<char*>(ring) + stage * slot_bytes;
      x.copy(slot);
      dh.copy(slot);
      if constexpr (kRes) {
        y.copy(slot);
        dz.copy(slot);
      }
      if constexpr (kRow) {
        scale.copy(slot);
        if constexpr (kRes) gate.copy(slot);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  clear_ring(ring, stages * slot_bytes);
  for (int i = 0; i < stages - 1; ++i) fetch(i);
  Vals<P> w, gv;
  w.fill(1.f);
  gv.fill(1.f);
  if constexpr (!kRow) {
    const RowId& id = run.group;
    if (op.scale) {
      load_columns<MT, P>((const MT*)op.scale + id.b * op.scale_sb + id.t * op.scale_st, c, w);
      add_offset<P>(w, op.scale_offset);
    }
    if (kRes && op.gate) load_columns<MT, P>((const MT*)op.gate + id.b * op.gate_sb + id.t * op.gate_st, c, gv);
  }
  Sums<P, 1> st;
  st.clear();
  float next_mean = op.mean[run.row0], next_rstd = op.rstd[run.row0];
  if (stages == 4) asm volatile("cp.async.wait_group 2;" ::: "memory");
  else asm volatile("cp.async.wait_group 1;" ::: "memory");
  __syncthreads();
  int stage = 0;
  for (int r = 0; r < run.rows; ++r) {
    const char* slot = reinterpret_cast<const char*>(ring) + stage * slot_bytes;
    const int64_t row = run.row0 + r * run.step;
    const uint64_t minus = pair(-next_mean, -next_mean), rs = pair(next_rstd, next_rstd);
    if (r + 1 < run.rows) {
      next_mean = op.mean[row + run.step];
      next_rstd = op.rstd[row + run.step];
    }
    Vals<P> z, d, n, u;
    x.read<T, P>(slot, z);
    dh.read<T, P>(slot, d);
    if (kRow && scale.at) {
      scale.read<MT, P>(slot, w);
      add_offset<P>(w, op.scale_offset);
    }
    if constexpr (kRow) st.clear();  // a row's own: written below, not added up
    uint64_t s0 = 0, s1 = 0;
    st.first(0, z, d, w, minus, rs, n, u, s0, s1);
    if constexpr (kRow) {
      if (gr.dshift) store_columns<MT, P>((MT*)gr.dshift + row * c, c, st.shift[0]);
      if (gr.dscale) store_columns<MT, P>((MT*)gr.dscale + row * c, c, st.scale[0]);
    }
    const float2 a = halves(s0), b = halves(s1);
    uint64_t sums = team_sum2(pair(a.x + a.y, b.x + b.y), 32);
    if ((lane & 31) == 0) red[r & 1][lane >> 5] = sums;
    wait_for_next_row(stages);
    __syncthreads();
    fetch(stage == 0 ? stages - 1 : stage - 1);
    sums = red[r & 1][lane & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sums = add2(sums, __shfl_xor_sync(0xffffffffu, sums, o, 16));
    const float2 m = halves(sums);
    Vals<P> g, dzv;
    dzv.fill(0.f);
    if (kRes && dz.at) dz.read<T, P>(slot, dzv);
    second<P>(n, u, pair(-m.x * inv_c, -m.x * inv_c), pair(-m.y * inv_c, -m.y * inv_c), rs, dzv, g);
    if constexpr (kRes) {
      Vals<P> yv, dy = gv;
      y.read<T, P>(slot, yv);
      if (kRow && gate.at) gate.read<MT, P>(slot, dy);
      st.branch(0, g, yv, dy);
      if (kRow && gr.dgate) store_columns<MT, P>((MT*)gr.dgate + row * c, c, st.gate[0]);
      store_columns<T, P>((T*)gr.dy + row * c, c, dy);
    }
    store_columns<T, P>((T*)gr.dx + row * c, c, g);
    x.advance();
    dh.advance();
    y.advance();
    dz.advance();
    scale.advance();
    gate.advance();
    stage = stage + 1 == stages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if constexpr (!kRow) {
    if (gp.chunks == 1) {
      const int64_t at = (int64_t)blockIdx.x * c;
      if (gr.dshift) store_columns<MT, P>((MT*)gr.dshift + at, c, st.shift[0]);
      if (gr.dscale) store_columns<MT, P>((MT*)gr.dscale + at, c, st.scale[0]);
      if (gr.dgate) store_columns<MT, P>((MT*)gr.dgate + at, c, st.gate[0]);
    } else {
      float* p = partial + (int64_t)blockIdx.x * 3 * c;
      if (gr.dshift) store_columns<float, P>(p, c, st.shift[0]);
      if (gr.dscale) store_columns<float, P>(p + c, c, st.scale[0]);
      if (gr.dgate) store_columns<float, P>(p + 2 * c, c, st.gate[0]);
    }
  }
}

// Joins the runs' column sums in their order: 32 columns by 32 threads each, each thread
// every 32nd run.  The sums mostly still lie in L2: 6 to 27 MB in 8 to 13 us.
template <typename MT>
__global__ void __launch_bounds__(1024) adaln_join_kernel(const SprAdalnGrad gr, int c, int chunks,
                                                          const float* partial) {
  __shared__ float part[32][33];
  const int64_t g = blockIdx.x;
  const int what = blockIdx.z, col = blockIdx.y * 32 + threadIdx.x;
  MT* out = (MT*)(what == 0 ? gr.dshift : what == 1 ? gr.dscale : gr.dgate);
  if (!out) return;
  const float* p = partial + (g * chunks * 3 + what) * c + col;
  float v = 0.f;
  if (col < c)
    for (int s = threadIdx.y; s < chunks; s += 32) v += p[(int64_t)s * 3 * c];
  part[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  v = part[threadIdx.x][threadIdx.y];  // lane = the thread's share, warp = the column
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  const int mine = blockIdx.y * 32 + threadIdx.y;
  if (threadIdx.x == 0 && mine < c) out[g * c + mine] = from_f32<MT>(v);
}

int sm_count() {
  static thread_local int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!sms[dev] && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  return sms[dev];
}

// Threads of a CTA that takes whole rows: whole warps.
int cta_for(int vectors, int per) { return ((vectors + per - 1) / per + 31) / 32 * 32; }

// Threads a row: a power of two of lanes up to a warp, whole warps above.
int team_for(int vectors) {
  if (vectors > 32) return (vectors + 31) / 32 * 32;
  int t = 1;
  while (t < vectors) t *= 2;
  return t;
}

bool rows_fit(int64_t batch, int64_t tokens) { return tokens == 0 || batch <= 0x7fffffffLL / tokens; }

int check_adaln(const SprAdaln* op) {
  if (!op) return fail(SPR_ERR_ARG, "adaln: no operands");
  if (op->batch < 0 || op->tokens < 0 || op->channels < 1 || op->channels > kMaxChannels)
    return fail(SPR_ERR_SHAPE, "adaln: batch=%lld tokens=%lld channels=%d (channels must be 1..%d)",
                (long long)op->batch, (long long)op->tokens, op->channels, kMaxChannels);
  if (!rows_fit(op->batch, op->tokens)) return fail(SPR_ERR_SHAPE, "adaln: batch*tokens too large");
  if (op->dtype != SPR_F32 && op->dtype != SPR_BF16 && op->dtype != SPR_F16)
    return fail(SPR_ERR_DTYPE, "adaln: unsupported dtype %d", op->dtype);
  if (op->mod_dtype != op->dtype && op->mod_dtype != SPR_F32)
    return fail(SPR_ERR_DTYPE, "adaln: shift/scale/gate dtype %d must be the element type %d or fp32", op->mod_dtype,
                op->dtype);
  if (op->gate && !op->y && op->batch * op->tokens) return fail(SPR_ERR_ARG, "adaln: a gate without a branch");
  return SPR_OK;
}

// Whether every operand begins on one of its elements, and the statistics come together.
int check_pointers(const SprAdaln* op, const SprAdalnGrad* g) {
  const size_t e = dtype_bytes(op->dtype), m = dtype_bytes(op->mod_dtype);
  bool ok = aligned(op->mean, 4) && aligned(op->rstd, 4);
  for (const void* p : {op->x, op->y, (const void*)op->z, (const void*)op->h}) ok &= aligned(p, e);
  for (const void* p : {op->shift, op->scale, op->gate}) ok &= aligned(p, m);
  if (g) {
    for (const void* p : {g->dh, g->dz, (const void*)g->dx, (const void*)g->dy}) ok &= aligned(p, e);
    for (const void* p : {g->dshift, g->dscale, g->dgate}) ok &= aligned(p, m);
  }
  if (!ok) return fail(SPR_ERR_ALIGN, "adaln: an operand is not aligned to its elements");
  if (!op->mean != !op->rstd) return fail(SPR_ERR_ARG, "adaln: mean without rstd, or rstd without mean");
  return SPR_OK;
}

// Whether 16-byte vectors fit the width, a pointer and its strides.
bool vectors_fit(const void* p, int64_t sb, int64_t st, int dtype) {
  const int e = dtype_bytes(dtype);
  return !p || (aligned(p, 16) && sb * e % 16 == 0 && st * e % 16 == 0);
}
bool vectors_fit(const SprAdaln* op) {
  return op->channels % (16 / dtype_bytes(op->dtype)) == 0 && vectors_fit(op->x, op->x_sb, op->x_st, op->dtype) &&
         vectors_fit(op->y, op->y_sb, op->y_st, op->dtype) &&
         vectors_fit(op->shift, op->shift_sb, op->shift_st, op->mod_dtype) &&
         vectors_fit(op->scale, op->scale_sb, op->scale_st, op->mod_dtype) &&
         vectors_fit(op->gate, op->gate_sb, op->gate_st, op->mod_dtype) && vectors_fit(op->z, 0, 0, op->dtype) &&
         vectors_fit(op->h, 0, 0, op->dtype);
}
bool vectors_fit(const SprAdaln* op, const SprAdalnGrad* g) {
  return vectors_fit(op) && vectors_fit(g->dh, g->dh_sb, g->dh_st, op->dtype) &&
         vectors_fit(g->dz, g->dz_sb, g->dz_st, op->dtype) && vectors_fit(g->dx, 0, 0, op->dtype) &&
         vectors_fit(g->dy, 0, 0, op->dtype) && vectors_fit(g->dshift, 0, 0, op->mod_dtype) &&
         vectors_fit(g->dscale, 0, 0, op->mod_dtype) && vectors_fit(g->dgate, 0, 0, op->mod_dtype);
}

// Calls f(T{}, MT{}) for the operands' types.
template <typename F>
int by_type(const SprAdaln* op, F f) {
  if (op->dtype == SPR_F32) return f(float{}, float{});
  if (op->dtype == SPR_BF16)
    return op->mod_dtype == SPR_F32 ? f(__nv_bfloat16{}, float{}) : f(__nv_bfloat16{}, __nv_bfloat16{});
  return op->mod_dtype == SPR_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
}

// Rows without gaps between the samples are one sample of batch*tokens rows.
bool dense_batch(int64_t sb, int64_t st, int64_t tokens) { return sb == tokens * st; }
void merge_batch(SprAdaln& op, SprAdalnGrad* g) {
  if (op.batch == 1) return;
  for (auto [p, sb, st] : {std::tuple(op.shift, op.shift_sb, op.shift_st), std::tuple(op.scale, op.scale_sb, op.scale_st),
                           std::tuple(op.gate, op.gate_sb, op.gate_st)})
    if (p && !dense_batch(sb, st, op.tokens)) return;  // one vector (0, 0), or one for each row
  if (!dense_batch(op.x_sb, op.x_st, op.tokens) || (op.y && !dense_batch(op.y_sb, op.y_st, op.tokens))) return;
  if (g && (g->mod_batch != g->mod_tokens || !dense_batch(g->dh_sb, g->dh_st, op.tokens) ||
            (g->dz && !dense_batch(g->dz_sb, g->dz_st, op.tokens))))
    return;
  op.tokens *= op.batch;
  op.batch = 1;
  if (g) g->mod_batch = 0;
}

template <int N>
struct Int {
  static constexpr int value = N;
};

// Calls f(Int<V>{}, Int<P>{}) for V elements a vector and P vectors a thread.
template <typename T, typename F>
int by_shape(bool vec, int per, F f) {
  if (vec) {
    if (per <= 1) return f(Int<kVec<T>>{}, Int<1>{});
    if (per <= 2) return f(Int<kVec<T>>{}, Int<2>{});
    return f(Int<kVec<T>>{}, Int<4>{});
  }
  if (per <= 1) return f(Int<1>{}, Int<1>{});
  if (per <= 4) return f(Int<1>{}, Int<4>{});
  return f(Int<1>{}, Int<16>{});
}

constexpr int kAnySmem = 200 * 1024;
constexpr int kCtaThreads = 256;  // of a CTA whose teams are at most a warp

// Whether a run's rows are equally spaced in every operand: within one sample, or
// the same token of every sample, or all rows of operands without gaps.  One vector for
// the rows of several samples with gaps between them is the form that is not, and takes
// the kernels for any rows (2 x 37,800 x 5120 bf16 forward 367 us, with a vector a sample
// 248; backward 1,104 and 381).
bool even_rows(const Groups& g, int64_t batch) { return batch == 1 || g.row_step != 1 || g.count % batch == 0; }

Groups make_groups(int64_t batch, int64_t tokens, int mod_batch, int mod_tokens) {
  Groups g{};
  g.count = (mod_batch ? batch : 1) * (mod_tokens ? tokens : 1);
  g.rows = (mod_batch ? 1 : batch) * (mod_tokens ? 1 : tokens);
  g.group_step = mod_tokens ? 1 : tokens;
  g.row_step = mod_tokens ? tokens : 1;
  return g;
}

// Runs a group is cut into: enough for `ctas` CTAs, of at least `least` rows each.
void cut_groups(Groups& g, int64_t ctas, int64_t least) {
  const int64_t want = std::max<int64_t>(1, std::min(ctas / g.count, g.rows / least));
  g.chunk_rows = (g.rows + want - 1) / want;
  g.chunks = (int)((g.rows + g.chunk_rows - 1) / g.chunk_rows);
}

template <typename T>
int forward_per_thread(bool vec, int nvec) {
  if (nvec <= 32) return 1;
  if (vec) return nvec <= 64 ? 1 : nvec <= 128 ? 2 : 4;
  return nvec <= 4096 ? 4 : 16;
}

// CTAs of a kernel that an SM of the current device holds, asked once for each device and
// number of warps (a kernel's shared memory follows from them); an answer that failed is
// not kept.
template <auto kern>
int resident(int threads, int smem) {
  constexpr int kDevices = 16;
  static std::atomic<int> known[kDevices][17] = {};
  int dev = -1, got = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  std::atomic<int>* kept = dev < kDevices && threads <= 512 ? &known[dev][threads / 32] : nullptr;
  if (kept && (got = kept->load(std::memory_order_relaxed)) != 0) return got;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&got, kern, threads, smem) != cudaSuccess) return 1;
  got = std::max(1, got);
  if (kept) kept->store(got, std::memory_order_relaxed);
  return got;
}

// How a streaming launch cuts its groups: as many runs as fit on the GPU at once, and
// up to `most_waves` times that while a run still reads `least` bytes.  More waves
// leave uneven SMs less to wait for at the end, each run costs its start (and in
// the backward pass a set of column sums).  Of measured bandwidth, 1 / 6 waves:
// 75,600 x 5120 bf16 forward 92% / 98%, 60,000 x 1024 fp16 forward 86% / 80%,
// 75,600 x 5120 bf16 gated backward 89% / 98%, ungated 101% / 88%.
void cut_stream(Groups& g, int64_t at_once, int64_t row_bytes, int64_t most_waves, int64_t least, int64_t most) {
  const int64_t waves = g.count * g.rows * row_bytes / (at_once * least);
  cut_groups(g, std::min(most, at_once * std::max<int64_t>(1, std::min(most_waves, waves))), 4);
}

// Stages of a ring whose stage takes `bytes` at the kernel's most threads; 0: none fits.
constexpr int ring_stages(int bytes) {
  return 4 * bytes <= 200 * 1024 ? 4 : 3 * bytes <= 200 * 1024 ? 3 : 2 * bytes <= 200 * 1024 ? 2 : 0;
}

template <typename T, typename MT, bool kRes, int P, bool kFull, bool kRow, int kThreads, int kMin>
int launch_forward_stream(const SprAdaln* op, Groups g, cudaStream_t st) {
  static_assert(kThreads <= 512, "sums of at most 16 warps are joined");
  constexpr int kIn = (kRes ? 2 : 1) + (kRow ? row_pieces<T, MT> * (kRes ? 3 : 2) : 0);
  constexpr int kStages = ring_stages(kIn * P * kThreads * 16);
  static_assert(kStages >= 2, "no ring fits");
  constexpr auto kern = adaln_forward_stream_kernel<T, MT, P, kRes, kFull, kRow, kThreads, kMin, kStages>;
  const int team = cta_for(op->channels / kVec<T>, P);
  const int smem = kStages * kIn * P * team * 16;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kStages * kIn * P * kThreads * 16) !=
      cudaSuccess)
    return check_launch("adaln forward");
  cut_stream(g, (int64_t)sm_count() * resident<kern>(team, smem), (int64_t)kIn * op->channels * sizeof(T), 6, 65536,
             INT64_MAX);
  kern<<<(unsigned)(g.count * g.chunks), team, smem, st>>>(*op, g);
  return check_launch("adaln forward");
}

// Slots of a row's operands that a CTA holds: 4, or 3, or 0 where they do not fit.
constexpr int any_stages(int slot_bytes) { return 4 * slot_bytes <= kAnySmem ? 4 : 3 * slot_bytes <= kAnySmem ? 3 : 0; }
template <typename T, typename MT, bool kRes, bool kRow, bool kBackward>
constexpr int any_slot(int columns) {
  const int rows = kBackward ? (kRes ? 4 : 2) : kRes ? 2 : 1;
  const int vecs = kRow ? (kBackward ? (kRes ? 2 : 1) : kRes ? 3 : 2) : 0;
  return rows * window_bytes(columns, sizeof(T)) + vecs * window_bytes(columns, sizeof(MT));
}
// Columns a thread: 16, so that a row's fixed instructions serve more columns (30,000 x 1537
// bf16 forward 66 us, with 8 96 us; gated 117 and 126; only with vectors for every row 8
// are a little faster, 72 against 77 us at 10,000 rows), and 8 where one warp of those holds
// the row (75,600 x 131 bf16 gated 37 us, with 16 54 us).
constexpr int any_per(int channels) { return channels <= 256 ? 8 : 16; }
// Whether slots of the narrowest rows that need more than 256 threads fit.
template <typename T, typename MT, bool kRes, bool kRow, bool kBackward>
constexpr bool any_wide = any_stages(any_slot<T, MT, kRes, kRow, kBackward>(16 * 288)) > 0;
// From 64 columns on a CTA of one warp a row is faster than several rows to a warp (75,600 x
// 65 bf16: forward 26 and 33 us, backward 38 and 54 us; x 193: 27 and 79, 42 and 357 us).
template <typename T, typename MT, bool kRes, bool kRow, bool kBackward>
bool any_fits(int channels) {
  const int per = any_per(channels), team = cta_for(channels, per);
  return channels >= 64 && team <= 512 && any_stages(any_slot<T, MT, kRes, kRow, kBackward>(team * per)) > 0;
}

template <typename T, typename MT, bool kRes, bool kRow, int P, int kThreads>
int launch_forward_any(const SprAdaln* op, Groups g, cudaStream_t st) {
  constexpr auto kern = adaln_forward_any_kernel<T, MT, P, kRes, kRow, kThreads>;
  const int team = cta_for(op->channels, P), slot = any_slot<T, MT, kRes, kRow, false>(team * P);
  const int stages = any_stages(slot), smem = stages * slot;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kAnySmem) != cudaSuccess)
    return check_launch("adaln forward");
  cut_stream(g, (int64_t)sm_count() * resident<kern>(team, smem), slot, 6, 65536, INT64_MAX);
  kern<<<(unsigned)(g.count * g.chunks), team, smem, st>>>(*op, g, stages, slot);
  return check_launch("adaln forward");
}
template <typename T, typename MT, bool kRes, bool kRow>
int launch_forward_any(const SprAdaln* op, const Groups& g, cudaStream_t st) {
  if (any_per(op->channels) == 8) return launch_forward_any<T, MT, kRes, kRow, 8, 32>(op, g, st);
  if constexpr (any_wide<T, MT, kRes, kRow, false>)
    if (op->channels > 16 * 256) return launch_forward_any<T, MT, kRes, kRow, 16, 512>(op, g, st);
  return launch_forward_any<T, MT, kRes, kRow, 16, 256>(op, g, st);
}

template <typename MT>
int join(const SprAdaln* op, const SprAdalnGrad* gr, const Groups& g, const float* partial, cudaStream_t st);
int64_t most_runs(int channels);

template <typename T, typename MT, bool kRes, bool kRow, int P, int kThreads>
int launch_backward_any(const SprAdaln* op, const SprAdalnGrad* gr, Groups g, float* partial, cudaStream_t st) {
  constexpr auto kern = adaln_backward_any_kernel<T, MT, P, kRes, kRow, kThreads>;
  const int team = cta_for(op->channels, P), slot = any_slot<T, MT, kRes, kRow, true>(team * P);
  const int stages = any_stages(slot), smem = stages * slot;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kAnySmem) != cudaSuccess)
    return check_launch("adaln backward");
  cut_stream(g, (int64_t)sm_count() * resident<kern>(team, smem), slot, kRow || kRes ? 6 : 1, kRow ? 65536 : 3 << 19,
             kRow ? INT64_MAX : most_runs(op->channels));
  kern<<<(unsigned)(g.count * g.chunks), team, smem, st>>>(*op, *gr, g, stages, slot, partial);
  if constexpr (kRow) return check_launch("adaln backward");
  return join<MT>(op, gr, g, partial, st);
}
template <typename T, typename MT, bool kRes, bool kRow>
int launch_backward_any(const SprAdaln* op, const SprAdalnGrad* gr, const Groups& g, float* partial, cudaStream_t st) {
  if (any_per(op->channels) == 8) return launch_backward_any<T, MT, kRes, kRow, 8, 32>(op, gr, g, partial, st);
  if constexpr (any_wide<T, MT, kRes, kRow, true>)
    if (op->channels > 16 * 256) return launch_backward_any<T, MT, kRes, kRow, 16, 512>(op, gr, g, partial, st);
  return launch_backward_any<T, MT, kRes, kRow, 16, 256>(op, gr, g, partial, st);
}

// Whether P/2 vectors a thread leave fewer idle places in a CTA of at most 512.
bool half_fits_better(int nvec, int P) {
  const int half = cta_for(nvec, P / 2);
  return half <= 512 && half * (P / 2) < cta_for(nvec, P) * P;
}

template <typename T, typename MT, bool kRes>
int launch_forward(const SprAdaln* op, cudaStream_t st) {
  const bool vec = vectors_fit(op);
  const int nvec = op->channels / (vec ? kVec<T> : 1);
  auto kept = [&](int64_t scale, int64_t shift, int64_t gate) { return scale || shift || gate; };
  const Groups g = make_groups(op->batch, op->tokens, kept(op->scale_sb, op->shift_sb, op->gate_sb),
                               kept(op->scale_st, op->shift_st, op->gate_st));
  // Vectors for every token: 8 values a thread, so that a stage of them and the rows is
  // small enough for several CTAs an SM (of measured bandwidth, 40,000 gated rows of 1536
  // bf16: 95%, with a CTA a row 69%).  Wider rows keep a CTA a row: one CTA an SM with two
  // or three stages is slower (20,000 x 5120 gated, fp32 vectors: 67%, with a CTA a row 89%).
  if (vec && nvec > 32 && kept(op->scale_st, op->shift_st, op->gate_st) && op->tokens >= 8) {
    constexpr int Q = 8 / kVec<T>;
    const Groups rows = make_groups(op->batch, op->tokens, 1, 0);  // the samples' rows, one after the other
    if (nvec <= 512 * Q) {
      if (nvec % (32 * Q) == 0) return launch_forward_stream<T, MT, kRes, Q, true, true, 512, 1>(op, rows, st);
      return launch_forward_stream<T, MT, kRes, Q, false, true, 512, 1>(op, rows, st);
    }
  }
  constexpr int P = 16 / kVec<T>;  // 16 values a thread, or 8 where that leaves fewer threads idle
  if (vec && nvec > 32 && nvec <= 512 * P && g.rows >= 8 && even_rows(g, op->batch)) {
    // 16-bit rows of 4,096 channels and more that are whole warps of 32 values a thread take
    // those: fewer warps pay a row's fixed instructions, which bound the pass at the clocks
    // of a sustained load.  387 M elements of bf16, us with 16 and 32 values a thread: 1024
    // channels 246 and 254, 2048 255 and 253, 4096 277 and 256, 5120 268 and 248, 6144 319
    // and 254, 7168 305 and 254, 8192 303 and 251.  An fp32 row has twice the bytes for its
    // fixed instructions: 193 M elements, 4096 channels 254 and 265, 6144 257 and 271, 8192
    // 272 and 277.  With a branch the vectors leave no room for 32 values (75,600 x 5120 bf16:
    // 490 and 513).  Few rows are bound by the time of one, which more threads shorten: up to
    // six rows for each CTA of the 16-value form that an SM holds (two, above 5,120 channels
    // one).  600 rows of 5120 6.4 and 7.0, 1,200 7.5 and 8.0, 2,400 10.9 and 10.4; 740 rows of
    // 6144 6.3 and 7.3, 900 7.6 and 7.3, 2,400 18.0 and 12.4.
    if constexpr (!kRes && sizeof(T) == 2) {
      const bool wide = nvec > 320 * P;
      if (nvec % (64 * P) == 0 && nvec >= 256 * P && g.count * g.rows >= (wide ? 6 : 12) * (int64_t)sm_count())
        return wide ? launch_forward_stream<T, MT, false, 2 * P, true, false, 256, 2>(op, g, st)
                    : launch_forward_stream<T, MT, false, 2 * P, true, false, 160, 3>(op, g, st);
    }
    if (nvec % (32 * P) == 0)
      return nvec <= 320 * P ? launch_forward_stream<T, MT, kRes, P, true, false, 320, 2>(op, g, st)
                             : launch_forward_stream<T, MT, kRes, P, true, false, 512, 1>(op, g, st);
    if (half_fits_better(nvec, P)) return launch_forward_stream<T, MT, kRes, P / 2, false, false, 512, 1>(op, g, st);
    return launch_forward_stream<T, MT, kRes, P, false, false, 512, 1>(op, g, st);
  }
  if (!vec) {
    const bool own = kept(op->scale_st, op->shift_st, op->gate_st);
    if (own && op->tokens >= 8 && any_fits<T, MT, kRes, true, false>(op->channels))
      return launch_forward_any<T, MT, kRes, true>(op, make_groups(op->batch, op->tokens, 1, 0), st);
    if (!own && g.rows >= 8 && even_rows(g, op->batch) && any_fits<T, MT, kRes, false, false>(op->channels))
      return launch_forward_any<T, MT, kRes, false>(op, g, st);
  }
  return by_shape<T>(vec, forward_per_thread<T>(vec, nvec), [&](auto v, auto p) {
    constexpr int V = decltype(v)::value, P = decltype(p)::value;
    const int team = team_for((nvec + P - 1) / P);
    const int threads = team > 32 ? team : kCtaThreads;
    const int64_t rows = op->batch * op->tokens, teams = threads / team;
    adaln_forward_kernel<T, MT, V, P, kRes><<<(unsigned)((rows + teams - 1) / teams), threads, 0, st>>>(*op, team);
    return check_launch("adaln forward");
  });
}

// Runs of a backward launch, all groups together: sixteen an SM, and no more than
// 48 MB of column sums.  The workspace is sized for that many.
int64_t most_runs(int channels) {
  const int64_t sms = sm_count();
  return std::min(16 * sms, std::max(sms, (int64_t)(1 << 22) / channels));
}

template <typename MT>
int join(const SprAdaln* op, const SprAdalnGrad* gr, const Groups& g, const float* partial, cudaStream_t st) {
  if (g.chunks > 1 && (gr->dshift || gr->dscale || gr->dgate))
    adaln_join_kernel<MT><<<dim3((unsigned)g.count, (op->channels + 31) / 32, gr->dgate ? 3 : 2), dim3(32, 32), 0, st>>>(
        *gr, op->channels, g.chunks, partial);
  return check_launch("adaln backward");
}

template <typename T, typename MT, bool kRes, int P, bool kFull, bool kRow, bool kAgain, int R, int kThreads>
int launch_backward_stream(const SprAdaln* op, const SprAdalnGrad* gr, Groups g, float* partial, cudaStream_t st) {
  static_assert(kThreads <= 512, "sums of at most 16 warps are joined");
  constexpr int kIn = (kRes ? 4 : 2) + (kRow ? row_pieces<T, MT> * (kRes ? 2 : 1) : 0);
  constexpr int kStages = std::min(kRes ? 4 : 3, ring_stages(R * kIn * P * kThreads * 16));
  static_assert(kStages >= 2, "no ring fits");
  constexpr auto kern = adaln_backward_stream_kernel<T, MT, P, kRes, kFull, kRow, kAgain, R, kThreads, kStages>;
  const int team = cta_for(op->channels / kVec<T>, P);
  const int smem = kStages * R * kIn * P * team * 16;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kStages * R * kIn * P * kThreads * 16) !=
      cudaSuccess)
    return check_launch("adaln backward");
  cut_stream(g, (int64_t)sm_count() * resident<kern>(team, smem), (int64_t)kIn * op->channels * sizeof(T),
             kRow || kRes ? 6 : 1, kRow ? 65536 : 3 << 19, kRow ? INT64_MAX : most_runs(op->channels));
  kern<<<(unsigned)(g.count * g.chunks), team, smem, st>>>(*op, *gr, g, partial);
  if constexpr (kRow) return check_launch("adaln backward");
  return join<MT>(op, gr, g, partial, st);
}

template <typename T, typename MT, bool kRes>
int launch_backward(const SprAdaln* op, const SprAdalnGrad* gr, float* partial, cudaStream_t st) {
  const bool vec = vectors_fit(op, gr);
  const int nvec = op->channels / (vec ? kVec<T> : 1);
  Groups g = make_groups(op->batch, op->tokens, gr->mod_batch, gr->mod_tokens);
  if (vec && nvec > 32 && gr->mod_tokens && op->tokens >= 8 && (gr->mod_batch || op->batch == 1)) {
    constexpr int Q = 8 / kVec<T>;
    const Groups rows = make_groups(op->batch, op->tokens, 1, 0);
    if (nvec <= 512 * Q) {
      if (nvec % (32 * Q) == 0)
        return launch_backward_stream<T, MT, kRes, Q, true, true, false, 1, 512>(op, gr, rows, partial, st);
      return launch_backward_stream<T, MT, kRes, Q, false, true, false, 1, 512>(op, gr, rows, partial, st);
    }
    if constexpr (!kRes || sizeof(T) == 2)  // six fp32 operands of that width leave no room for two stages
      if (nvec <= 640 * Q)
        return launch_backward_stream<T, MT, kRes, 2 * Q, false, true, false, 1, 320>(op, gr, rows, partial, st);
  }
  constexpr int kPer = 16 / kVec<T>;  // 16 values a thread, or 8 where that leaves fewer threads idle
  constexpr int kWide = kRes && sizeof(T) == 4 ? 320 : 512;  // threads whose ring fits
  if (vec && nvec > 32 && nvec <= kWide * kPer && g.rows >= 8 && even_rows(g, op->batch)) {
    if (nvec % (32 * kPer) == 0) {
      if (nvec <= 320 * kPer)
        return launch_backward_stream<T, MT, kRes, kPer, true, false, false, kRes ? 1 : 2, 320>(op, gr, g, partial, st);
      return launch_backward_stream<T, MT, kRes, kPer, true, false, kRes, 1, kWide>(op, gr, g, partial, st);
    }
    if (half_fits_better(nvec, kPer))
      return launch_backward_stream<T, MT, kRes, kPer / 2, false, false, false, 1, 512>(op, gr, g, partial, st);
    return launch_backward_stream<T, MT, kRes, kPer, false, false, kRes, 1, kWide>(op, gr, g, partial, st);
  }
  if (!vec) {
    if (gr->mod_tokens && op->tokens >= 8 && (gr->mod_batch || op->batch == 1) &&
        any_fits<T, MT, kRes, true, true>(op->channels))
      return launch_backward_any<T, MT, kRes, true>(op, gr, make_groups(op->batch, op->tokens, 1, 0), partial, st);
    if (!gr->mod_tokens && g.rows >= 8 && even_rows(g, op->batch) && any_fits<T, MT, kRes, false, true>(op->channels))
      return launch_backward_any<T, MT, kRes, false>(op, gr, g, partial, st);
  }
  const int per = nvec <= 32 ? 1 : vec ? (nvec <= 1024 ? 1 : nvec <= 2048 ? 2 : 4) : nvec <= 4096 ? 4 : 16;
  return by_shape<T>(vec, per, [&](auto v, auto p) {
    constexpr int V = decltype(v)::value, P = decltype(p)::value;
    const int team = team_for((nvec + P - 1) / P);
    const int threads = team > 32 ? team : kCtaThreads, teams = threads / team;
    const int own = g.rows < 4 * teams;
    if (own) {
      g.chunks = 1;
      g.chunk_rows = g.rows;
    } else {
      cut_groups(g, std::min((int64_t)sm_count() * 4, most_runs(op->channels)), 4 * teams);
    }
    const int64_t units = g.count * g.chunks, ctas = own ? (units + teams - 1) / teams : units;
    const size_t smem = !own && teams > 1 ? (size_t)teams * 3 * op->channels * sizeof(float) : 0;
    adaln_backward_kernel<T, MT, V, P, kRes><<<(unsigned)ctas, threads, smem, st>>>(*op, *gr, g, team, own, partial);
    return join<MT>(op, gr, g, partial, st);
  });
}

}  // namespace

}  // namespace spr

using namespace spr;

extern "C" int spr_adaln_forward(const SprAdaln* op, void* stream) {
  if (int rc = check_adaln(op)) return rc;
  if (op->batch * op->tokens == 0) return SPR_OK;
  if (!op->x || !op->h || (op->y && !op->z)) return fail(SPR_ERR_ARG, "adaln forward: null operand");
  if (int rc = check_pointers(op, nullptr)) return rc;
  SprAdaln o = *op;
  merge_batch(o, nullptr);
  return by_type(op, [&](auto t, auto m) {
    using T = decltype(t);
    using MT = decltype(m);
    return op->y ? launch_forward<T, MT, true>(&o, (cudaStream_t)stream)
                 : launch_forward<T, MT, false>(&o, (cudaStream_t)stream);
  });
}

extern "C" size_t spr_adaln_backward_workspace_bytes(int64_t batch, int64_t tokens, int channels, int mod_batch,
                                                     int mod_tokens) {
  if (batch <= 0 || tokens <= 0 || channels <= 0 || channels > kMaxChannels || !rows_fit(batch, tokens)) return 0;
  Groups g = make_groups(batch, tokens, mod_batch, mod_tokens);
  cut_groups(g, most_runs(channels), 4);  // as many runs as any launch takes
  return g.chunks == 1 ? 0 : (size_t)g.count * g.chunks * 3 * channels * sizeof(float);
}

extern "C" int spr_adaln_backward(const SprAdaln* op, const SprAdalnGrad* grad, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_adaln(op)) return rc;
  if (!grad) return fail(SPR_ERR_ARG, "adaln backward: no gradients");
  if (op->batch * op->tokens == 0) return SPR_OK;
  if (!op->x || !op->mean || !op->rstd || !grad->dh || !grad->dx || (op->y && !grad->dy) || (grad->dgate && !op->y))
    return fail(SPR_ERR_ARG, "adaln backward: null operand");
  if (grad->dz && !op->y) return fail(SPR_ERR_ARG, "adaln backward: a gradient of z without a branch");
  if (int rc = check_pointers(op, grad)) return rc;
  for (auto [p, sb, st] : {std::tuple(op->scale, op->scale_sb, op->scale_st), std::tuple(op->gate, op->gate_sb, op->gate_st)})
    if (p && ((sb && op->batch > 1 && !grad->mod_batch) || (st && op->tokens > 1 && !grad->mod_tokens)))
      return fail(SPR_ERR_ARG, "adaln backward: a vector has a stride along an axis that its gradient is summed over");
  const size_t need =
      spr_adaln_backward_workspace_bytes(op->batch, op->tokens, op->channels, grad->mod_batch, grad->mod_tokens);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(SPR_ERR_WORKSPACE, "adaln backward: workspace %zu < %zu bytes or not 16-byte aligned", workspace_bytes,
                need);
  SprAdaln o = *op;
  SprAdalnGrad gr = *grad;
  merge_batch(o, &gr);
  return by_type(op, [&](auto t, auto m) {
    using T = decltype(t);
    using MT = decltype(m);
    return op->y ? launch_backward<T, MT, true>(&o, &gr, (float*)workspace, (cudaStream_t)stream)
                 : launch_backward<T, MT, false>(&o, &gr, (float*)workspace, (cudaStream_t)stream);
  });
}
