// Modulated layer norm with an optional gated residual in front of it, forward
// and backward (the operands are described at SprAdaln in the header):
//   z = x + gate*y,  n = (z - mean z) * rstd,  h = n*w + shift,  w = offset + scale
//   u = dh*w,  g = dz + rstd*(u - mean u - n*mean(u*n)),  dx = g,  dy = g*gate
//   dshift = sum dh,  dscale = sum dh*n,  dgate = sum g*y   over the rows of a group
// Statistics and sums are fp32.
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
  for (int o = min(team, 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ uint64_t team_sum2(uint64_t v, int team) {
  for (int o = min(team, 32) / 2; o > 0; o >>= 1) v = add2(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ uint64_t warp_sum2(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = add2(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Two sums over a CTA's warps with one barrier.  Two buffers in turn: a warp that
// writes the next row's pair does not meet readers of this row's.  `red` starts
// as zeros, so an odd number of warps reads a zero pair.
__device__ __forceinline__ uint64_t warps_sum2(uint64_t v, ulonglong2* red, int warps) {
  if ((threadIdx.x & 31) == 0) reinterpret_cast<uint64_t*>(red)[threadIdx.x >> 5] = v;
  __syncthreads();
  uint64_t a = 0, b = 0;
#pragma unroll 4
  for (int w = 0; w < (warps + 1) / 2; ++w) {
    const ulonglong2 e = red[w];
    a = add2(a, e.x);
    b = add2(b, e.y);
  }
  return add2(a, b);
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

// One row per team.  The row stays in registers; the variance is taken about the
// warp's own mean and the warps' values are joined by
//   M2 = sum_w M2_w + n_w (mean_w - mean)^2,
// so that a row costs one barrier and loses nothing to an offset.
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
  // Mean and centred squares of the warp's (or the smaller team's) elements.
  const int first = lane & ~31;  // the warp's first vector in its team
  uint64_t acc = 0;
  int n = 0;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    n += min(max(nvec - first - p * team, 0), min(team, 32)) * V;
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i) acc = add2(acc, z[p].q[i]);
  }
  float2 h = halves(acc);
  const float sum = team_sum(h.x + h.y, team);
  float mean = sum * __frcp_rn((float)n);
  uint64_t minus = both<V>(-mean);
  acc = 0;
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (lane + p * team < nvec)
#pragma unroll
      for (int i = 0; i < Vals<V>::kPairs; ++i) {
        const uint64_t d = add2(z[p].q[i], minus);
        acc = fma2(d, d, acc);
      }
  h = halves(acc);
  float m2 = team_sum(h.x + h.y, team);
  const float inv_c = __frcp_rn((float)c);
  if (team > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = make_float4(sum, mean, m2, (float)n);
    __syncthreads();
    const int warps = team / 32;
    float total = 0.f;
    m2 = 0.f;
#pragma unroll 4
    for (int w = 0; w < warps; ++w) total += red[w].x;
    mean = total * inv_c;
#pragma unroll 4
    for (int w = 0; w < warps; ++w) {
      const float4 e = red[w];
      const float d = e.y - mean;
      m2 += fmaf(d * d, e.w, e.z);
    }
  }
  const float rstd = rsqrtf(m2 * inv_c + op.eps);
  if (!valid) return;
  minus = both<V>(-mean);
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

// The rows that share one vector: row r of group g is g*group_step + r*row_step.
// A group's rows are cut into `chunks` runs; run s of group g writes its column
// sums to partial[g][s] (or, with one run, the gradients themselves).
struct Groups {
  int64_t count, rows, group_step, row_step;
  int chunks;
  int64_t chunk_rows;
};

// The row arithmetic that both backward kernels share: n, u and the sums before
// the reduction, the gradients after it.
template <int V, int P>
struct Backward {
  Vals<V> n[P], u[P];
  Vals<V> shift[P], scale[P], gate[P];  // column sums

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      shift[p].fill(0.f);
      scale[p].fill(0.f);
      gate[p].fill(0.f);
      n[p].fill(0.f);
      u[p].fill(0.f);
    }
  }
  __device__ __forceinline__ void first(int p, const Vals<V>& z, const Vals<V>& dh, const Vals<V>& w, uint64_t minus,
                                        uint64_t rstd, uint64_t& s0, uint64_t& s1) {
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i) {
      n[p].q[i] = mul2(add2(z.q[i], minus), rstd);
      u[p].q[i] = mul2(dh.q[i], w.q[i]);
      s0 = add2(s0, u[p].q[i]);
      s1 = fma2(u[p].q[i], n[p].q[i], s1);
      shift[p].q[i] = add2(shift[p].q[i], dh.q[i]);
      scale[p].q[i] = fma2(dh.q[i], n[p].q[i], scale[p].q[i]);
    }
  }
  // rstd*(u - m0 - n*m1) + dz
  __device__ __forceinline__ void second(int p, uint64_t minus_m0, uint64_t minus_m1, uint64_t rstd, const Vals<V>& dz,
                                         Vals<V>& g) const {
#pragma unroll
    for (int i = 0; i < Vals<V>::kPairs; ++i)
      g.q[i] = fma2(fma2(n[p].q[i], minus_m1, add2(u[p].q[i], minus_m0)), rstd, dz.q[i]);
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
// itself (groups of few rows, such as a vector for every token).
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
  Backward<V, P> st;
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
        st.first(p, z, dh, w, minus, rstd, s0, s1);
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
        st.second(p, m0, m1, rstd, dz, gx);
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

__device__ __forceinline__ void copy16_async(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}

// A thread's place in one operand, moved row by row along a group.
struct Cursor {
  const char* p;
  int64_t step, wrap;  // bytes to the group's next row, and further where the batch ends
  __device__ __forceinline__ Cursor(const void* base, int64_t sb, int64_t st, int e, const RowId& id, int64_t tokens,
                                    bool along_tokens, int first)
      : p((const char*)base + (id.b * sb + id.t * st) * e + first * 16),
        step((along_tokens ? st : sb) * e),
        wrap((sb - tokens * st) * e) {}
  __device__ __forceinline__ void next(bool ends) { p += ends ? step + wrap : step; }
};

// Long groups of wide rows: a few CTAs per SM walk runs of rows with their column
// sums in registers.  Each thread copies its own 16-byte vectors of the next
// kStages - 1 rows into shared memory, so the copies need no barrier and stay in
// flight across the one that joins a row's two sums.
template <typename T, typename MT, int P, bool kRes, int kThreads, int kStages>
__global__ void __launch_bounds__(kThreads)
adaln_backward_stream_kernel(const SprAdaln op, const SprAdalnGrad gr, const Groups gp, float* partial) {
  constexpr int V = kVec<T>, kIn = kRes ? 4 : 2, e = sizeof(T);
  __shared__ ulonglong2 red[2][16];
  extern __shared__ uint4 ring[];  // [stage][operand][P][thread]
  const int c = op.channels, nvec = c / V, team = blockDim.x, lane = threadIdx.x;
  const int64_t g = blockIdx.x / gp.chunks, s = blockIdx.x % gp.chunks;
  const int64_t r0 = s * gp.chunk_rows;
  const int rows = (int)(min(gp.rows, r0 + gp.chunk_rows) - r0);
  const float inv_c = 1.f / c;
  const int64_t row0 = g * gp.group_step + r0 * gp.row_step;
  const RowId gid = row_id(op, g * gp.group_step), id0 = row_id(op, row0);
  const bool along = gp.row_step == 1;
  if (lane < 64) (&red[0][0].x)[lane] = 0;
  __syncthreads();
  Backward<V, P> st;
  st.clear();
  Vals<V> w[P], gate[P];
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (lane + p * team < nvec) {
      load_factor<MT, V>(op, gid, lane + p * team, w[p]);
      if constexpr (kRes) load_gate<MT, V>(op, gid, lane + p * team, gate[p]);
    }
  Cursor cx(op.x, op.x_sb, op.x_st, e, id0, op.tokens, along, lane);
  Cursor cd(gr.dh, gr.dh_sb, gr.dh_st, e, id0, op.tokens, along, lane);
  Cursor cy(kRes ? op.y : op.x, op.y_sb, op.y_st, e, id0, op.tokens, along, lane);
  Cursor cz(kRes && gr.dz ? gr.dz : op.x, gr.dz_sb, gr.dz_st, e, id0, op.tokens, along, lane);
  int left = along ? (int)(op.tokens - id0.t) : 0x7fffffff;  // rows before the batch ends
  int fetched = 0;
  auto fetch = [&](int stage) {
    if (fetched < rows) {
      uint4* to = ring + stage * (kIn * P) * team + lane;
#pragma unroll
      for (int p = 0; p < P; ++p)
        if (lane + p * team < nvec) {
          copy16_async(to + (0 * P + p) * team, cx.p + p * team * 16);
          copy16_async(to + (1 * P + p) * team, cd.p + p * team * 16);
          if constexpr (kRes) {
            copy16_async(to + (2 * P + p) * team, cy.p + p * team * 16);
            if (gr.dz) copy16_async(to + (3 * P + p) * team, cz.p + p * team * 16);
          }
        }
      const bool ends = --left == 0;
      if (ends) left = (int)op.tokens;
      cx.next(ends);
      cd.next(ends);
      if constexpr (kRes) {
        cy.next(ends);
        cz.next(ends);
      }
      ++fetched;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) fetch(i);
  int stage = 0;
  const float *mean_at = op.mean + row0, *rstd_at = op.rstd + row0;
  float mean = *mean_at, rstd = *rstd_at;
  char* dx = (char*)gr.dx + ((row0 * c) * e + lane * 16);
  char* dy = (char*)gr.dy + ((row0 * c) * e + lane * 16);
  const int64_t out_step = gp.row_step * c * e;
  for (int r = 0; r < rows; ++r) {
    if (r + 1 < rows) {
      mean_at += gp.row_step;
      rstd_at += gp.row_step;
    }
    const float next_mean = *mean_at, next_rstd = *rstd_at;
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    const uint4* slot = ring + stage * (kIn * P) * team + lane;
    uint64_t s0 = 0, s1 = 0;
    const uint64_t rs = pair(rstd, rstd);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (lane + p * team >= nvec) continue;
      Vals<V> z, dh;
      unpack16<T>(slot[(0 * P + p) * team], z.q);
      unpack16<T>(slot[(1 * P + p) * team], dh.q);
      st.first(p, z, dh, w[p], pair(-mean, -mean), rs, s0, s1);
    }
    const float2 a = halves(s0), b = halves(s1);
    uint64_t sums = warp_sum2(pair(a.x + a.y, b.x + b.y));
    // The slot that this fetch fills was read in the round before.
    fetch(stage == 0 ? kStages - 1 : stage - 1);
    sums = warps_sum2(sums, red[r & 1], team / 32);
    const float2 m = halves(sums);
    const uint64_t m0 = both<V>(-m.x * inv_c), m1 = both<V>(-m.y * inv_c);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (lane + p * team >= nvec) continue;
      Vals<V> gx, dz;
      if (kRes && gr.dz) unpack16<T>(slot[(3 * P + p) * team], dz.q);
      else dz.fill(0.f);
      st.second(p, m0, m1, rs, dz, gx);
      if constexpr (kRes) {
        Vals<V> y, gy = gate[p];
        unpack16<T>(slot[(2 * P + p) * team], y.q);
        st.branch(p, gx, y, gy);
        *reinterpret_cast<uint4*>(dy + p * team * 16) = pack16<T>(gy.q);
      }
      *reinterpret_cast<uint4*>(dx + p * team * 16) = pack16<T>(gx.q);
    }
    dx += out_step;
    if constexpr (kRes) dy += out_step;
    mean = next_mean;
    rstd = next_rstd;
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int v = lane + p * team;
    if (v < nvec) store_sums<MT, V>(gr, gp, blockIdx.x, c, v, partial, st.shift[p], st.scale[p], st.gate[p]);
  }
}

// Joins the runs' column sums in their order: 32 columns by 32 threads each.
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

// Threads a row: a power of two of lanes up to a warp, whole warps above.
int team_for(int vectors) {
  if (vectors > 32) return (vectors + 31) / 32 * 32;
  int t = 1;
  while (t < vectors) t *= 2;
  return t;
}

int check_adaln(const SprAdaln* op) {
  if (!op) return fail(SPR_ERR_ARG, "adaln: no operands");
  if (op->batch < 0 || op->tokens < 0 || op->channels < 1 || op->channels > kMaxChannels)
    return fail(SPR_ERR_SHAPE, "adaln: batch=%lld tokens=%lld channels=%d (channels must be 1..%d)",
                (long long)op->batch, (long long)op->tokens, op->channels, kMaxChannels);
  if (op->tokens && op->batch > 0x7fffffffLL / op->tokens) return fail(SPR_ERR_SHAPE, "adaln: batch*tokens too large");
  if (op->dtype != SPR_F32 && op->dtype != SPR_BF16 && op->dtype != SPR_F16)
    return fail(SPR_ERR_DTYPE, "adaln: unsupported dtype %d", op->dtype);
  if (op->mod_dtype != op->dtype && op->mod_dtype != SPR_F32)
    return fail(SPR_ERR_DTYPE, "adaln: shift/scale/gate dtype %d must be the element type %d or fp32", op->mod_dtype,
                op->dtype);
  if (op->gate && !op->y) return fail(SPR_ERR_ARG, "adaln: a gate without a branch");
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

constexpr int kCtaThreads = 256;  // of a CTA whose teams are at most a warp

template <typename T>
int forward_per_thread(bool vec, int nvec) {
  if (nvec <= 32) return 1;
  if (vec) return nvec <= 64 ? 1 : nvec <= 128 ? 2 : 4;
  return nvec <= 4096 ? 4 : 16;
}

template <typename T, typename MT, bool kRes>
int launch_forward(const SprAdaln* op, cudaStream_t st) {
  const bool vec = vectors_fit(op);
  const int nvec = op->channels / (vec ? kVec<T> : 1);
  return by_shape<T>(vec, forward_per_thread<T>(vec, nvec), [&](auto v, auto p) {
    constexpr int V = decltype(v)::value, P = decltype(p)::value;
    const int team = team_for((nvec + P - 1) / P);
    const int threads = team > 32 ? team : kCtaThreads;
    const int64_t rows = op->batch * op->tokens, teams = threads / team;
    adaln_forward_kernel<T, MT, V, P, kRes><<<(unsigned)((rows + teams - 1) / teams), threads, 0, st>>>(*op, team);
    return check_launch("adaln forward");
  });
}

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

constexpr int kMaxCtasPerSm = 4;

template <typename MT>
int join(const SprAdaln* op, const SprAdalnGrad* gr, const Groups& g, const float* partial, cudaStream_t st) {
  if (g.chunks > 1 && (gr->dshift || gr->dscale || gr->dgate))
    adaln_join_kernel<MT><<<dim3((unsigned)g.count, (op->channels + 31) / 32, gr->dgate ? 3 : 2), dim3(32, 32), 0, st>>>(
        *gr, op->channels, g.chunks, partial);
  return check_launch("adaln backward");
}

template <typename T, typename MT, bool kRes, int P, int kThreads, int kStages>
int launch_stream(const SprAdaln* op, const SprAdalnGrad* gr, Groups g, int team, float* partial, cudaStream_t st) {
  auto kern = adaln_backward_stream_kernel<T, MT, P, kRes, kThreads, kStages>;
  const int smem = kStages * (kRes ? 4 : 2) * P * team * 16;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("adaln backward");
  cut_groups(g, (int64_t)sm_count() * std::min(kMaxCtasPerSm, std::max(1, 320 / team)), 4);
  kern<<<(unsigned)(g.count * g.chunks), team, smem, st>>>(*op, *gr, g, partial);
  return join<MT>(op, gr, g, partial, st);
}

template <typename T, typename MT, bool kRes>
int launch_backward(const SprAdaln* op, const SprAdalnGrad* gr, float* partial, cudaStream_t st) {
  const bool vec = vectors_fit(op, gr);
  const int nvec = op->channels / (vec ? kVec<T> : 1);
  Groups g = make_groups(op->batch, op->tokens, gr->mod_batch, gr->mod_tokens);
  if (vec && nvec > 32 && nvec <= 1024 && g.rows >= 8) {
    if (nvec <= 128) return launch_stream<T, MT, kRes, 1, 128, 4>(op, gr, g, team_for(nvec), partial, st);
    const int team = team_for((nvec + 1) / 2);
    if (team <= 384) return launch_stream<T, MT, kRes, 2, 384, 4>(op, gr, g, team, partial, st);
    return launch_stream<T, MT, kRes, 2, 512, 3>(op, gr, g, team, partial, st);
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
      cut_groups(g, (int64_t)sm_count() * kMaxCtasPerSm, 4 * teams);
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
  return by_type(op, [&](auto t, auto m) {
    using T = decltype(t);
    using MT = decltype(m);
    return op->y ? launch_forward<T, MT, true>(op, (cudaStream_t)stream)
                 : launch_forward<T, MT, false>(op, (cudaStream_t)stream);
  });
}

extern "C" size_t spr_adaln_backward_workspace_bytes(int64_t batch, int64_t tokens, int channels, int mod_batch,
                                                     int mod_tokens) {
  if (batch <= 0 || tokens <= 0 || channels <= 0) return 0;
  Groups g = make_groups(batch, tokens, mod_batch, mod_tokens);
  cut_groups(g, (int64_t)sm_count() * kMaxCtasPerSm, 4);  // as many runs as any launch takes
  return g.chunks == 1 ? 0 : (size_t)g.count * g.chunks * 3 * channels * sizeof(float);
}

extern "C" int spr_adaln_backward(const SprAdaln* op, const SprAdalnGrad* grad, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  if (int rc = check_adaln(op)) return rc;
  if (!grad) return fail(SPR_ERR_ARG, "adaln backward: no gradients");
  if (op->batch * op->tokens == 0) return SPR_OK;
  if (!op->x || !op->mean || !op->rstd || !grad->dh || !grad->dx || (op->y && !grad->dy) || (grad->dgate && !op->y))
    return fail(SPR_ERR_ARG, "adaln backward: null operand");
  const size_t need =
      spr_adaln_backward_workspace_bytes(op->batch, op->tokens, op->channels, grad->mod_batch, grad->mod_tokens);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(SPR_ERR_WORKSPACE, "adaln backward: workspace %zu < %zu bytes or not 16-byte aligned", workspace_bytes,
                need);
  return by_type(op, [&](auto t, auto m) {
    using T = decltype(t);
    using MT = decltype(m);
    return op->y ? launch_backward<T, MT, true>(op, grad, (float*)workspace, (cudaStream_t)stream)
                 : launch_backward<T, MT, false>(op, grad, (float*)workspace, (cudaStream_t)stream);
  });
}
