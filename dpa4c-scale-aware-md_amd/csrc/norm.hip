// Group norm with an activation, channels last, forward and backward, of one element kind (ELEM_KIND, one
// object file each):
//
//   v = (x - m) r, z = gamma v + beta, y = act(z)      m, r = 1 / sqrt(variance + eps) of a frame and group
//   dz = dy act'(z), w = gamma dz
//   dx = r (w - mean(w) - v mean(w v)),  dgamma = sum dz v,  dbeta = sum dz        (sums over all frames' rows)
//
// Every pass is bound by the bytes it moves, so the forms differ in how often they read x: once where a row
// is a frame (in registers), twice where a block sees a whole frame (the second time from the caches while
// the frame's part fits them), twice and with one more launch where frames are cut into slices.
//
// Means and squared deviations are joined from those of parts: a thread forms both over the values that it
// holds, around their own mean, and parts are joined by
//   m = sum n_i m_i / n,  M = sum M_i + sum n_i (m_i - m)^2,
// so that no difference of large sums occurs whatever the mean is. All in fp32; slices are joined in
// fp64. Sums have an order that sizes alone fix.
#include <algorithm>

#include "norm.h"
#include "quant8.h"

namespace dpamd {

namespace {

constexpr int kThreads = 256;

struct Pair {
  float a, b;
};

// Rows of frame f: [first, first + count)
struct Frame {
  long first;
  int count;
};
__device__ __forceinline__ Frame frame_of(const NormArgs& p, int f) {
  if (!p.starts) {
    const long each = p.rows / p.frames;
    return Frame{f * each, (int)each};
  }
  // (whatever starts holds, no row outside the matrix is touched)
  const long a = min(max((long)p.starts[f], 0l), p.rows), b = min(max((long)p.starts[f + 1], a), p.rows);
  return Frame{a, (int)(b - a)};
}

// VE elements as they lie in memory: what is loaded ahead, or kept for long, takes no more registers than that
// (held in words: single elements of 16 or 8 bits would take a register each).
template <int KIND, int VE>
struct Raw {
  using E = typename ElemOf<KIND>::T;
  static constexpr int kBytes = VE * sizeof(E), kWords = (kBytes + 3) / 4;
  unsigned w[kWords];
  __device__ __forceinline__ void load(const E* p) {
    if constexpr (kBytes == 2)
      w[0] = *p;
    else
      __builtin_memcpy(w, p, kBytes);  // (the hardware takes addresses of any alignment)
  }
  __device__ __forceinline__ void zeros() {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = 0;
  }
  __device__ __forceinline__ void ones() {
    const unsigned one = KIND == kF32 ? 0x3f800000u : KIND == kBf16 ? 0x3f803f80u : 0x3c003c00u;
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = one;
  }
  __device__ __forceinline__ void get(float (&out)[VE]) const {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      if constexpr (KIND == kF32)
        out[e] = __builtin_bit_cast(float, w[e]);
      else
        out[e] = to_f32<KIND>((unsigned short)(w[e / 2] >> (16 * (e % 2))));
    }
  }
};
// the same of x or its checkpoint
// v = x r - m r: one instruction a value. (m r is rounded, by no more than m itself is.)
template <int KIND, int VE, bool KEPT>
struct RawX : Raw<KIND, VE> {
  __device__ __forceinline__ void load_at(const NormArgs& p, long row, int chunk) {
    this->load(static_cast<const typename ElemOf<KIND>::T*>(p.x) + row * p.ld_x + (long)chunk * VE);
  }
  __device__ __forceinline__ void normalized(const Pair& s, float (&out)[VE]) const {
    this->get(out);
#pragma unroll
    for (int e = 0; e < VE; ++e) out[e] = __builtin_fmaf(out[e], s.b, -s.a * s.b);
  }
};
template <int KIND, int VE>
struct RawX<KIND, VE, true> {
  static constexpr int kWords = (VE + 3) / 4;
  unsigned w[kWords];
  unsigned char field;
  __device__ __forceinline__ void load_at(const NormArgs& p, long row, int chunk) {
    const unsigned char* at = p.kept + row * p.wide + chunk * VE;
    if constexpr (VE == 1) {
      w[0] = *at;
    } else if constexpr (VE == 2) {
      unsigned short v;
      __builtin_memcpy(&v, at, 2);
      w[0] = v;
    } else {
      __builtin_memcpy(w, at, VE);
    }
    field = p.kept[p.rows * p.wide + row * (p.wide / 32) + chunk * VE / 32];
  }
  __device__ __forceinline__ void normalized(const Pair& s, float (&out)[VE]) const {
    const float unit = unit_of(field) * s.b;
#pragma unroll
    for (int e = 0; e < VE; ++e)
      out[e] = __builtin_fmaf((float)(signed char)(w[e / 4] >> (8 * (e % 4))), unit, -s.a * s.b);
  }
};

template <int KIND, int VE>
__device__ __forceinline__ void load_vec(float (&v)[VE], const typename ElemOf<KIND>::T* p) {
  Raw<KIND, VE> r;
  r.load(p);
  r.get(v);
}
template <int KIND, int VE>
__device__ __forceinline__ void store_vec(typename ElemOf<KIND>::T* p, const float (&v)[VE]) {
  struct Some {
    typename ElemOf<KIND>::T v[VE];
  } s;
#pragma unroll
  for (int e = 0; e < VE; ++e) s.v[e] = from_f32<KIND>(v[e]);
  __builtin_memcpy(p, &s, sizeof(s));
}
template <int KIND, int VE>
__device__ __forceinline__ void load_affine(const NormArgs& p, int chunk, float (&gamma)[VE], float (&beta)[VE]) {
  using T = typename ElemOf<KIND>::T;
#pragma unroll
  for (int e = 0; e < VE; ++e) gamma[e] = 1.0f, beta[e] = 0.0f;
  if (p.gamma) load_vec<KIND, VE>(gamma, static_cast<const T*>(p.gamma) + (long)chunk * VE);
  if (p.beta) load_vec<KIND, VE>(beta, static_cast<const T*>(p.beta) + (long)chunk * VE);
}

// The same past the caches, where `once` (uniform).
template <int KIND, int VE>
__device__ __forceinline__ void store_out(typename ElemOf<KIND>::T* p, const float (&v)[VE], bool once) {
  if constexpr (VE * sizeof(*p) == 16) {
    if (once) {
      struct Some {
        typename ElemOf<KIND>::T v[VE];
      } s;
#pragma unroll
      for (int e = 0; e < VE; ++e) s.v[e] = from_f32<KIND>(v[e]);
      return store16<true>(p, __builtin_bit_cast(u4any, s));
    }
  }
  store_vec<KIND, VE>(p, v);
}

// act and its derivative over a thread's values (one uniform branch for all of them)
template <int KIND, int VE>
__device__ __forceinline__ void activate_vec(int act, const float (&z)[VE], float (&a)[VE], float (&da)[VE]) {
  auto all = [&](auto k) {
#pragma unroll
    for (int e = 0; e < VE; ++e) activate_as<KIND, decltype(k)::value>(z[e], a[e], da[e]);
  };
  if (act == kActNone) {
#pragma unroll
    for (int e = 0; e < VE; ++e) a[e] = z[e], da[e] = 1.0f;
  } else if (act == kActTanh) {
    all(std::integral_constant<int, kActTanh>{});
  } else if (act == kActSilu) {
    all(std::integral_constant<int, kActSilu>{});
  } else {
    all(std::integral_constant<int, kActGelu>{});
  }
}
// x -> act(x scale + shift)
template <int KIND, int VE>
__device__ __forceinline__ void forward_vec(int act, const float (&scale)[VE], const float (&shift)[VE],
                                            float (&x)[VE]) {
  float z[VE], da[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) z[e] = __builtin_fmaf(x[e], scale[e], shift[e]);
  activate_vec<KIND, VE>(act, z, x, da);
}
// dy -> dz
template <int KIND, int VE>
__device__ __forceinline__ void grad_vec(int act, const float (&gamma)[VE], const float (&beta)[VE],
                                         const float (&v)[VE], float (&dy)[VE]) {
  float z[VE], a[VE], da[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) z[e] = __builtin_fmaf(gamma[e], v[e], beta[e]);
  activate_vec<KIND, VE>(act, z, a, da);
#pragma unroll
  for (int e = 0; e < VE; ++e) dy[e] *= da[e];
}
// w = gamma dz -> dx = r (w - mean w - v mean(w v))
template <int VE>
__device__ __forceinline__ void dx_vec(float r, const Pair& means, const float (&v)[VE], float (&w)[VE]) {
  const float a = -r * means.a, b = -r * means.b;
#pragma unroll
  for (int e = 0; e < VE; ++e) w[e] = __builtin_fmaf(v[e], b, __builtin_fmaf(w[e], r, a));
}

// mean and squared deviations of VE values
template <int VE>
__device__ __forceinline__ Pair moments(const float (&v)[VE]) {
  float s = 0.0f, q = 0.0f;
#pragma unroll
  for (int e = 0; e < VE; ++e) s += v[e];
  const float m = s * (1.0f / VE);
#pragma unroll
  for (int e = 0; e < VE; ++e) q += (v[e] - m) * (v[e] - m);
  return Pair{m, q};
}
// (m, M) of n values joined with that of k more
__device__ __forceinline__ void join_moments(Pair& p, float n, const Pair& q, float k) {
  const float d = q.a - p.a, w = n == 0.0f ? 1.0f : k * __builtin_amdgcn_rcpf(n + k);
  p.a += d * w;
  p.b += q.b + d * d * n * w;
}

// The sum over 2^log_lanes neighbouring lanes, in each of them (every lane of the wave takes part).
__device__ __forceinline__ float sum_lanes(float v, int log_lanes) {
  if (log_lanes > 0) v = add_dpp<0xB1>(v);   // lane ^ 1
  if (log_lanes > 1) v = add_dpp<0x4E>(v);   // lane ^ 2
  if (log_lanes > 2) v = add_dpp<0x141>(v);  // 7 - lane: the other quad, whose lanes are alike by now
  if (log_lanes > 3) v = add_dpp<0x140>(v);  // 15 - lane
  if (log_lanes > 4) v = add_xor16(v);
  if (log_lanes > 5) v = add_xor32(v);
  return v;
}
// 1 / sqrt(M / n + eps), inv = 1 / n
__device__ __forceinline__ float deviation(float M, float inv, float eps) {
  return __builtin_amdgcn_rsqf(__builtin_fmaf(M, inv, eps));
}

// A barrier among the threads that share a row: a wave's, or the block's.
template <int T>
__device__ __forceinline__ void row_sync() {
  if constexpr (T > 64)
    __syncthreads();
  else
    wave_lds_sync();
}

// f(group, lane, whether there is such a group) for all groups, each by 2^lanes neighbouring threads.
template <int T, class F>
__device__ __forceinline__ void each_group(int t, int groups, int lanes, F&& f) {
  const int width = 1 << lanes;
  for (int q0 = 0; q0 < groups; q0 += T >> lanes) {
    const int q = q0 + (t >> lanes);
    f(min(q, groups - 1), t & (width - 1), q < groups);  // (every lane takes part in the shuffles)
  }
}

// ---- every row a frame -----------------------------------------------------------------
// T threads a row, C chunks of VE channels a thread (at neighbouring places for neighbouring threads). With
// LANES a group is a power of two of chunks, at most 64, so that it is that many neighbouring lanes, which
// add up without LDS or a barrier; else the parts of a row meet in LDS, a pair for each chunk and then one
// for each group. (16,384 x 2048 in bf16, groups of 64, gelu: XXX.)
// A block takes rows one after another: gamma and beta stay in registers, and the next row is loaded
// while this one is computed.
template <int KIND, int VE, int T, int C, bool LANES>
__global__ __launch_bounds__(kThreads) void k_norm_rows(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  extern __shared__ __align__(16) char lds[];
  constexpr int R = kThreads / T;
  const int t = threadIdx.x % T, mine = threadIdx.x / T;
  Pair* parts = reinterpret_cast<Pair*>(lds) + (size_t)mine * (p.chunks + p.groups);
  Pair* whole = parts + p.chunks;
  float gamma[C][VE], beta[C][VE];
#pragma unroll
  for (int k = 0; k < C; ++k) load_affine<KIND, VE>(p, min(k * T + t, p.chunks - 1), gamma[k], beta[k]);
  Raw<KIND, VE> raw[C];
  auto fetch = [&](long row) {
    const E* x = static_cast<const E*>(p.x) + min(row, p.rows - 1) * p.ld_x;
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (k * T + t < p.chunks) raw[k].load(x + (long)(k * T + t) * VE);
  };
  const long step = (long)gridDim.x * R;
  fetch((long)blockIdx.x * R + mine);
  for (long row0 = (long)blockIdx.x * R; row0 < p.rows; row0 += step) {
    const long row = row0 + mine;
    const bool there = row < p.rows;
    float v[C][VE];
    Pair stat[C];
    auto keep = [&](int q, const Pair& s) {
      if (p.stats && there) *reinterpret_cast<Pair*>(p.stats + 2 * (row * p.groups + q)) = s;
    };
    if constexpr (LANES) {
#pragma unroll
      for (int k = 0; k < C; ++k) {
        raw[k].get(v[k]);
        const Pair s = moments<VE>(v[k]);
        const float m = sum_lanes(s.a, p.lanes) * p.inv_chunks;
        const float M = sum_lanes(s.b + VE * (s.a - m) * (s.a - m), p.lanes);
        stat[k] = Pair{m, deviation(M, p.inv_per, p.eps)};
        const int chunk = k * T + t;
        if (chunk < p.chunks && (t & (p.chunks_per - 1)) == 0) keep(chunk / p.chunks_per, stat[k]);
      }
      if (row0 + step < p.rows) fetch(row + step);
    } else {
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k * T + t < p.chunks) {
          raw[k].get(v[k]);
          parts[k * T + t] = moments<VE>(v[k]);
        }
      if (row0 + step < p.rows) fetch(row + step);
      row_sync<T>();
      each_group<T>(t, p.groups, p.lanes, [&](int q, int lane, bool in) {
        const Pair* s = parts + q * p.chunks_per;
        float m = 0.0f, M = 0.0f;
        for (int k = lane; k < p.chunks_per; k += 1 << p.lanes) m += s[k].a;
        m = sum_lanes(m, p.lanes) * p.inv_chunks;
        for (int k = lane; k < p.chunks_per; k += 1 << p.lanes) M += s[k].b + VE * (s[k].a - m) * (s[k].a - m);
        const Pair r = {m, deviation(sum_lanes(M, p.lanes), p.inv_per, p.eps)};
        if (in && lane == 0) {
          whole[q] = r;
          keep(q, r);
        }
      });
      row_sync<T>();
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k * T + t < p.chunks) stat[k] = whole[(k * T + t) / p.chunks_per];
      row_sync<T>();  // (the next row's parts go where these are read)
    }
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int chunk = k * T + t;
      if (chunk >= p.chunks) continue;
#pragma unroll
      for (int e = 0; e < VE; ++e) v[k][e] = __builtin_fmaf(v[k][e], stat[k].b, -stat[k].a * stat[k].b);
      forward_vec<KIND, VE>(p.act, gamma[k], beta[k], v[k]);
      if (there) store_out<KIND, VE>(static_cast<E*>(p.y) + row * p.ld_y + (long)chunk * VE, v[k], p.once);
    }
  }
}

// Its gradients: dgamma and dbeta of a thread's channels are summed over all rows that its block takes, and
// then over the block's row lanes; partial [blocks][2][channels].
template <int KIND, int VE, int T, int C, bool LANES, bool KEPT>
__global__ __launch_bounds__(kThreads) void k_norm_rows_grad(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  extern __shared__ __align__(16) char lds[];
  constexpr int R = kThreads / T;
  const int t = threadIdx.x % T, mine = threadIdx.x / T;
  Pair* parts = reinterpret_cast<Pair*>(lds) + (size_t)mine * (p.chunks + p.groups);
  Pair* whole = parts + p.chunks;
  float gamma[C][VE], beta[C][VE];
#pragma unroll
  for (int k = 0; k < C; ++k) load_affine<KIND, VE>(p, min(k * T + t, p.chunks - 1), gamma[k], beta[k]);
  float ga[C][VE] = {}, be[C][VE] = {};
  // two rows are under way (with one, 16 waves of a compute unit wait for too few bytes)
  struct Ahead {
    RawX<KIND, VE, KEPT> x[C];
    Raw<KIND, VE> dy[C];
    Pair stat[C];
  } ahead[2];
  auto fetch = [&](long row, Ahead& to) {  // (dy of rows past the last: zeros)
    const bool there = row < p.rows;
    row = min(row, p.rows - 1);
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int chunk = k * T + t;
      if (chunk >= p.chunks) continue;
      to.x[k].load_at(p, row, chunk);
      if (there)
        to.dy[k].load(static_cast<const E*>(p.dy) + row * p.ld_y + (long)chunk * VE);
      else
        to.dy[k].zeros();
      to.stat[k] = *reinterpret_cast<const Pair*>(p.stats + 2 * (row * p.groups + chunk / p.chunks_per));
    }
  };
  const long step = (long)gridDim.x * R;
  auto compute = [&](long row0, Ahead& from) {
    const long row = row0 + mine;
    const bool there = row < p.rows;
    float v[C][VE], w[C][VE], r[C];
    Pair means[C];
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int chunk = k * T + t;
      means[k] = Pair{0.0f, 0.0f};
      if (chunk >= p.chunks) continue;
      from.x[k].normalized(from.stat[k], v[k]);
      from.dy[k].get(w[k]);
      r[k] = from.stat[k].b;
      grad_vec<KIND, VE>(p.act, gamma[k], beta[k], v[k], w[k]);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        be[k][e] += w[k][e];
        ga[k][e] += w[k][e] * v[k][e];
        w[k][e] *= gamma[k][e];
        means[k].a += w[k][e];
        means[k].b += w[k][e] * v[k][e];
      }
      if constexpr (!LANES) parts[chunk] = means[k];
    }
    if (row0 + 2 * step < p.rows) fetch(row + 2 * step, from);
    if constexpr (LANES) {
#pragma unroll
      for (int k = 0; k < C; ++k)
        means[k] = Pair{sum_lanes(means[k].a, p.lanes) * p.inv_per, sum_lanes(means[k].b, p.lanes) * p.inv_per};
    } else {
      row_sync<T>();
      each_group<T>(t, p.groups, p.lanes, [&](int q, int lane, bool in) {
        const Pair* s = parts + q * p.chunks_per;
        float a = 0.0f, b = 0.0f;
        for (int k = lane; k < p.chunks_per; k += 1 << p.lanes) a += s[k].a, b += s[k].b;
        a = sum_lanes(a, p.lanes) * p.inv_per;
        b = sum_lanes(b, p.lanes) * p.inv_per;
        if (in && lane == 0) whole[q] = Pair{a, b};
      });
      row_sync<T>();
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k * T + t < p.chunks) means[k] = whole[(k * T + t) / p.chunks_per];
      row_sync<T>();
    }
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int chunk = k * T + t;
      if (chunk >= p.chunks || !there || !p.dx) continue;
      dx_vec<VE>(r[k], means[k], v[k], w[k]);
      store_out<KIND, VE>(static_cast<E*>(p.dx) + row * p.ld_x + (long)chunk * VE, w[k], p.once);
    }
  };
  const long first = (long)blockIdx.x * R;
  fetch(first + mine, ahead[0]);
  if (first + step < p.rows) fetch(first + step + mine, ahead[1]);
  for (long row0 = first; row0 < p.rows; row0 += 2 * step) {
    compute(row0, ahead[0]);
    if (row0 + step < p.rows) compute(row0 + step, ahead[1]);
  }
  if (!p.partial) return;
  float* out = p.partial + (long)blockIdx.x * 2 * p.channels;
  float* sums = reinterpret_cast<float*>(lds);  // [R][T][VE]
#pragma unroll
  for (int k = 0; k < C; ++k)
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VE; ++e) sums[threadIdx.x * VE + e] = which ? be[k][e] : ga[k][e];
      __syncthreads();
      for (int c = threadIdx.x; c < T * VE; c += kThreads) {
        float s = 0.0f;
        for (int m = 0; m < R; ++m) s += sums[m * T * VE + c];
        if (k * T * VE + c < p.channels) out[which * p.channels + k * T * VE + c] = s;
      }
    }
}

// ---- a block's part of a frame ---------------------------------------------------------------
// Threads (column tc of `part` chunks, row tr): part is at most 256; the threads left over by 256 / part
// idle. Rows tr, tr + TR, ...
struct Lay {
  int tc, tr, TR;
  bool in;
};
__device__ __forceinline__ Lay lay_of(int part, int cols) {
  const int TR = kThreads / part, tr = threadIdx.x / part, tc = threadIdx.x - tr * part;
  return Lay{tc, tr, TR, tr < TR && tc < cols};
}

constexpr int kBatch = 4;  // rows under way

// The moments s of a thread's chunk, joined with those of its rows from the `from`-th on: first + tr + i TR below
// first + count
template <int KIND, int VE>
__device__ __forceinline__ void thread_moments(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                               int from, Pair& s) {
  const typename ElemOf<KIND>::T* x = static_cast<const typename ElemOf<KIND>::T*>(p.x) + (long)chunk * VE;
  int n = from, r = l.tr + from * l.TR;
  for (; r + (kBatch - 1) * l.TR < count; r += kBatch * l.TR) {
    float v[kBatch][VE];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) load_vec<KIND, VE>(v[b], x + (first + r + (long)b * l.TR) * p.ld_x);
    float m = 0.0f, M = 0.0f;
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int e = 0; e < VE; ++e) m += v[b][e];
    m *= 1.0f / (kBatch * VE);
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
#pragma unroll
      for (int e = 0; e < VE; ++e) M += (v[b][e] - m) * (v[b][e] - m);
    join_moments(s, (float)(n * VE), Pair{m, M}, (float)(kBatch * VE));
    n += kBatch;
  }
  for (; r < count; r += l.TR) {
    float v[VE];
    load_vec<KIND, VE>(v, x + (first + r) * p.ld_x);
    join_moments(s, (float)(n * VE), moments<VE>(v), (float)VE);
    ++n;
  }
}
// rows of a thread in row lane tr
__device__ __forceinline__ int rows_of(int count, int tr, int TR) { return count > tr ? (count - tr + TR - 1) / TR : 0; }

// y = act(x scale + shift) of a thread's chunk over its rows
template <int KIND, int VE>
__device__ __forceinline__ void thread_apply(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                             int from, const float (&scale)[VE], const float (&shift)[VE]) {
  using E = typename ElemOf<KIND>::T;
  const E* x = static_cast<const E*>(p.x) + (long)chunk * VE;
  E* y = static_cast<E*>(p.y) + (long)chunk * VE;
  int r = l.tr + from * l.TR;
  for (; r + (kBatch - 1) * l.TR < count; r += kBatch * l.TR) {
    Raw<KIND, VE> raw[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) raw[b].load(x + (first + r + (long)b * l.TR) * p.ld_x);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      float v[VE];
      raw[b].get(v);
      forward_vec<KIND, VE>(p.act, scale, shift, v);
      store_out<KIND, VE>(y + (first + r + (long)b * l.TR) * p.ld_y, v, p.once);
    }
  }
  for (; r < count; r += l.TR) {
    float v[VE];
    load_vec<KIND, VE>(v, x + (first + r) * p.ld_x);
    forward_vec<KIND, VE>(p.act, scale, shift, v);
    store_out<KIND, VE>(y + (first + r) * p.ld_y, v, p.once);
  }
}
// gamma v + beta = x scale + shift
template <int VE>
__device__ __forceinline__ void scale_shift(const Pair& s, const float (&gamma)[VE], const float (&beta)[VE],
                                            float (&scale)[VE], float (&shift)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    scale[e] = gamma[e] * s.b;
    shift[e] = __builtin_fmaf(-s.a, scale[e], beta[e]);
  }
}

// x and dy of a thread's chunk, both kRows rows of them, under way together.
template <int KIND, int VE, bool KEPT, class F>
__device__ __forceinline__ void thread_rows(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                            int from, const Pair& s, F&& f) {
  constexpr int kRows = 2;
  using E = typename ElemOf<KIND>::T;
  const E* dy = static_cast<const E*>(p.dy) + (long)chunk * VE;
  for (int r = l.tr + from * l.TR; r < count; r += kRows * l.TR) {
    RawX<KIND, VE, KEPT> raw_x[kRows];
    Raw<KIND, VE> raw_dy[kRows];
#pragma unroll
    for (int b = 0; b < kRows; ++b)
      if (r + b * l.TR < count) {
        raw_x[b].load_at(p, first + r + (long)b * l.TR, chunk);
        raw_dy[b].load(dy + (first + r + (long)b * l.TR) * p.ld_y);
      }
#pragma unroll
    for (int b = 0; b < kRows; ++b)
      if (r + b * l.TR < count) {
        float v[VE], d[VE];
        raw_x[b].normalized(s, v);
        raw_dy[b].get(d);
        f(v, d, first + r + (long)b * l.TR);
      }
  }
}
// dz and dz v of a thread's chunk summed over its rows
template <int KIND, int VE, bool KEPT>
__device__ __forceinline__ void thread_sums(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                            int from, const Pair& s, const float (&gamma)[VE],
                                            const float (&beta)[VE], float (&be)[VE], float (&ga)[VE]) {
  thread_rows<KIND, VE, KEPT>(p, first, count, chunk, l, from, s, [&](float (&v)[VE], float (&d)[VE], long) {
    grad_vec<KIND, VE>(p.act, gamma, beta, v, d);
#pragma unroll
    for (int e = 0; e < VE; ++e) be[e] += d[e], ga[e] += d[e] * v[e];
  });
}
template <int KIND, int VE, bool KEPT>
__device__ __forceinline__ void thread_dx(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                          int from, const Pair& s, const Pair& means, const float (&gamma)[VE],
                                          const float (&beta)[VE]) {
  using E = typename ElemOf<KIND>::T;
  E* dx = static_cast<E*>(p.dx) + (long)chunk * VE;
  thread_rows<KIND, VE, KEPT>(p, first, count, chunk, l, from, s, [&](float (&v)[VE], float (&d)[VE], long row) {
    grad_vec<KIND, VE>(p.act, gamma, beta, v, d);
#pragma unroll
    for (int e = 0; e < VE; ++e) d[e] *= gamma[e];
    dx_vec<VE>(s.b, means, v, d);
    store_out<KIND, VE>(dx + row * p.ld_x, d, p.once);
  });
}

// Whole frames: grid (parts, frames, or fewer in y: strided). A thread's first kHold rows stay in registers
// between the sums and the output; what is beyond them is read again.
template <int KIND, int VE>
__global__ __launch_bounds__(kThreads) void k_norm_frames(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  constexpr int kHold = 8;
  __shared__ Pair parts[kThreads], whole[kThreads];
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0), groups = cols / p.chunks_per;
  const Lay l = lay_of(p.part, cols);
  const int chunk = c0 + min(l.tc, cols - 1);
  float gamma[VE], beta[VE];
  load_affine<KIND, VE>(p, chunk, gamma, beta);
  for (int f = blockIdx.y; f < p.frames; f += gridDim.y) {
    const Frame w = frame_of(p, f);
    const int have = l.in ? min(rows_of(w.count, l.tr, l.TR), kHold) : 0;
    // (rows past the thread's last stay zeros)
    Raw<KIND, VE> raw[kHold];
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      raw[i].zeros();
      if (i < have)
        raw[i].load(static_cast<const E*>(p.x) + (w.first + l.tr + (long)i * l.TR) * p.ld_x + (long)chunk * VE);
    }
    Pair mine = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      float v[VE];
      raw[i].get(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) mine.a += v[e];
    }
    mine.a = have ? mine.a / (float)(have * VE) : 0.0f;
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (i < have) {
        float v[VE];
        raw[i].get(v);
#pragma unroll
        for (int e = 0; e < VE; ++e) mine.b += (v[e] - mine.a) * (v[e] - mine.a);
      }
    if (l.in) thread_moments<KIND, VE>(p, w.first, w.count, chunk, l, kHold, mine);
    parts[threadIdx.x] = mine;
    __syncthreads();
    const float total = (float)w.count * (float)p.per;
    each_group<kThreads>(threadIdx.x, groups, p.lanes, [&](int q, int lane, bool in) {
      float m = 0.0f, M = 0.0f;
      const int all = l.TR * p.chunks_per;
      for (int k = lane; k < all; k += 1 << p.lanes) {
        const int tr = k / p.chunks_per;
        m += (float)rows_of(w.count, tr, l.TR) * parts[tr * p.part + q * p.chunks_per + k - tr * p.chunks_per].a;
      }
      m = sum_lanes(m, p.lanes) * VE / total;
      for (int k = lane; k < all; k += 1 << p.lanes) {
        const int tr = k / p.chunks_per;
        const Pair s = parts[tr * p.part + q * p.chunks_per + k - tr * p.chunks_per];
        M += s.b + (float)(rows_of(w.count, tr, l.TR) * VE) * (s.a - m) * (s.a - m);
      }
      M = sum_lanes(M, p.lanes);
      const Pair s = w.count ? Pair{m, deviation(M, 1.0f / total, p.eps)} : Pair{0.0f, 0.0f};
      if (in && lane == 0) {
        whole[q] = s;
        if (p.stats)
          *reinterpret_cast<Pair*>(p.stats + 2 * ((long)f * p.groups + c0 / p.chunks_per + q)) = s;
      }
    });
    __syncthreads();
    if (l.in) {
      float scale[VE], shift[VE];
      scale_shift<VE>(whole[l.tc / p.chunks_per], gamma, beta, scale, shift);
#pragma unroll
      for (int i = 0; i < kHold; ++i)
        if (i < have) {
          float v[VE];
          raw[i].get(v);
          forward_vec<KIND, VE>(p.act, scale, shift, v);
          store_vec<KIND, VE>(static_cast<E*>(p.y) + (w.first + l.tr + (long)i * l.TR) * p.ld_y + (long)chunk * VE, v);
        }
      thread_apply<KIND, VE>(p, w.first, w.count, chunk, l, kHold, scale, shift);
    }
    __syncthreads();
  }
}

// partial [gridDim.y][2][channels]
template <int KIND, int VE, bool KEPT>
__global__ __launch_bounds__(kThreads) void k_norm_frames_grad(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  constexpr int kHold = VE == 8 ? 4 : 8;  // rows whose v and dz stay in registers: 64 of these
  __shared__ Pair parts[kThreads], whole[kThreads];
  __shared__ float sums[kThreads * VE];
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0), groups = cols / p.chunks_per;
  const Lay l = lay_of(p.part, cols);
  const int chunk = c0 + min(l.tc, cols - 1);
  float gamma[VE], beta[VE], ga[VE] = {}, be[VE] = {};
  load_affine<KIND, VE>(p, chunk, gamma, beta);
  for (int f = blockIdx.y; f < p.frames; f += gridDim.y) {
    const Frame w = frame_of(p, f);
    const Pair s = *reinterpret_cast<const Pair*>(p.stats + 2 * ((long)f * p.groups + chunk / p.chunks_per));
    const int have = l.in ? min(rows_of(w.count, l.tr, l.TR), kHold) : 0;
    RawX<KIND, VE, KEPT> raw_x[kHold];
    Raw<KIND, VE> raw_dy[kHold];
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (i < have) {
        const long row = w.first + l.tr + (long)i * l.TR;
        raw_x[i].load_at(p, row, chunk);
        raw_dy[i].load(static_cast<const E*>(p.dy) + row * p.ld_y + (long)chunk * VE);
      }
    float b[VE] = {}, g[VE] = {}, v[kHold][VE], d[kHold][VE];
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (i < have) {
        raw_x[i].normalized(s, v[i]);
        raw_dy[i].get(d[i]);
        grad_vec<KIND, VE>(p.act, gamma, beta, v[i], d[i]);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          b[e] += d[i][e], g[e] += d[i][e] * v[i][e];
          d[i][e] *= gamma[e];
        }
      }
    if (l.in) thread_sums<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, kHold, s, gamma, beta, b, g);
    Pair sum = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      sum.a += gamma[e] * b[e];
      sum.b += gamma[e] * g[e];
      be[e] += b[e];
      ga[e] += g[e];
    }
    if (!p.dx) continue;
    parts[threadIdx.x] = sum;
    __syncthreads();
    const float total = fmaxf((float)w.count * (float)p.per, 1.0f);
    each_group<kThreads>(threadIdx.x, groups, p.lanes, [&](int q, int lane, bool in) {
      float x = 0.0f, y = 0.0f;
      for (int k = lane; k < l.TR * p.chunks_per; k += 1 << p.lanes) {
        const int tr = k / p.chunks_per;
        const Pair v = parts[tr * p.part + q * p.chunks_per + k - tr * p.chunks_per];
        x += v.a;
        y += v.b;
      }
      x = sum_lanes(x, p.lanes);
      y = sum_lanes(y, p.lanes);
      if (in && lane == 0) whole[q] = Pair{x / total, y / total};
    });
    __syncthreads();
    if (l.in) {
      const Pair q = whole[l.tc / p.chunks_per];
#pragma unroll
      for (int i = 0; i < kHold; ++i)
        if (i < have) {
          dx_vec<VE>(s.b, q, v[i], d[i]);
          store_vec<KIND, VE>(static_cast<E*>(p.dx) + (w.first + l.tr + (long)i * l.TR) * p.ld_x + (long)chunk * VE, d[i]);
        }
      thread_dx<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, kHold, s, q, gamma, beta);
    }
    __syncthreads();
  }
  if (!p.partial) return;
  float* out = p.partial + (long)blockIdx.y * 2 * p.channels + (long)c0 * VE;
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VE; ++e) sums[threadIdx.x * VE + e] = which ? be[e] : ga[e];
    __syncthreads();
    for (int c = threadIdx.x; c < cols * VE; c += kThreads) {
      float v = 0.0f;
      for (int m = 0; m < l.TR; ++m) v += sums[m * p.part * VE + c];
      out[which * p.channels + c] = v;
    }
  }
}

// ---- frames cut into slices --------------------------------------------------------------------
// Slice z of a frame's rows
__device__ __forceinline__ Frame slice_of(const Frame& w, int z, int slices) {
  // (the first `more` slices have a row more)
  const int each = w.count / slices, more = w.count - each * slices;
  return Frame{w.first + (long)each * z + min(z, more), each + (z < more)};
}

// Moments of each chunk over a slice: pairs [frames][slices][chunks]. Grid (parts, slices, frames).
template <int KIND, int VE>
__global__ __launch_bounds__(kThreads) void k_norm_stats(const NormArgs p) {
  __shared__ Pair parts[kThreads];
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0);
  const Lay l = lay_of(p.part, cols);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), blockIdx.y, p.slices);
    Pair mine = {0.0f, 0.0f};
    if (l.in) thread_moments<KIND, VE>(p, w.first, w.count, c0 + l.tc, l, 0, mine);
    parts[threadIdx.x] = mine;
    __syncthreads();
    if ((int)threadIdx.x < cols) {
      Pair s = parts[threadIdx.x];
      int have = rows_of(w.count, 0, l.TR);
      for (int tr = 1; tr < l.TR; ++tr) {
        const int k = rows_of(w.count, tr, l.TR);
        if (k) join_moments(s, (float)(have * VE), parts[tr * p.part + threadIdx.x], (float)(k * VE));
        have += k;
      }
      *reinterpret_cast<Pair*>(p.pairs + 2 * (((long)f * p.slices + blockIdx.y) * p.chunks + c0 + threadIdx.x)) = s;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
  for (int m = 32; m; m /= 2) v += shfl_xor_d(v, m);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// The slices' moments of each (frame, group) joined, in fp64: a block each.
template <int VE>
__global__ __launch_bounds__(kThreads) void k_norm_stats_join(const NormArgs p) {
  __shared__ double lds[4];
  const long all = (long)p.frames * p.groups;
  for (long at = blockIdx.x; at < all; at += gridDim.x) {
    const int f = (int)(at / p.groups), q = (int)(at % p.groups);
    const Frame w = frame_of(p, f);
    const float* s = p.pairs + 2 * ((long)f * p.slices * p.chunks + (long)q * p.chunks_per);
    const unsigned per = p.chunks_per, n = (unsigned)p.slices * per;
    // an entry's moments, and how many values it stands for
    auto entry = [&](unsigned k, Pair& e) {
      const unsigned z = k / per;
      e = *reinterpret_cast<const Pair*>(s + 2 * ((long)z * p.chunks + (k - z * per)));
      return (double)(slice_of(w, z, p.slices).count * VE);
    };
    // one pass, around the first part's mean (in fp64, and the parts' means lie together)
    Pair first;
    entry(0, first);
    constexpr int kUnder = 8;
    double d = 0.0, M = 0.0;
    for (unsigned k = threadIdx.x; k < n; k += kUnder * kThreads) {
      Pair e[kUnder];
      double count[kUnder];
#pragma unroll
      for (int u = 0; u < kUnder; ++u) {
        count[u] = entry(min(k + u * kThreads, n - 1), e[u]);
        if (k + u * kThreads >= n) count[u] = 0.0, e[u].b = 0.0f;
      }
#pragma unroll
      for (int u = 0; u < kUnder; ++u) {
        const double off = (double)e[u].a - first.a;
        if (count[u] > 0.0) d += count[u] * off, M += e[u].b + count[u] * off * off;
      }
    }
    const double total = (double)w.count * p.per, inv = total > 0.0 ? 1.0 / total : 0.0;
    d = block_sum(d, lds) * inv;
    M = block_sum(M, lds) - total * d * d;
    const double m = first.a + d;
    double var = M * inv;
    if (var < 0.0) var = 0.0;  // (and a NaN stays one)
    if (threadIdx.x == 0)
      *reinterpret_cast<Pair*>(p.stats + 2 * at) =
          total > 0.0 ? Pair{(float)m, (float)(1.0 / sqrt(var + (double)p.eps))} : Pair{0.0f, 0.0f};
  }
}

template <int KIND, int VE>
__global__ __launch_bounds__(kThreads) void k_norm_apply(const NormArgs p) {
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0);
  const Lay l = lay_of(p.part, cols);
  if (!l.in) return;
  const int chunk = c0 + l.tc;
  float gamma[VE], beta[VE];
  load_affine<KIND, VE>(p, chunk, gamma, beta);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), gridDim.y - 1 - blockIdx.y, gridDim.y);
    const Pair s = *reinterpret_cast<const Pair*>(p.stats + 2 * ((long)f * p.groups + chunk / p.chunks_per));
    float scale[VE], shift[VE];
    scale_shift<VE>(s, gamma, beta, scale, shift);
    thread_apply<KIND, VE>(p, w.first, w.count, chunk, l, 0, scale, shift);
  }
}

// Sums of w and w v over a slice for each chunk: pairs [frames][slices][chunks]. dgamma and dbeta over all frames
// that a block takes: partial [gridDim.z][slices][2][channels].
template <int KIND, int VE, bool KEPT>
__global__ __launch_bounds__(kThreads) void k_norm_sums(const NormArgs p) {
  __shared__ Pair parts[kThreads];
  __shared__ float sums[kThreads * VE];
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0);
  const Lay l = lay_of(p.part, cols);
  const int chunk = c0 + min(l.tc, cols - 1);
  float gamma[VE], beta[VE], ga[VE] = {}, be[VE] = {};
  load_affine<KIND, VE>(p, chunk, gamma, beta);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), blockIdx.y, p.slices);
    const Pair s = *reinterpret_cast<const Pair*>(p.stats + 2 * ((long)f * p.groups + chunk / p.chunks_per));
    float b[VE] = {}, g[VE] = {};
    if (l.in) thread_sums<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, 0, s, gamma, beta, b, g);
    Pair sum = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      sum.a += gamma[e] * b[e];
      sum.b += gamma[e] * g[e];
      be[e] += b[e];
      ga[e] += g[e];
    }
    if (!p.dx) continue;
    __syncthreads();
    parts[threadIdx.x] = sum;
    __syncthreads();
    if ((int)threadIdx.x < cols) {
      for (int tr = 1; tr < l.TR; ++tr) {
        const Pair q = parts[tr * p.part + threadIdx.x];
        sum.a += q.a;
        sum.b += q.b;
      }
      *reinterpret_cast<Pair*>(p.pairs + 2 * (((long)f * p.slices + blockIdx.y) * p.chunks + chunk)) = sum;
    }
  }
  if (!p.partial) return;
  float* out = p.partial + ((long)blockIdx.z * p.slices + blockIdx.y) * 2 * p.channels + (long)c0 * VE;
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VE; ++e) sums[threadIdx.x * VE + e] = which ? be[e] : ga[e];
    __syncthreads();
    for (int c = threadIdx.x; c < cols * VE; c += kThreads) {
      float v = 0.0f;
      for (int m = 0; m < l.TR; ++m) v += sums[m * p.part * VE + c];
      out[which * p.channels + c] = v;
    }
  }
}

// The slices' (or blocks') sums joined in fp64. The first `group_blocks` blocks: means of w and w v for each
// (frame, group), a block each. The others: dgamma and dbeta of `parts` partial sums, 16 channels a block, 16
// threads a channel.
template <int KIND>
__global__ __launch_bounds__(kThreads) void k_norm_sums_join(const NormArgs p, int group_blocks, long parts) {
  __shared__ double lds[2][kThreads];
  if ((int)blockIdx.x < group_blocks) {
    const long all = (long)p.frames * p.groups;
    for (long at = blockIdx.x; at < all; at += group_blocks) {
      const int f = (int)(at / p.groups), q = (int)(at % p.groups);
      const float* s = p.pairs + 2 * ((long)f * p.slices * p.chunks + (long)q * p.chunks_per);
      double a = 0.0, b = 0.0;
      const unsigned per = p.chunks_per, n = (unsigned)p.slices * per;
#pragma unroll 4
      for (unsigned k = threadIdx.x; k < n; k += kThreads) {
        const unsigned z = k / per;
        const Pair e = *reinterpret_cast<const Pair*>(s + 2 * ((long)z * p.chunks + (k - z * per)));
        a += e.a;
        b += e.b;
      }
      a = block_sum(a, lds[0]);
      b = block_sum(b, lds[0]);
      const double total = (double)frame_of(p, f).count * p.per, inv = total > 0.0 ? 1.0 / total : 0.0;
      if (threadIdx.x == 0) *reinterpret_cast<Pair*>(p.sums + 2 * at) = Pair{(float)(a * inv), (float)(b * inv)};
    }
    return;
  }
  const int slot = threadIdx.x % 16, share = threadIdx.x / 16;
  const long c = (long)(blockIdx.x - group_blocks) * 16 + slot;
  double a = 0.0, b = 0.0;
  if (c < p.channels) {
    const long end = parts * (share + 1) / 16;
    const float* s = p.partial + c;
    long k = parts * share / 16;
    for (; k + 8 <= end; k += 8) {
      float x[8], y[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        x[u] = s[(k + u) * 2 * p.channels];
        y[u] = s[((k + u) * 2 + 1) * p.channels];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) b += x[u], a += y[u];
    }
    for (; k < end; ++k) {
      b += s[k * 2 * p.channels];
      a += s[(k * 2 + 1) * p.channels];
    }
  }
  lds[0][threadIdx.x] = a;
  lds[1][threadIdx.x] = b;
  __syncthreads();
  if (share || c >= p.channels) return;
  for (int m = 1; m < 16; ++m) a += lds[0][m * 16 + slot], b += lds[1][m * 16 + slot];
  using E = typename ElemOf<KIND>::T;
  if (p.dgamma) static_cast<E*>(p.dgamma)[c] = from_f32<KIND>((float)b);
  if (p.dbeta) static_cast<E*>(p.dbeta)[c] = from_f32<KIND>((float)a);
}

template <int KIND, int VE, bool KEPT>
__global__ __launch_bounds__(kThreads) void k_norm_dx(const NormArgs p) {
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0);
  const Lay l = lay_of(p.part, cols);
  if (!l.in) return;
  const int chunk = c0 + l.tc;
  float gamma[VE], beta[VE];
  load_affine<KIND, VE>(p, chunk, gamma, beta);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), gridDim.y - 1 - blockIdx.y, gridDim.y);
    const long at = 2 * ((long)f * p.groups + chunk / p.chunks_per);
    thread_dx<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, 0, *reinterpret_cast<const Pair*>(p.stats + at),
                              *reinterpret_cast<const Pair*>(p.sums + at), gamma, beta);
  }
}

// ---- launches ---------------------------------------------------------------------------------
template <class F>
void by_vec(int vec, F&& f) {
  if constexpr (ELEM_KIND != kF32)
    if (vec == 8) return f(std::integral_constant<int, 8>{});
  if constexpr (ELEM_KIND == kF32)
    if (vec == 4) return f(std::integral_constant<int, 4>{});
  if (vec == 2) return f(std::integral_constant<int, 2>{});
  f(std::integral_constant<int, 1>{});
}
// threads of a row, chunks of a thread, and whether groups are lanes
template <class F>
void by_row(const NormArgs& p, F&& f) {
  using std::integral_constant;
  auto lanes = [&](auto t, auto c) {
    if (p.by_lanes)
      f(t, c, std::true_type{});
    else
      f(t, c, std::false_type{});
  };
  if (p.chunks <= 16)
    lanes(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (p.chunks <= 64)
    lanes(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (p.chunks <= 256)
    lanes(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (p.chunks <= 512)
    lanes(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else
    lanes(integral_constant<int, 256>{}, integral_constant<int, 4>{});
}
size_t row_lds(const NormArgs& p, int T, int VE, bool grad) {
  const size_t parts = (size_t)(kThreads / T) * (p.chunks + p.groups) * sizeof(Pair);
  return grad ? std::max(parts, (size_t)kThreads * VE * sizeof(float)) : parts;
}
dim3 frame_grid(const NormArgs& p) { return dim3(p.parts, std::min(p.frames, p.blocks)); }
dim3 out_grid(const NormArgs& p) { return dim3(p.parts, p.out_slices, std::min(p.frames, 65535)); }
dim3 slice_grid(const NormArgs& p, int most) { return dim3(p.parts, p.slices, std::min(p.frames, most)); }
constexpr int kGrid = 65535;

}  // namespace

template <>
void norm_launch<ELEM_KIND>(hipStream_t st, const NormArgs& p) {
  constexpr int KIND = ELEM_KIND;
  by_vec(p.vec, [&](auto ve) {
    constexpr int VE = decltype(ve)::value;
    if (p.form == kNormRows) {
      by_row(p, [&](auto t, auto c, auto lanes) {
        constexpr int T = decltype(t)::value, C = decltype(c)::value;
        constexpr bool LANES = decltype(lanes)::value;
        hipLaunchKernelGGL((k_norm_rows<KIND, VE, T, C, LANES>), dim3(p.blocks), dim3(kThreads),
                           LANES ? 0 : row_lds(p, T, VE, false), st, p);
      });
    } else if (p.form == kNormFrames) {
      hipLaunchKernelGGL((k_norm_frames<KIND, VE>), frame_grid(p), dim3(kThreads), 0, st, p);
    } else {
      hipLaunchKernelGGL((k_norm_stats<KIND, VE>), slice_grid(p, kGrid), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
      const long all = (long)p.frames * p.groups;
      hipLaunchKernelGGL((k_norm_stats_join<VE>), dim3((unsigned)std::min(all, 1L << 20)), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
      hipLaunchKernelGGL((k_norm_apply<KIND, VE>), out_grid(p), dim3(kThreads), 0, st, p);
    }
  });
  DPAMD_LAUNCH_CHECK();
}

template <>
void norm_grad_launch<ELEM_KIND>(hipStream_t st, const NormArgs& p) {
  constexpr int KIND = ELEM_KIND;
  const int channel_blocks = p.dgamma || p.dbeta ? (p.channels + 15) / 16 : 0;
  auto launch = [&](auto ve, auto kept) {
    constexpr int VE = decltype(ve)::value;
    constexpr bool KEPT = decltype(kept)::value;
    int group_blocks = 0;
    long parts = 0;
    if (p.form == kNormRows) {
      by_row(p, [&](auto t, auto c, auto lanes) {
        constexpr int T = decltype(t)::value, C = decltype(c)::value;
        constexpr bool LANES = decltype(lanes)::value;
        hipLaunchKernelGGL((k_norm_rows_grad<KIND, VE, T, C, LANES, KEPT>), dim3(p.blocks), dim3(kThreads),
                           row_lds(p, T, VE, true), st, p);
      });
      parts = p.blocks;
    } else if (p.form == kNormFrames) {
      hipLaunchKernelGGL((k_norm_frames_grad<KIND, VE, KEPT>), frame_grid(p), dim3(kThreads), 0, st, p);
      parts = frame_grid(p).y;
    } else {
      hipLaunchKernelGGL((k_norm_sums<KIND, VE, KEPT>), slice_grid(p, p.blocks), dim3(kThreads), 0, st, p);
      parts = (long)slice_grid(p, p.blocks).z * p.slices;
      if (p.dx) group_blocks = (int)std::min((long)p.frames * p.groups, 1L << 20);
    }
    DPAMD_LAUNCH_CHECK();
    if (group_blocks + channel_blocks) {
      hipLaunchKernelGGL((k_norm_sums_join<KIND>), dim3(group_blocks + channel_blocks), dim3(kThreads), 0, st, p,
                         group_blocks, parts);
      DPAMD_LAUNCH_CHECK();
    }
    if (p.form == kNormSlices && p.dx) {
      hipLaunchKernelGGL((k_norm_dx<KIND, VE, KEPT>), out_grid(p), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
    }
  };
  by_vec(p.vec, [&](auto ve) {
    if (p.kept)
      launch(ve, std::true_type{});
    else
      launch(ve, std::false_type{});
  });
}

}  // namespace dpamd
