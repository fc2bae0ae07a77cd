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

template <int KIND, int VE>
__device__ __forceinline__ void load_vec(float (&v)[VE], const typename ElemOf<KIND>::T* p) {
  struct Some {
    typename ElemOf<KIND>::T v[VE];
  } s;
  __builtin_memcpy(&s, p, sizeof(s));  // (the hardware takes addresses of any alignment)
#pragma unroll
  for (int e = 0; e < VE; ++e) v[e] = to_f32<KIND>(s.v[e]);
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
// x at (row, chunk): the matrix's, or what the checkpoint restores
template <int KIND, int VE, bool KEPT>
__device__ __forceinline__ void load_x(const NormArgs& p, float (&v)[VE], long row, int chunk) {
  if constexpr (KEPT) {
    struct Some {
      signed char v[VE];
    } s;
    __builtin_memcpy(&s, p.kept + row * p.wide + chunk * VE, sizeof(s));
    const int field = p.kept[p.rows * p.wide + row * (p.wide / 32) + chunk * VE / 32];
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = restore_one(s.v[e], field);
  } else {
    load_vec<KIND, VE>(v, static_cast<const typename ElemOf<KIND>::T*>(p.x) + row * p.ld_x + (long)chunk * VE);
  }
}
template <int KIND, int VE>
__device__ __forceinline__ void load_affine(const NormArgs& p, int chunk, float (&gamma)[VE], float (&beta)[VE]) {
  using T = typename ElemOf<KIND>::T;
#pragma unroll
  for (int e = 0; e < VE; ++e) gamma[e] = 1.0f, beta[e] = 0.0f;
  if (p.gamma) load_vec<KIND, VE>(gamma, static_cast<const T*>(p.gamma) + (long)chunk * VE);
  if (p.beta) load_vec<KIND, VE>(beta, static_cast<const T*>(p.beta) + (long)chunk * VE);
}

// act and its derivative over a thread's values (one uniform branch for all of them)
template <int VE>
__device__ __forceinline__ void activate_vec(int act, const float (&z)[VE], float (&a)[VE], float (&da)[VE]) {
  auto all = [&](auto k) {
#pragma unroll
    for (int e = 0; e < VE; ++e) activate<decltype(k)::value>(z[e], a[e], da[e]);
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
template <int VE>
__device__ __forceinline__ void forward_vec(int act, float m, float r, const float (&gamma)[VE],
                                            const float (&beta)[VE], float (&v)[VE]) {
  float z[VE], da[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) z[e] = gamma[e] * ((v[e] - m) * r) + beta[e];
  activate_vec<VE>(act, z, v, da);
}
// x -> v and dy -> dz
template <int VE>
__device__ __forceinline__ void grad_vec(int act, float m, float r, const float (&gamma)[VE], const float (&beta)[VE],
                                         float (&x)[VE], float (&dy)[VE]) {
  float z[VE], a[VE], da[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    x[e] = (x[e] - m) * r;
    z[e] = gamma[e] * x[e] + beta[e];
  }
  activate_vec<VE>(act, z, a, da);
#pragma unroll
  for (int e = 0; e < VE; ++e) dy[e] *= da[e];
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

__device__ __forceinline__ float sum_lanes(float v, int log_lanes) {
  for (int m = 0; m < log_lanes; ++m) v += __shfl_xor(v, 1 << m, kWave);
  return v;
}
__device__ __forceinline__ float deviation(float M, float n, float eps) {
  return 1.0f / sqrtf(M / n + eps);
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
// T threads a row, C chunks of VE channels a thread (at neighbouring places for neighbouring threads). Parts
// of a row in LDS: a pair for each chunk, then one for each group.
template <int KIND, int VE, int T, int C>
__global__ __launch_bounds__(kThreads) void k_norm_rows(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  extern __shared__ __align__(16) char lds[];
  constexpr int R = kThreads / T;
  const int t = threadIdx.x % T, mine = threadIdx.x / T;
  Pair* parts = reinterpret_cast<Pair*>(lds) + (size_t)mine * (p.chunks + p.groups);
  Pair* whole = parts + p.chunks;
  for (long row0 = (long)blockIdx.x * R; row0 < p.rows; row0 += (long)gridDim.x * R) {
    const bool there = row0 + mine < p.rows;
    const long row = there ? row0 + mine : p.rows - 1;
    float v[C][VE];
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (k * T + t < p.chunks) load_x<KIND, VE, false>(p, v[k], row, k * T + t);
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (k * T + t < p.chunks) parts[k * T + t] = moments<VE>(v[k]);
    row_sync<T>();
    each_group<T>(t, p.groups, p.lanes, [&](int q, int lane, bool in) {
      const Pair* s = parts + q * p.chunks_per;
      float m = 0.0f, M = 0.0f;
      for (int k = lane; k < p.chunks_per; k += 1 << p.lanes) m += s[k].a;
      m = sum_lanes(m, p.lanes) / (float)p.chunks_per;
      for (int k = lane; k < p.chunks_per; k += 1 << p.lanes) M += s[k].b + VE * (s[k].a - m) * (s[k].a - m);
      const float r = deviation(sum_lanes(M, p.lanes), (float)p.per, p.eps);
      if (in && lane == 0) {
        whole[q] = Pair{m, r};
        if (p.stats && there) *reinterpret_cast<Pair*>(p.stats + 2 * (row * p.groups + q)) = Pair{m, r};
      }
    });
    row_sync<T>();
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int chunk = k * T + t;
      if (chunk >= p.chunks) continue;
      const Pair s = whole[chunk / p.chunks_per];
      float gamma[VE], beta[VE];
      load_affine<KIND, VE>(p, chunk, gamma, beta);
      forward_vec<VE>(p.act, s.a, s.b, gamma, beta, v[k]);
      if (there) store_vec<KIND, VE>(static_cast<E*>(p.y) + row * p.ld_y + (long)chunk * VE, v[k]);
    }
    row_sync<T>();  // (the next row's parts go where these are read)
  }
}

// Its gradients: dgamma and dbeta of a thread's channels are summed over all rows that its block takes, and
// then over the block's row lanes; partial [blocks][2][channels].
template <int KIND, int VE, int T, int C, bool KEPT>
__global__ __launch_bounds__(kThreads) void k_norm_rows_grad(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  extern __shared__ __align__(16) char lds[];
  constexpr int R = kThreads / T;
  const int t = threadIdx.x % T, mine = threadIdx.x / T;
  Pair* parts = reinterpret_cast<Pair*>(lds) + (size_t)mine * (p.chunks + p.groups);
  Pair* whole = parts + p.chunks;
  float ga[C][VE] = {}, be[C][VE] = {};
  for (long row0 = (long)blockIdx.x * R; row0 < p.rows; row0 += (long)gridDim.x * R) {
    const bool there = row0 + mine < p.rows;
    const long row = there ? row0 + mine : p.rows - 1;
    float v[C][VE], dz[C][VE], r[C];
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (k * T + t < p.chunks) {
        load_x<KIND, VE, KEPT>(p, v[k], row, k * T + t);
        load_vec<KIND, VE>(dz[k], static_cast<const E*>(p.dy) + row * p.ld_y + (long)(k * T + t) * VE);
      }
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int chunk = k * T + t;
      if (chunk >= p.chunks) continue;
      const Pair s = *reinterpret_cast<const Pair*>(p.stats + 2 * (row * p.groups + chunk / p.chunks_per));
      r[k] = s.b;
      float gamma[VE], beta[VE];
      load_affine<KIND, VE>(p, chunk, gamma, beta);
      grad_vec<VE>(p.act, s.a, s.b, gamma, beta, v[k], dz[k]);
      Pair sum = {0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const float w = gamma[e] * dz[k][e];
        sum.a += w;
        sum.b += w * v[k][e];
        if (there) {
          be[k][e] += dz[k][e];
          ga[k][e] += dz[k][e] * v[k][e];
        }
      }
      parts[chunk] = sum;
    }
    row_sync<T>();
    each_group<T>(t, p.groups, p.lanes, [&](int q, int lane, bool in) {
      const Pair* s = parts + q * p.chunks_per;
      float a = 0.0f, b = 0.0f;
      for (int k = lane; k < p.chunks_per; k += 1 << p.lanes) a += s[k].a, b += s[k].b;
      a = sum_lanes(a, p.lanes) / (float)p.per;
      b = sum_lanes(b, p.lanes) / (float)p.per;
      if (in && lane == 0) whole[q] = Pair{a, b};
    });
    row_sync<T>();
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const int chunk = k * T + t;
      if (chunk >= p.chunks) continue;
      const Pair s = whole[chunk / p.chunks_per];
      float gamma[VE], beta[VE];
      load_affine<KIND, VE>(p, chunk, gamma, beta);
#pragma unroll
      for (int e = 0; e < VE; ++e) dz[k][e] = r[k] * (gamma[e] * dz[k][e] - s.a - v[k][e] * s.b);
      if (there && p.dx) store_vec<KIND, VE>(static_cast<E*>(p.dx) + row * p.ld_x + (long)chunk * VE, dz[k]);
    }
    row_sync<T>();
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

// Moments of a thread's chunk over rows first + tr, + TR, ... below first + count; n: their number
template <int KIND, int VE>
__device__ __forceinline__ Pair thread_moments(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                               int& n) {
  Pair s = {0.0f, 0.0f};
  n = 0;
  int r = l.tr;
  for (; r + (kBatch - 1) * l.TR < count; r += kBatch * l.TR) {
    float v[kBatch][VE];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) load_x<KIND, VE, false>(p, v[b], first + r + (long)b * l.TR, chunk);
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
    load_x<KIND, VE, false>(p, v, first + r, chunk);
    join_moments(s, (float)(n * VE), moments<VE>(v), (float)VE);
    ++n;
  }
  return s;
}
// rows of a thread in row lane tr
__device__ __forceinline__ int rows_of(int count, int tr, int TR) { return count > tr ? (count - tr + TR - 1) / TR : 0; }

// y of a thread's chunk over its rows
template <int KIND, int VE>
__device__ __forceinline__ void thread_apply(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                             const Pair& s) {
  using E = typename ElemOf<KIND>::T;
  float gamma[VE], beta[VE];
  load_affine<KIND, VE>(p, chunk, gamma, beta);
  E* y = static_cast<E*>(p.y) + (long)chunk * VE;
  int r = l.tr;
  for (; r + (kBatch - 1) * l.TR < count; r += kBatch * l.TR) {
    float v[kBatch][VE];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) load_x<KIND, VE, false>(p, v[b], first + r + (long)b * l.TR, chunk);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      forward_vec<VE>(p.act, s.a, s.b, gamma, beta, v[b]);
      store_vec<KIND, VE>(y + (first + r + (long)b * l.TR) * p.ld_y, v[b]);
    }
  }
  for (; r < count; r += l.TR) {
    float v[VE];
    load_x<KIND, VE, false>(p, v, first + r, chunk);
    forward_vec<VE>(p.act, s.a, s.b, gamma, beta, v);
    store_vec<KIND, VE>(y + (first + r) * p.ld_y, v);
  }
}

// dz and dz v of a thread's chunk summed over its rows
template <int KIND, int VE, bool KEPT>
__device__ __forceinline__ void thread_sums(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                            const Pair& s, const float (&gamma)[VE], const float (&beta)[VE],
                                            float (&be)[VE], float (&ga)[VE]) {
  using E = typename ElemOf<KIND>::T;
  const E* dy = static_cast<const E*>(p.dy) + (long)chunk * VE;
  auto add = [&](float (&v)[VE], float (&d)[VE]) {
    grad_vec<VE>(p.act, s.a, s.b, gamma, beta, v, d);
#pragma unroll
    for (int e = 0; e < VE; ++e) be[e] += d[e], ga[e] += d[e] * v[e];
  };
  int r = l.tr;
  for (; r + l.TR < count; r += 2 * l.TR) {
    float v[2][VE], d[2][VE];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      load_x<KIND, VE, KEPT>(p, v[b], first + r + (long)b * l.TR, chunk);
      load_vec<KIND, VE>(d[b], dy + (first + r + (long)b * l.TR) * p.ld_y);
    }
    add(v[0], d[0]);
    add(v[1], d[1]);
  }
  if (r < count) {
    float v[VE], d[VE];
    load_x<KIND, VE, KEPT>(p, v, first + r, chunk);
    load_vec<KIND, VE>(d, dy + (first + r) * p.ld_y);
    add(v, d);
  }
}
template <int KIND, int VE, bool KEPT>
__device__ __forceinline__ void thread_dx(const NormArgs& p, long first, int count, int chunk, const Lay& l,
                                          const Pair& s, const Pair& sums, const float (&gamma)[VE],
                                          const float (&beta)[VE]) {
  using E = typename ElemOf<KIND>::T;
  const E* dy = static_cast<const E*>(p.dy) + (long)chunk * VE;
  E* dx = static_cast<E*>(p.dx) + (long)chunk * VE;
  auto put = [&](float (&v)[VE], float (&d)[VE], long row) {
    grad_vec<VE>(p.act, s.a, s.b, gamma, beta, v, d);
#pragma unroll
    for (int e = 0; e < VE; ++e) d[e] = s.b * (gamma[e] * d[e] - sums.a - v[e] * sums.b);
    store_vec<KIND, VE>(dx + row * p.ld_x, d);
  };
  int r = l.tr;
  for (; r + l.TR < count; r += 2 * l.TR) {
    float v[2][VE], d[2][VE];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      load_x<KIND, VE, KEPT>(p, v[b], first + r + (long)b * l.TR, chunk);
      load_vec<KIND, VE>(d[b], dy + (first + r + (long)b * l.TR) * p.ld_y);
    }
    put(v[0], d[0], first + r);
    put(v[1], d[1], first + r + l.TR);
  }
  if (r < count) {
    float v[VE], d[VE];
    load_x<KIND, VE, KEPT>(p, v, first + r, chunk);
    load_vec<KIND, VE>(d, dy + (first + r) * p.ld_y);
    put(v, d, first + r);
  }
}

// Whole frames: grid (parts, frames, or fewer in y: strided).
template <int KIND, int VE>
__global__ __launch_bounds__(kThreads) void k_norm_frames(const NormArgs p) {
  __shared__ Pair parts[kThreads], whole[kThreads];
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0), groups = cols / p.chunks_per;
  const Lay l = lay_of(p.part, cols);
  const int chunk = c0 + min(l.tc, cols - 1);
  for (int f = blockIdx.y; f < p.frames; f += gridDim.y) {
    const Frame w = frame_of(p, f);
    int n = 0;
    const Pair mine = l.in ? thread_moments<KIND, VE>(p, w.first, w.count, chunk, l, n) : Pair{0.0f, 0.0f};
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
      const Pair s = w.count ? Pair{m, deviation(M, total, p.eps)} : Pair{0.0f, 0.0f};
      if (in && lane == 0) {
        whole[q] = s;
        if (p.stats)
          *reinterpret_cast<Pair*>(p.stats + 2 * ((long)f * p.groups + c0 / p.chunks_per + q)) = s;
      }
    });
    __syncthreads();
    if (l.in) thread_apply<KIND, VE>(p, w.first, w.count, chunk, l, whole[l.tc / p.chunks_per]);
    __syncthreads();
  }
}

// partial [gridDim.y][2][channels]
template <int KIND, int VE, bool KEPT>
__global__ __launch_bounds__(kThreads) void k_norm_frames_grad(const NormArgs p) {
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
    float b[VE] = {}, g[VE] = {};
    if (l.in) thread_sums<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, s, gamma, beta, b, g);
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
    if (l.in)
      thread_dx<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, s, whole[l.tc / p.chunks_per], gamma, beta);
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
  const long a = (long)w.count * z / slices, b = (long)w.count * (z + 1) / slices;
  return Frame{w.first + a, (int)(b - a)};
}

// Moments of each chunk over a slice: pairs [frames][slices][chunks]. Grid (parts, slices, frames).
template <int KIND, int VE>
__global__ __launch_bounds__(kThreads) void k_norm_stats(const NormArgs p) {
  __shared__ Pair parts[kThreads];
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0);
  const Lay l = lay_of(p.part, cols);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), blockIdx.y, p.slices);
    int n = 0;
    parts[threadIdx.x] =
        l.in ? thread_moments<KIND, VE>(p, w.first, w.count, c0 + l.tc, l, n) : Pair{0.0f, 0.0f};
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
    const long n = (long)p.slices * p.chunks_per;
    auto entry = [&](long k, int& rows) {
      const int z = (int)(k / p.chunks_per);
      rows = slice_of(w, z, p.slices).count;
      return *reinterpret_cast<const Pair*>(s + 2 * ((long)z * p.chunks + k % p.chunks_per));
    };
    double m = 0.0, M = 0.0;
    for (long k = threadIdx.x; k < n; k += kThreads) {
      int rows;
      const Pair e = entry(k, rows);
      m += (double)rows * VE * e.a;
    }
    const double total = (double)w.count * p.per;
    m = block_sum(m, lds) / (total > 0.0 ? total : 1.0);
    for (long k = threadIdx.x; k < n; k += kThreads) {
      int rows;
      const Pair e = entry(k, rows);
      M += e.b + (double)rows * VE * (e.a - m) * (e.a - m);
    }
    M = block_sum(M, lds);
    if (threadIdx.x == 0)
      *reinterpret_cast<Pair*>(p.stats + 2 * at) =
          total > 0.0 ? Pair{(float)m, (float)(1.0 / sqrt(M / total + (double)p.eps))} : Pair{0.0f, 0.0f};
  }
}

template <int KIND, int VE>
__global__ __launch_bounds__(kThreads) void k_norm_apply(const NormArgs p) {
  const int c0 = blockIdx.x * p.part, cols = min(p.part, p.chunks - c0);
  const Lay l = lay_of(p.part, cols);
  if (!l.in) return;
  const int chunk = c0 + l.tc;
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), blockIdx.y, p.slices);
    const Pair s = *reinterpret_cast<const Pair*>(p.stats + 2 * ((long)f * p.groups + chunk / p.chunks_per));
    thread_apply<KIND, VE>(p, w.first, w.count, chunk, l, s);
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
    if (l.in) thread_sums<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, s, gamma, beta, b, g);
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
      const long n = (long)p.slices * p.chunks_per;
      for (long k = threadIdx.x; k < n; k += kThreads) {
        const Pair e = *reinterpret_cast<const Pair*>(s + 2 * (k / p.chunks_per * p.chunks + k % p.chunks_per));
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
  if (c < p.channels)
    for (long k = parts * share / 16; k < parts * (share + 1) / 16; ++k) {
      b += p.partial[k * 2 * p.channels + c];
      a += p.partial[(k * 2 + 1) * p.channels + c];
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
    const Frame w = slice_of(frame_of(p, f), blockIdx.y, p.slices);
    const long at = 2 * ((long)f * p.groups + chunk / p.chunks_per);
    thread_dx<KIND, VE, KEPT>(p, w.first, w.count, chunk, l, *reinterpret_cast<const Pair*>(p.stats + at),
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
// threads of a row and chunks of a thread
template <class F>
void by_row(int chunks, F&& f) {
  using std::integral_constant;
  if (chunks <= 16)
    f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (chunks <= 64)
    f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (chunks <= 256)
    f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
  else
    f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
}
size_t row_lds(const NormArgs& p, int T, int VE, bool grad) {
  const size_t parts = (size_t)(kThreads / T) * (p.chunks + p.groups) * sizeof(Pair);
  return grad ? std::max(parts, (size_t)kThreads * VE * sizeof(float)) : parts;
}
dim3 frame_grid(const NormArgs& p) { return dim3(p.parts, std::min(p.frames, p.blocks)); }
dim3 slice_grid(const NormArgs& p, int most) { return dim3(p.parts, p.slices, std::min(p.frames, most)); }
constexpr int kGrid = 65535;

}  // namespace

template <>
void norm_launch<ELEM_KIND>(hipStream_t st, const NormArgs& p) {
  constexpr int KIND = ELEM_KIND;
  by_vec(p.vec, [&](auto ve) {
    constexpr int VE = decltype(ve)::value;
    if (p.form == kNormRows) {
      by_row(p.chunks, [&](auto t, auto c) {
        constexpr int T = decltype(t)::value, C = decltype(c)::value;
        const long want = (p.rows + kThreads / T - 1) / (kThreads / T);
        hipLaunchKernelGGL((k_norm_rows<KIND, VE, T, C>), dim3((unsigned)std::min(want, 1L << 20)), dim3(kThreads),
                           row_lds(p, T, VE, false), st, p);
      });
    } else if (p.form == kNormFrames) {
      hipLaunchKernelGGL((k_norm_frames<KIND, VE>), frame_grid(p), dim3(kThreads), 0, st, p);
    } else {
      hipLaunchKernelGGL((k_norm_stats<KIND, VE>), slice_grid(p, kGrid), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
      const long all = (long)p.frames * p.groups;
      hipLaunchKernelGGL((k_norm_stats_join<VE>), dim3((unsigned)std::min(all, 1L << 20)), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
      hipLaunchKernelGGL((k_norm_apply<KIND, VE>), slice_grid(p, kGrid), dim3(kThreads), 0, st, p);
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
      by_row(p.chunks, [&](auto t, auto c) {
        constexpr int T = decltype(t)::value, C = decltype(c)::value;
        hipLaunchKernelGGL((k_norm_rows_grad<KIND, VE, T, C, KEPT>), dim3(p.blocks), dim3(kThreads),
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
      hipLaunchKernelGGL((k_norm_dx<KIND, VE, KEPT>), slice_grid(p, kGrid), dim3(kThreads), 0, st, p);
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
