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
// fp64. Sums have an order that sizes, row lengths and the card's compute units fix.
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

// ---- a thread's channels -----------------------------------------------------------------
// A thread takes VE neighbouring channels, 16 bytes, from c on; `count` of them are there (VE but at the
// end of a row). Where groups are multiples of VE (not GEN) all of them are of one group, and are one entry of
// the sums; else (GEN: groups of 5, of 47) each channel is an entry of its own, and knows its group. (With vectors as
// narrow as a common divisor of groups and 16 bytes instead, odd groups went element by element:
// 113,120 x 235 in groups of 5, bf16, with its gradients 491 us, so 147.) With groups of VE channels or more (GEN ==
// kPieces, every row a frame) a thread's channels are of two groups at most, and are two entries.
constexpr int kPieces = 2;
struct Cols {
  int c, count;
};
template <int VE, int GEN>
constexpr int entries_of() {
  return GEN == kPieces ? 2 : GEN ? VE : 1;
}
// channels from c on to the end of its group
__device__ __forceinline__ int left_of(const Cols& x, int per) { return per - x.c % per; }
// what each entry has: a mean and a deviation, two sums, ...
template <int VE, int GEN>
struct Entries {
  static constexpr int N = entries_of<VE, GEN>();
  Pair e[N];
  __device__ __forceinline__ const Pair& of(int channel) const { return e[GEN ? channel : 0]; }
};
template <int VE>
struct Entries<VE, kPieces> {
  static constexpr int N = 2;
  Pair e[N];
  int left;  // channels of the first
  __device__ __forceinline__ Pair of(int channel) const {
    return Pair{channel < left ? e[0].a : e[1].a, channel < left ? e[0].b : e[1].b};
  }
};
// Nothing that takes the means is moved ahead of this: x - m beside each load would have every load waited for by itself
// (64 ragged frames of 12,288 x 1600 in fp32, gradients 68 us, and 58 so).
template <int VE, int GEN>
__device__ __forceinline__ void hold_back(Entries<VE, GEN>& s) {
#pragma unroll
  for (int i = 0; i < Entries<VE, GEN>::N; ++i) asm volatile("" : "+v"(s.e[i].a));
}
// Pairs of the entries' groups, from an array of one for each group.
template <int VE, int GEN>
__device__ __forceinline__ Entries<VE, GEN> of_groups(const Pair* groups, const Cols& x, int per) {
  Entries<VE, GEN> s;
  if constexpr (GEN == kPieces) {
    const int q = x.c / per;
    s.left = (q + 1) * per - x.c;
    s.e[0] = groups[q];
    s.e[1] = s.left < x.count ? groups[q + 1] : s.e[0];
  } else if constexpr (GEN) {
    // (one division: the group's channels are counted from it)
    int q = x.c / per, left = (q + 1) * per - x.c;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      s.e[e] = e < x.count ? groups[q] : Pair{0.0f, 0.0f};
      if (--left == 0) ++q, left = per;
    }
  } else {
    s.e[0] = groups[x.c / per];
  }
  return s;
}

// VE elements as they lie in memory: what is loaded ahead, or kept for long, takes no more registers than that
// (held in words: single elements of 16 or 8 bits would take a register each).
template <int KIND, int VE>
struct Raw {
  using E = typename ElemOf<KIND>::T;
  static constexpr int kBytes = VE * sizeof(E), kWords = (kBytes + 3) / 4;
  unsigned w[kWords];
  __device__ __forceinline__ void zeros() {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = 0;
  }
  // the elements from p on; those past x's count: zeros
  template <int GEN>
  __device__ __forceinline__ void load(const E* p, const Cols& x) {
    if constexpr (kBytes == 2) {
      w[0] = *p;
    } else if (!GEN || x.count == VE) {
      __builtin_memcpy(w, p, kBytes);  // (the hardware takes addresses of any alignment)
    } else {
      zeros();
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (e < x.count) {
          if constexpr (KIND == kF32)
            w[e] = __builtin_bit_cast(unsigned, p[e]);
          else
            w[e / 2] |= (unsigned)p[e] << (16 * (e % 2));
        }
    }
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
// x or its checkpoint, and v = (x - m) r from it. (As x r - m r, one instruction a value, it is off by the rounding of
// m r, which is not small beside v where a group has hardly any deviation: three values of 16,384 each gave 0.2.)
template <int KIND, int VE, int GEN, bool KEPT>
struct RawX : Raw<KIND, VE> {
  __device__ __forceinline__ void load_at(const NormArgs& p, long row, const Cols& x) {
    this->template load<GEN>(static_cast<const typename ElemOf<KIND>::T*>(p.x) + row * p.ld_x + x.c, x);
  }
  __device__ __forceinline__ void normalized(const Entries<VE, GEN>& s, float (&out)[VE]) const {
    this->get(out);
#pragma unroll
    for (int e = 0; e < VE; ++e) out[e] = (out[e] - s.of(e).a) * s.of(e).b;
  }
};
template <int KIND, int VE, int GEN>
struct RawX<KIND, VE, GEN, true> {
  static constexpr int kWords = (VE + 3) / 4;
  unsigned w[kWords];
  unsigned char field, second;  // (GEN: the last elements may be of the next 32)
  unsigned char split;          // elements of the first
  __device__ __forceinline__ void load_at(const NormArgs& p, long row, const Cols& x) {
    const unsigned char* at = p.kept + row * p.wide;
    if constexpr (VE == 1) {
      w[0] = at[x.c];
    } else if constexpr (GEN) {
      // (from any channel on, but not past the row's end: there the last ones, shifted)
      const int c = min(x.c, p.wide - VE);
      std::conditional_t<VE == 8, unsigned long long, unsigned> v;
      __builtin_memcpy(&v, at + c, VE);
      v >>= 8 * (x.c - c);
      __builtin_memcpy(w, &v, VE);
    } else {
      __builtin_memcpy(w, at + x.c, VE);
    }
    const unsigned char* fields = p.kept + p.rows * p.wide + row * (p.wide / 32);
    field = fields[x.c / 32];
    if constexpr (GEN) {
      second = fields[min((x.c + VE - 1) / 32, p.wide / 32 - 1)];
      split = (unsigned char)(32 - x.c % 32);
    }
  }
  __device__ __forceinline__ void normalized(const Entries<VE, GEN>& s, float (&out)[VE]) const {
    const float unit = unit_of(field), other = GEN ? unit_of(second) : unit;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float u = GEN && e >= split ? other : unit;
      // (the product of the unit is exact)
      out[e] = __builtin_fmaf((float)(signed char)(w[e / 4] >> (8 * (e % 4))), u, -s.of(e).a) * s.of(e).b;
    }
  }
};

// With ONCE stored past the caches. (Not a test: the compiler makes one store of two, and that an ordinary one.)
template <int KIND, int VE, int GEN, bool ONCE>
__device__ __forceinline__ void store_out(typename ElemOf<KIND>::T* p, const float (&v)[VE], const Cols& x) {
  struct Some {
    typename ElemOf<KIND>::T v[VE];
  } s;
#pragma unroll
  for (int e = 0; e < VE; ++e) s.v[e] = from_f32<KIND>(v[e]);
  if constexpr (VE == 1) {
    *p = s.v[0];
  } else if (!GEN || x.count == VE) {
    static_assert(sizeof(s) == 16, "a thread's channels are 16 bytes");
    store16<ONCE>(p, __builtin_bit_cast(u4any, s));
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (e < x.count) p[e] = s.v[e];
  }
}

template <int KIND, int VE, int GEN>
__device__ __forceinline__ void load_affine(const NormArgs& p, const Cols& x, float (&gamma)[VE], float (&beta)[VE]) {
  using T = typename ElemOf<KIND>::T;
#pragma unroll
  for (int e = 0; e < VE; ++e) gamma[e] = 1.0f, beta[e] = 0.0f;
  Raw<KIND, VE> r;
  if (p.gamma) {
    r.template load<GEN>(static_cast<const T*>(p.gamma) + x.c, x);
    r.get(gamma);
  }
  if (p.beta) {
    r.template load<GEN>(static_cast<const T*>(p.beta) + x.c, x);
    r.get(beta);
  }
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
// x -> act((x - mean) scale + beta)
template <int KIND, int VE>
__device__ __forceinline__ void forward_vec(int act, const float (&mean)[VE], const float (&scale)[VE],
                                            const float (&beta)[VE], float (&x)[VE]) {
  float z[VE], da[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) z[e] = __builtin_fmaf(x[e] - mean[e], scale[e], beta[e]);
  activate_vec<KIND, VE>(act, z, x, da);
}
// of each channel, from its group: the mean, and gamma r
template <int VE, int GEN>
__device__ __forceinline__ void mean_scale(const Entries<VE, GEN>& s, const float (&gamma)[VE], float (&mean)[VE],
                                           float (&scale)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    mean[e] = s.of(e).a;
    scale[e] = gamma[e] * s.of(e).b;
  }
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
// w = gamma dz -> dx = r (w - mean w - v mean(w v)); s: m and r, means: of w and w v
template <int VE, int GEN>
__device__ __forceinline__ void dx_vec(const Entries<VE, GEN>& s, const Entries<VE, GEN>& means, const float (&v)[VE],
                                       float (&w)[VE]) {
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const float r = s.of(e).b;
    w[e] = __builtin_fmaf(v[e], -r * means.of(e).b, __builtin_fmaf(w[e], r, -r * means.of(e).a));
  }
}

// ---- sums --------------------------------------------------------------------------------
// Mean and squared deviations of ROWS rows of each entry (of VE values, or one, a row)
template <int VE, int GEN, int ROWS>
__device__ __forceinline__ Entries<VE, GEN> moments(const float (&v)[ROWS][VE]) {
  constexpr int N = entries_of<VE, GEN>(), W = VE / N;
  Entries<VE, GEN> s;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    float m = 0.0f, M = 0.0f;
#pragma unroll
    for (int b = 0; b < ROWS; ++b)
#pragma unroll
      for (int w = 0; w < W; ++w) m += v[b][i * W + w];
    m *= 1.0f / (ROWS * W);
#pragma unroll
    for (int b = 0; b < ROWS; ++b)
#pragma unroll
      for (int w = 0; w < W; ++w) M += (v[b][i * W + w] - m) * (v[b][i * W + w] - m);
    s.e[i] = Pair{m, M};
  }
  return s;
}
// (m, M) of n values joined with that of k more. (Numbers of values are floats: a frame of 2^28 rows has more than
// an integer counts.)
__device__ __forceinline__ void join_moments(Pair& p, float n, const Pair& q, float k) {
  const float d = q.a - p.a, w = n == 0.0f ? 1.0f : k * __builtin_amdgcn_rcpf(n + k);
  p.a += d * w;
  p.b += q.b + d * (d * (n * w));  // (with n == 0 d is q's mean, whose square may leave the range)
}
template <int VE, int GEN>
__device__ __forceinline__ void join_rows(Entries<VE, GEN>& s, int n, const Entries<VE, GEN>& q, int k) {
  constexpr int N = entries_of<VE, GEN>(), W = VE / N;
#pragma unroll
  for (int i = 0; i < N; ++i) join_moments(s.e[i], (float)n * W, q.e[i], (float)k * W);
}
// Sums of each entry's channels: of b (a) and of g (b)
template <int VE, int GEN>
__device__ __forceinline__ Entries<VE, GEN> entry_sums(const float (&b)[VE], const float (&g)[VE]) {
  constexpr int N = entries_of<VE, GEN>(), W = VE / N;
  Entries<VE, GEN> s;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    s.e[i] = Pair{0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < W; ++w) s.e[i].a += b[i * W + w], s.e[i].b += g[i * W + w];
  }
  return s;
}
// Both for two pieces: moments of one row, and sums.
template <int VE>
__device__ __forceinline__ Entries<VE, kPieces> piece_moments(const float (&v)[VE], const Cols& x, int left) {
  Entries<VE, kPieces> s;
  s.left = left;
  const int n = min(left, x.count);
  float m[2] = {0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < VE; ++e) m[0] += e < n ? v[e] : 0.0f, m[1] += e >= n && e < x.count ? v[e] : 0.0f;
  m[0] *= 1.0f / (float)n;
  m[1] *= 1.0f / (float)max(x.count - n, 1);
  float M[2] = {0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const float d = v[e] - (e < n ? m[0] : m[1]), dd = d * d;
    M[0] += e < n ? dd : 0.0f, M[1] += e >= n && e < x.count ? dd : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) s.e[i] = Pair{m[i], M[i]};
  return s;
}
template <int VE>
__device__ __forceinline__ Entries<VE, kPieces> piece_sums(const float (&b)[VE], const float (&g)[VE], int left) {
  Entries<VE, kPieces> s;
  s.left = left;
  s.e[0] = s.e[1] = Pair{0.0f, 0.0f};
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    s.e[0].a += e < left ? b[e] : 0.0f, s.e[0].b += e < left ? g[e] : 0.0f;
    s.e[1].a += e < left ? 0.0f : b[e], s.e[1].b += e < left ? 0.0f : g[e];
  }
  return s;
}
template <int VE, int GEN>
__device__ __forceinline__ void put_entries(Pair* to, const Entries<VE, GEN>& s, const Cols& x) {
#pragma unroll
  for (int i = 0; i < entries_of<VE, GEN>(); ++i)
    if (!GEN || i < x.count) to[i] = s.e[i];
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
// 1 / sqrt(M / n + eps), inv = 1 / n. NaN where squares or their sum have left fp32's range (1 / sqrt would be zero,
// and y act(beta) without a word), and infinite below the normal numbers, whose squares have lost their digits.
__device__ __forceinline__ float deviation(float M, float inv, float eps) {
  const float var = __builtin_fmaf(M, inv, eps);
  const float r = var < __builtin_inff() ? __builtin_amdgcn_rsqf(var) : __builtin_nanf("");
  return var < 0x1p-126f ? __builtin_inff() : r;
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

// f(entry, its channels) for the entries of group q of a row, every 2^lanes-th of them.
template <int VE, int GEN, class F>
__device__ __forceinline__ void each_entry(const NormArgs& p, const Pair* parts, int q, int lane, F&& f) {
  if constexpr (GEN == kPieces) {
    const int first = q * p.per, end = first + p.per, last = (end - 1) / VE;
    for (int v = first / VE + lane; v <= last; v += 1 << p.lanes)
      f(parts[2 * v + (v * VE < first)], (float)(min(end, (v + 1) * VE) - max(first, v * VE)));
  } else {
    const Pair* s = parts + q * p.group_entries;
    for (int k = lane; k < p.group_entries; k += 1 << p.lanes) f(s[k], (float)(VE / entries_of<VE, GEN>()));
  }
}

// ---- every row a frame -----------------------------------------------------------------
// T threads a row, C vectors of VE channels a thread (at neighbouring places for neighbouring threads). With
// LANES a group is a power of two of vectors, at most 64, so that it is that many neighbouring lanes, which
// add up without LDS or a barrier; else the entries of a row meet in LDS, and then a pair for each group.
// (16,384 x 2048 in bf16, groups of 64, gelu: 50 us through LDS, 38 by lanes, and 34 with gelu in six terms; a copy's
// rate would be 26.) A block takes rows one after another: gamma and beta stay in registers, and the next row is
// loaded while this one is computed.
template <int KIND, int VE, int GEN, int T, int C, bool LANES, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_norm_rows(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  constexpr int W = VE / entries_of<VE, GEN>();  // (kPieces: a vector is two entries too)
  extern __shared__ __align__(16) char lds[];
  constexpr int R = kThreads / T;
  const int t = threadIdx.x % T, mine = threadIdx.x / T;
  Pair* parts = reinterpret_cast<Pair*>(lds) + (size_t)mine * (p.entries + p.groups);
  Pair* whole = parts + p.entries;
  Cols x[C];
  float gamma[C][VE], beta[C][VE];
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = min(k * T + t, p.vecs - 1) * VE;
    x[k] = Cols{c, min(VE, p.channels - c)};
    load_affine<KIND, VE, GEN>(p, x[k], gamma[k], beta[k]);
  }
  Raw<KIND, VE> raw[C];
  auto fetch = [&](long row) {
    const E* at = static_cast<const E*>(p.x) + min(row, p.rows - 1) * p.ld_x;
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (k * T + t < p.vecs) raw[k].template load<GEN>(at + x[k].c, x[k]);
  };
  const long step = (long)gridDim.x * R;
  fetch((long)blockIdx.x * R + mine);
  for (long row0 = (long)blockIdx.x * R; row0 < p.rows; row0 += step) {
    const long row = row0 + mine;
    const bool there = row < p.rows;
    float v[C][1][VE];
    Entries<VE, GEN> stat[C];
    auto keep = [&](int q, const Pair& s) {
      if (p.stats && there) *reinterpret_cast<Pair*>(p.stats + 2 * (row * p.groups + q)) = s;
    };
    if constexpr (LANES) {
#pragma unroll
      for (int k = 0; k < C; ++k) {
        raw[k].get(v[k][0]);
        const Pair s = moments<VE, GEN, 1>(v[k]).e[0];
        const float m = sum_lanes(s.a, p.lanes) * p.inv_entries;
        const float M = sum_lanes(s.b + VE * (s.a - m) * (s.a - m), p.lanes);
        stat[k].e[0] = Pair{m, deviation(M, p.inv_per, p.eps)};
        if (k * T + t < p.vecs && (t & (p.group_entries - 1)) == 0) keep(x[k].c / p.per, stat[k].e[0]);
      }
      if (row0 + step < p.rows) fetch(row + step);
    } else {
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k * T + t < p.vecs) {
          raw[k].get(v[k][0]);
          if constexpr (GEN == kPieces)
            put_entries<VE, GEN>(parts + x[k].c / W, piece_moments<VE>(v[k][0], x[k], left_of(x[k], p.per)), x[k]);
          else
            put_entries<VE, GEN>(parts + x[k].c / W, moments<VE, GEN, 1>(v[k]), x[k]);
        }
      if (row0 + step < p.rows) fetch(row + step);
      row_sync<T>();
      each_group<T>(t, p.groups, p.lanes, [&](int q, int lane, bool in) {
        float m = 0.0f, M = 0.0f;
        each_entry<VE, GEN>(p, parts, q, lane, [&](const Pair& s, float n) { m += n * s.a; });
        m = sum_lanes(m, p.lanes) * p.inv_per;
        each_entry<VE, GEN>(p, parts, q, lane, [&](const Pair& s, float n) { M += s.b + n * (s.a - m) * (s.a - m); });
        const Pair r = {m, deviation(sum_lanes(M, p.lanes), p.inv_per, p.eps)};
        if (in && lane == 0) {
          whole[q] = r;
          keep(q, r);
        }
      });
      row_sync<T>();
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k * T + t < p.vecs) stat[k] = of_groups<VE, GEN>(whole, x[k], p.per);
      row_sync<T>();  // (the next row's parts go where these are read)
    }
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (k * T + t >= p.vecs) continue;
      float mean[VE], scale[VE];
      mean_scale<VE, GEN>(stat[k], gamma[k], mean, scale);
      forward_vec<KIND, VE>(p.act, mean, scale, beta[k], v[k][0]);
      if (there) store_out<KIND, VE, GEN, ONCE>(static_cast<E*>(p.y) + row * p.ld_y + x[k].c, v[k][0], x[k]);
    }
  }
}

// Its gradients: dgamma and dbeta of a thread's channels are summed over all rows that its block takes, and
// then over the block's row lanes; partial [blocks][2][channels]. (16,384 x 2048 from the checkpoint in bf16: 74 us
// with one row under way, 49 with two, 33 at a copy's rate.)
template <int KIND, int VE, int GEN, int T, int C, bool LANES, bool KEPT, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_norm_rows_grad(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  constexpr int W = VE / entries_of<VE, GEN>();  // (kPieces: a vector is two entries too)
  extern __shared__ __align__(16) char lds[];
  constexpr int R = kThreads / T;
  const int t = threadIdx.x % T, mine = threadIdx.x / T;
  Pair* parts = reinterpret_cast<Pair*>(lds) + (size_t)mine * (p.entries + p.groups);
  Pair* whole = parts + p.entries;
  Cols x[C];
  float gamma[C][VE], beta[C][VE], ga[C][VE] = {}, be[C][VE] = {};
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int c = min(k * T + t, p.vecs - 1) * VE;
    x[k] = Cols{c, min(VE, p.channels - c)};
    load_affine<KIND, VE, GEN>(p, x[k], gamma[k], beta[k]);
  }
  // two rows are under way (with one, 16 waves of a compute unit wait for too few bytes)
  // (m and r of each channel would take too many registers for that: they are loaded at the row's turn)
  struct Ahead {
    RawX<KIND, VE, GEN, KEPT> x[C];
    Raw<KIND, VE> dy[C];
    Entries<VE, GEN == 1 ? 0 : GEN> stat[C];
  } ahead[2];
  auto stats_of = [&](long row, const Cols& c) {
    return of_groups<VE, GEN>(reinterpret_cast<const Pair*>(p.stats + 2 * row * p.groups), c, p.per);
  };
  auto fetch = [&](long row, Ahead& to) {  // (dy of rows past the last: zeros)
    const bool there = row < p.rows;
    row = min(row, p.rows - 1);
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (k * T + t >= p.vecs) continue;
      to.x[k].load_at(p, row, x[k]);
      if (there)
        to.dy[k].template load<GEN>(static_cast<const E*>(p.dy) + row * p.ld_y + x[k].c, x[k]);
      else
        to.dy[k].zeros();
      if constexpr (GEN != 1) to.stat[k] = stats_of(row, x[k]);
    }
  };
  const long step = (long)gridDim.x * R;
  auto compute = [&](long row0, Ahead& from) {
    const long row = row0 + mine;
    const bool there = row < p.rows;
    float v[C][VE], w[C][VE];
    Entries<VE, GEN> means[C], stat[C];
#pragma unroll
    for (int k = 0; k < C; ++k) {
      means[k] = Entries<VE, GEN>{};
      if (k * T + t >= p.vecs) continue;
      if constexpr (GEN == 1)
        stat[k] = stats_of(min(row, p.rows - 1), x[k]);
      else
        stat[k] = from.stat[k];
      from.x[k].normalized(stat[k], v[k]);
      from.dy[k].get(w[k]);
      grad_vec<KIND, VE>(p.act, gamma[k], beta[k], v[k], w[k]);
      float wv[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        be[k][e] += w[k][e];
        ga[k][e] += w[k][e] * v[k][e];
        w[k][e] *= gamma[k][e];
        wv[e] = w[k][e] * v[k][e];
      }
      if constexpr (GEN == kPieces)
        means[k] = piece_sums<VE>(w[k], wv, left_of(x[k], p.per));
      else
        means[k] = entry_sums<VE, GEN>(w[k], wv);
      if constexpr (!LANES) put_entries<VE, GEN>(parts + x[k].c / W, means[k], x[k]);
    }
    if (row0 + 2 * step < p.rows) fetch(row + 2 * step, from);
    if constexpr (LANES) {
#pragma unroll
      for (int k = 0; k < C; ++k)
        means[k].e[0] = Pair{sum_lanes(means[k].e[0].a, p.lanes) * p.inv_per,
                             sum_lanes(means[k].e[0].b, p.lanes) * p.inv_per};
    } else {
      row_sync<T>();
      each_group<T>(t, p.groups, p.lanes, [&](int q, int lane, bool in) {
        float a = 0.0f, b = 0.0f;
        each_entry<VE, GEN>(p, parts, q, lane, [&](const Pair& s, float) { a += s.a, b += s.b; });
        a = sum_lanes(a, p.lanes) * p.inv_per;
        b = sum_lanes(b, p.lanes) * p.inv_per;
        if (in && lane == 0) whole[q] = Pair{a, b};
      });
      row_sync<T>();
#pragma unroll
      for (int k = 0; k < C; ++k)
        if (k * T + t < p.vecs) means[k] = of_groups<VE, GEN>(whole, x[k], p.per);
      row_sync<T>();
    }
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (k * T + t >= p.vecs || !there || !p.dx) continue;
      dx_vec<VE, GEN>(stat[k], means[k], v[k], w[k]);
      store_out<KIND, VE, GEN, ONCE>(static_cast<E*>(p.dx) + row * p.ld_x + x[k].c, w[k], x[k]);
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
// Threads (vector tc of `part`, row lane tr): part is at most 256; the threads left over by 256 / part
// idle. Rows tr, tr + TR, ... The part's channels: from c0 on, `channels` of them.
struct Lay {
  int tc, tr, TR, c0, channels;
  Cols x;
  bool in;
};
template <int VE>
__device__ __forceinline__ Lay lay_of(const NormArgs& p) {
  Lay l;
  l.TR = kThreads / p.part;
  l.tr = threadIdx.x / p.part;
  l.tc = threadIdx.x - l.tr * p.part;
  l.c0 = blockIdx.x * p.part_channels;
  l.channels = min(p.part_channels, p.channels - l.c0);
  l.in = l.tr < l.TR && l.tc * VE < l.channels;
  const int at = l.in ? l.tc * VE : 0;
  l.x = Cols{l.c0 + at, min(VE, l.channels - at)};
  return l;
}
// rows of row lane tr
__device__ __forceinline__ int rows_of(int count, int tr, int TR) { return count > tr ? (count - tr + TR - 1) / TR : 0; }

constexpr int kBatch = 4;  // rows under way

// The moments s of a thread's entries, joined with those of its rows from the `from`-th on: first + tr + i TR below
// first + count
template <int KIND, int VE, int GEN>
__device__ __forceinline__ void thread_moments(const NormArgs& p, long first, int count, const Lay& l, int from,
                                               Entries<VE, GEN>& s) {
  const typename ElemOf<KIND>::T* x = static_cast<const typename ElemOf<KIND>::T*>(p.x) + l.x.c;
  int n = from, r = l.tr + from * l.TR;
  for (; r + (kBatch - 1) * l.TR < count; r += kBatch * l.TR) {
    float v[kBatch][VE];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      Raw<KIND, VE> raw;
      raw.template load<GEN>(x + (first + r + (long)b * l.TR) * p.ld_x, l.x);
      raw.get(v[b]);
    }
    join_rows<VE, GEN>(s, n, moments<VE, GEN, kBatch>(v), kBatch);
    n += kBatch;
  }
  for (; r < count; r += l.TR) {
    float v[1][VE];
    Raw<KIND, VE> raw;
    raw.template load<GEN>(x + (first + r) * p.ld_x, l.x);
    raw.get(v[0]);
    join_rows<VE, GEN>(s, n, moments<VE, GEN, 1>(v), 1);
    ++n;
  }
}

// y = act((x - mean) scale + beta) of a thread's channels over its rows
template <int KIND, int VE, int GEN, bool ONCE>
__device__ __forceinline__ void thread_apply(const NormArgs& p, long first, int count, const Lay& l, int from,
                                             const float (&mean)[VE], const float (&scale)[VE],
                                             const float (&beta)[VE]) {
  using E = typename ElemOf<KIND>::T;
  const E* x = static_cast<const E*>(p.x) + l.x.c;
  E* y = static_cast<E*>(p.y) + l.x.c;
  int r = l.tr + from * l.TR;
  Raw<KIND, VE> raw[kBatch];
  float v[VE];
  for (; r + (kBatch - 1) * l.TR < count; r += kBatch * l.TR) {
#pragma unroll
    for (int b = 0; b < kBatch; ++b) raw[b].template load<GEN>(x + (first + r + (long)b * l.TR) * p.ld_x, l.x);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      raw[b].get(v);
      forward_vec<KIND, VE>(p.act, mean, scale, beta, v);
      store_out<KIND, VE, GEN, ONCE>(y + (first + r + (long)b * l.TR) * p.ld_y, v, l.x);
    }
  }
  for (; r < count; r += l.TR) {
    raw[0].template load<GEN>(x + (first + r) * p.ld_x, l.x);
    raw[0].get(v);
    forward_vec<KIND, VE>(p.act, mean, scale, beta, v);
    store_out<KIND, VE, GEN, ONCE>(y + (first + r) * p.ld_y, v, l.x);
  }
}

// f(v, dy, row) over a thread's rows, two of them under way together.
template <int KIND, int VE, int GEN, bool KEPT, class F>
__device__ __forceinline__ void thread_rows(const NormArgs& p, long first, int count, const Lay& l, int from,
                                            const Entries<VE, GEN>& s, F&& f) {
  constexpr int kRows = 2;
  using E = typename ElemOf<KIND>::T;
  const E* dy = static_cast<const E*>(p.dy) + l.x.c;
  for (int r = l.tr + from * l.TR; r < count; r += kRows * l.TR) {
    RawX<KIND, VE, GEN, KEPT> raw_x[kRows];
    Raw<KIND, VE> raw_dy[kRows];
#pragma unroll
    for (int b = 0; b < kRows; ++b)
      if (r + b * l.TR < count) {
        raw_x[b].load_at(p, first + r + (long)b * l.TR, l.x);
        raw_dy[b].template load<GEN>(dy + (first + r + (long)b * l.TR) * p.ld_y, l.x);
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
// dz and dz v of a thread's channels summed over its rows
template <int KIND, int VE, int GEN, bool KEPT>
__device__ __forceinline__ void thread_sums(const NormArgs& p, long first, int count, const Lay& l, int from,
                                            const Entries<VE, GEN>& s, const float (&gamma)[VE],
                                            const float (&beta)[VE], float (&be)[VE], float (&ga)[VE]) {
  thread_rows<KIND, VE, GEN, KEPT>(p, first, count, l, from, s, [&](float (&v)[VE], float (&d)[VE], long) {
    grad_vec<KIND, VE>(p.act, gamma, beta, v, d);
#pragma unroll
    for (int e = 0; e < VE; ++e) be[e] += d[e], ga[e] += d[e] * v[e];
  });
}
template <int KIND, int VE, int GEN, bool KEPT, bool ONCE>
__device__ __forceinline__ void thread_dx(const NormArgs& p, long first, int count, const Lay& l, int from,
                                          const Entries<VE, GEN>& s, const Entries<VE, GEN>& means,
                                          const float (&gamma)[VE], const float (&beta)[VE]) {
  using E = typename ElemOf<KIND>::T;
  E* dx = static_cast<E*>(p.dx) + l.x.c;
  thread_rows<KIND, VE, GEN, KEPT>(p, first, count, l, from, s, [&](float (&v)[VE], float (&d)[VE], long row) {
    grad_vec<KIND, VE>(p.act, gamma, beta, v, d);
#pragma unroll
    for (int e = 0; e < VE; ++e) d[e] *= gamma[e];
    dx_vec<VE, GEN>(s, means, v, d);
    store_out<KIND, VE, GEN, ONCE>(dx + row * p.ld_x, d, l.x);
  });
}
// be and ga of the block's threads summed over its row lanes, to out [2][channels] at the part's channels
template <int VE>
__device__ __forceinline__ void put_channel_sums(const NormArgs& p, const Lay& l, const float (&ga)[VE],
                                                 const float (&be)[VE], float* sums, float* out) {
  for (int which = 0; which < 2; ++which) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < VE; ++e) sums[threadIdx.x * VE + e] = which ? be[e] : ga[e];
    __syncthreads();
    for (int c = threadIdx.x; c < l.channels; c += kThreads) {
      float v = 0.0f;
      for (int m = 0; m < l.TR; ++m) v += sums[m * p.part * VE + c];
      out[which * p.channels + l.c0 + c] = v;
    }
  }
}

// Whole frames: grid (parts, frames, or fewer in y: strided). A thread's first kHold rows stay in registers
// between the sums and the output; what is beyond them is read again. (64 ragged frames of 12,288 x 1600 in fp32: 50 us
// reading all rows twice, 41 so; 30 at a copy's rate.)
template <int KIND, int VE, int GEN, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_norm_frames(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  constexpr int kHold = 8, N = entries_of<VE, GEN>(), W = VE / N;
  __shared__ Pair parts[kThreads * N], whole[kThreads * N];
  const Lay l = lay_of<VE>(p);
  const int wide = p.part * N, groups = l.channels / p.per;  // entries of a row lane
  float gamma[VE], beta[VE];
  load_affine<KIND, VE, GEN>(p, l.x, gamma, beta);
  for (int f = blockIdx.y; f < p.frames; f += gridDim.y) {
    const Frame w = frame_of(p, f);
    const int have = l.in ? min(rows_of(w.count, l.tr, l.TR), kHold) : 0;
    // (rows past the thread's last stay zeros)
    Raw<KIND, VE> raw[kHold];
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      raw[i].zeros();
      if (i < have)
        raw[i].template load<GEN>(static_cast<const E*>(p.x) + (w.first + l.tr + (long)i * l.TR) * p.ld_x + l.x.c, l.x);
    }
    Entries<VE, GEN> mine{};
#pragma unroll
    for (int i = 0; i < kHold; ++i) {
      float v[VE];
      raw[i].get(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) mine.e[GEN ? e : 0].a += v[e];
    }
    const float inv = have ? 1.0f / ((float)have * W) : 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) mine.e[i].a *= inv;
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (i < have) {
        float v[VE];
        raw[i].get(v);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float d = v[e] - mine.of(e).a;
          mine.e[GEN ? e : 0].b += d * d;
        }
      }
    if (l.in) {
      thread_moments<KIND, VE, GEN>(p, w.first, w.count, l, kHold, mine);
      put_entries<VE, GEN>(parts + l.tr * wide + l.tc * N, mine, l.x);
    }
    __syncthreads();
    const float total = (float)w.count * (float)p.per;
    each_group<kThreads>(threadIdx.x, groups, p.lanes, [&](int q, int lane, bool in) {
      float m = 0.0f, M = 0.0f;
      const int all = l.TR * p.group_entries;
      for (int k = lane; k < all; k += 1 << p.lanes) {
        const int tr = k / p.group_entries;
        m += (float)rows_of(w.count, tr, l.TR) * parts[tr * wide + q * p.group_entries + k - tr * p.group_entries].a;
      }
      m = sum_lanes(m, p.lanes) * W / total;
      for (int k = lane; k < all; k += 1 << p.lanes) {
        const int tr = k / p.group_entries, rows = rows_of(w.count, tr, l.TR);
        const Pair s = parts[tr * wide + q * p.group_entries + k - tr * p.group_entries];
        M += s.b + (float)rows * W * (s.a - m) * (s.a - m);
      }
      M = sum_lanes(M, p.lanes);
      const Pair s = w.count ? Pair{m, deviation(M, 1.0f / total, p.eps)} : Pair{0.0f, 0.0f};
      if (in && lane == 0) {
        whole[q] = s;
        if (p.stats) *reinterpret_cast<Pair*>(p.stats + 2 * ((long)f * p.groups + l.c0 / p.per + q)) = s;
      }
    });
    __syncthreads();
    if (l.in) {
      float mean[VE], scale[VE];
      mean_scale<VE, GEN>(of_groups<VE, GEN>(whole, Cols{l.x.c - l.c0, l.x.count}, p.per), gamma, mean, scale);
#pragma unroll
      for (int i = 0; i < kHold; ++i)
        if (i < have) {
          float v[VE];
          raw[i].get(v);
          forward_vec<KIND, VE>(p.act, mean, scale, beta, v);
          store_out<KIND, VE, GEN, ONCE>(static_cast<E*>(p.y) + (w.first + l.tr + (long)i * l.TR) * p.ld_y + l.x.c, v, l.x);
        }
      thread_apply<KIND, VE, GEN, ONCE>(p, w.first, w.count, l, kHold, mean, scale, beta);
    }
    __syncthreads();
  }
}

// partial [gridDim.y][2][channels]
template <int KIND, int VE, int GEN, bool KEPT, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_norm_frames_grad(const NormArgs p) {
  using E = typename ElemOf<KIND>::T;
  constexpr int kHold = VE == 8 ? 4 : 8;  // rows whose v and dz stay in registers: 64 of these
  constexpr int N = entries_of<VE, GEN>();
  __shared__ Pair parts[kThreads * N], whole[kThreads * N];
  __shared__ float sums[kThreads * VE];
  const Lay l = lay_of<VE>(p);
  const int wide = p.part * N, groups = l.channels / p.per;
  float gamma[VE], beta[VE], ga[VE] = {}, be[VE] = {};
  load_affine<KIND, VE, GEN>(p, l.x, gamma, beta);
  for (int f = blockIdx.y; f < p.frames; f += gridDim.y) {
    const Frame w = frame_of(p, f);
    Entries<VE, GEN> s =
        of_groups<VE, GEN>(reinterpret_cast<const Pair*>(p.stats + 2 * (long)f * p.groups), l.x, p.per);
    const int have = l.in ? min(rows_of(w.count, l.tr, l.TR), kHold) : 0;
    RawX<KIND, VE, GEN, KEPT> raw_x[kHold];
    Raw<KIND, VE> raw_dy[kHold];
#pragma unroll
    for (int i = 0; i < kHold; ++i)
      if (i < have) {
        const long row = w.first + l.tr + (long)i * l.TR;
        raw_x[i].load_at(p, row, l.x);
        raw_dy[i].template load<GEN>(static_cast<const E*>(p.dy) + row * p.ld_y + l.x.c, l.x);
      }
    hold_back(s);
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
    if (l.in) thread_sums<KIND, VE, GEN, KEPT>(p, w.first, w.count, l, kHold, s, gamma, beta, b, g);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      be[e] += b[e];
      ga[e] += g[e];
      b[e] *= gamma[e];
      g[e] *= gamma[e];
    }
    if (!p.dx) continue;
    if (l.in) put_entries<VE, GEN>(parts + l.tr * wide + l.tc * N, entry_sums<VE, GEN>(b, g), l.x);
    __syncthreads();
    const float total = fmaxf((float)w.count * (float)p.per, 1.0f);
    each_group<kThreads>(threadIdx.x, groups, p.lanes, [&](int q, int lane, bool in) {
      float a = 0.0f, c = 0.0f;
      for (int k = lane; k < l.TR * p.group_entries; k += 1 << p.lanes) {
        const int tr = k / p.group_entries;
        const Pair u = parts[tr * wide + q * p.group_entries + k - tr * p.group_entries];
        a += u.a;
        c += u.b;
      }
      a = sum_lanes(a, p.lanes);
      c = sum_lanes(c, p.lanes);
      if (in && lane == 0) whole[q] = Pair{a / total, c / total};
    });
    __syncthreads();
    if (l.in) {
      const Entries<VE, GEN> means = of_groups<VE, GEN>(whole, Cols{l.x.c - l.c0, l.x.count}, p.per);
#pragma unroll
      for (int i = 0; i < kHold; ++i)
        if (i < have) {
          dx_vec<VE, GEN>(s, means, v[i], d[i]);
          store_out<KIND, VE, GEN, ONCE>(static_cast<E*>(p.dx) + (w.first + l.tr + (long)i * l.TR) * p.ld_x + l.x.c, d[i],
                                   l.x);
        }
      thread_dx<KIND, VE, GEN, KEPT, ONCE>(p, w.first, w.count, l, kHold, s, means, gamma, beta);
    }
    __syncthreads();
  }
  if (p.partial) put_channel_sums<VE>(p, l, ga, be, sums, p.partial + (long)blockIdx.y * 2 * p.channels);
}

// ---- frames cut into slices --------------------------------------------------------------------
// Slice z of a frame's rows
__device__ __forceinline__ Frame slice_of(const Frame& w, int z, int slices) {
  // (the first `more` slices have a row more)
  const int each = w.count / slices, more = w.count - each * slices;
  return Frame{w.first + (long)each * z + min(z, more), each + (z < more)};
}

// The groups that a part of the columns meets (the first and the last one may go on beyond it), and
// where their sums of a slice are: pairs [frames][slices][parts][part_groups].
struct PartGroups {
  int first, count;
};
__device__ __forceinline__ PartGroups groups_of(const NormArgs& p, const Lay& l) {
  const int q = l.c0 / p.per;
  return PartGroups{q, (l.c0 + l.channels - 1) / p.per - q + 1};
}
__device__ __forceinline__ Pair* slice_pairs(const NormArgs& p, int f, int z, int part) {
  return reinterpret_cast<Pair*>(p.pairs) + (((long)f * p.slices + z) * p.parts + part) * p.part_groups;
}
// f(group's place in the part, its first entry there, the one past its last, lane, whether there is such a group)
template <class F>
__device__ __forceinline__ void each_part_group(const NormArgs& p, const Lay& l, int W, F&& f) {
  const PartGroups g = groups_of(p, l);
  each_group<kThreads>(threadIdx.x, g.count, p.lanes, [&](int k, int lane, bool in) {
    const int a = max((g.first + k) * p.per - l.c0, 0), b = min((g.first + k + 1) * p.per - l.c0, l.channels);
    f(k, a / W, b / W, lane, in);
  });
}

// Moments of each group over a slice, or of its channels in this part. Grid (parts, slices, frames).
template <int KIND, int VE, int GEN>
__global__ __launch_bounds__(kThreads) void k_norm_stats(const NormArgs p) {
  constexpr int N = entries_of<VE, GEN>(), W = VE / N;
  __shared__ Pair parts[kThreads * N];
  const Lay l = lay_of<VE>(p);
  const int wide = p.part * N, entries = (l.channels + W - 1) / W;
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), blockIdx.y, p.slices);
    Entries<VE, GEN> mine{};
    if (l.in) {
      thread_moments<KIND, VE, GEN>(p, w.first, w.count, l, 0, mine);
      put_entries<VE, GEN>(parts + l.tr * wide + l.tc * N, mine, l.x);
    }
    __syncthreads();
    for (int k = threadIdx.x; k < entries; k += kThreads) {
      Pair s = parts[k];
      int have = rows_of(w.count, 0, l.TR);
      for (int tr = 1; tr < l.TR; ++tr) {
        const int n = rows_of(w.count, tr, l.TR);
        if (n) join_moments(s, (float)have * W, parts[tr * wide + k], (float)n * W);
        have += n;
      }
      parts[k] = s;
    }
    __syncthreads();
    Pair* out = slice_pairs(p, f, blockIdx.y, blockIdx.x);
    each_part_group(p, l, W, [&](int q, int e0, int e1, int lane, bool in) {
      float m = 0.0f, M = 0.0f;
      for (int k = e0 + lane; k < e1; k += 1 << p.lanes) m += parts[k].a;
      m = sum_lanes(m, p.lanes) / (float)(e1 - e0);
      const float each = (float)w.count * W;
      for (int k = e0 + lane; k < e1; k += 1 << p.lanes) M += parts[k].b + each * (parts[k].a - m) * (parts[k].a - m);
      M = sum_lanes(M, p.lanes);
      if (in && lane == 0) out[q] = Pair{m, M};
    });
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

// The parts and slices that a group's sums come from: part p0 + k % parts, slice k / parts.
struct GroupSums {
  int p0, parts;
  unsigned n;
  __device__ __forceinline__ GroupSums(const NormArgs& p, int q) {
    p0 = q * p.per / p.part_channels;
    parts = ((q + 1) * p.per - 1) / p.part_channels - p0 + 1;
    n = (unsigned)p.slices * parts;
  }
  // (and how many of the group's channels are in the part)
  __device__ __forceinline__ Pair get(const NormArgs& p, int f, int q, unsigned k, int& z, int& channels) const {
    z = (int)(k / (unsigned)parts);
    const int part = p0 + (int)(k - (unsigned)z * parts), c0 = part * p.part_channels;
    channels = min((q + 1) * p.per, c0 + p.part_channels) - max(q * p.per, c0);
    return slice_pairs(p, f, z, part)[q - c0 / p.per];
  }
};

// The slices' moments of each (frame, group) joined, in fp64: a block each.
__global__ __launch_bounds__(kThreads) void k_norm_stats_join(const NormArgs p) {
  __shared__ double lds[4];
  const long all = (long)p.frames * p.groups;
  for (long at = blockIdx.x; at < all; at += gridDim.x) {
    const int f = (int)(at / p.groups), q = (int)(at % p.groups);
    const Frame w = frame_of(p, f);
    const GroupSums sums(p, q);
    // a part's moments, and how many values it stands for
    auto entry = [&](unsigned k, Pair& e) {
      int z, channels;
      e = sums.get(p, f, q, k, z, channels);
      return (double)slice_of(w, z, p.slices).count * channels;
    };
    // one pass, around the first part's mean (in fp64, and the parts' means lie together)
    Pair first;
    entry(0, first);
    constexpr int kUnder = 4;
    double d = 0.0, M = 0.0;
    for (unsigned k = threadIdx.x; k < sums.n; k += kUnder * kThreads) {
      Pair e[kUnder];
      double count[kUnder];
#pragma unroll
      for (int u = 0; u < kUnder; ++u) {
        count[u] = entry(min(k + u * kThreads, sums.n - 1), e[u]);
        if (k + u * kThreads >= sums.n) count[u] = 0.0;
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
    var += (double)p.eps;
    // (as deviation() has it)
    const float r = var < 0x1p-126 ? __builtin_inff() : var < __builtin_inf() ? (float)(1.0 / sqrt(var)) : __builtin_nanf("");
    if (threadIdx.x == 0) *reinterpret_cast<Pair*>(p.stats + 2 * at) = total > 0.0 ? Pair{(float)m, r} : Pair{0.0f, 0.0f};
  }
}

// (The output's slices from the last one on: what the sums' pass has read last is in the last cache yet.)
template <int KIND, int VE, int GEN, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_norm_apply(const NormArgs p) {
  const Lay l = lay_of<VE>(p);
  if (!l.in) return;
  float gamma[VE], beta[VE];
  load_affine<KIND, VE, GEN>(p, l.x, gamma, beta);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), gridDim.y - 1 - blockIdx.y, gridDim.y);
    float mean[VE], scale[VE];
    mean_scale<VE, GEN>(of_groups<VE, GEN>(reinterpret_cast<const Pair*>(p.stats + 2 * (long)f * p.groups), l.x, p.per),
                        gamma, mean, scale);
    thread_apply<KIND, VE, GEN, ONCE>(p, w.first, w.count, l, 0, mean, scale, beta);
  }
}

// Sums of w and w v over a slice for each group, or its channels in this part. dgamma and dbeta over all frames
// that a block takes: partial [gridDim.z][slices][2][channels].
template <int KIND, int VE, int GEN, bool KEPT>
__global__ __launch_bounds__(kThreads) void k_norm_sums(const NormArgs p) {
  constexpr int N = entries_of<VE, GEN>(), W = VE / N;
  __shared__ Pair parts[kThreads * N];
  __shared__ float sums[kThreads * VE];
  const Lay l = lay_of<VE>(p);
  const int wide = p.part * N, entries = (l.channels + W - 1) / W;
  float gamma[VE], beta[VE], ga[VE] = {}, be[VE] = {};
  load_affine<KIND, VE, GEN>(p, l.x, gamma, beta);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), blockIdx.y, p.slices);
    const Entries<VE, GEN> s =
        of_groups<VE, GEN>(reinterpret_cast<const Pair*>(p.stats + 2 * (long)f * p.groups), l.x, p.per);
    float b[VE] = {}, g[VE] = {};
    if (l.in) thread_sums<KIND, VE, GEN, KEPT>(p, w.first, w.count, l, 0, s, gamma, beta, b, g);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      be[e] += b[e];
      ga[e] += g[e];
      b[e] *= gamma[e];
      g[e] *= gamma[e];
    }
    if (!p.dx) continue;
    __syncthreads();
    if (l.in) put_entries<VE, GEN>(parts + l.tr * wide + l.tc * N, entry_sums<VE, GEN>(b, g), l.x);
    __syncthreads();
    for (int k = threadIdx.x; k < entries; k += kThreads) {
      Pair sum = parts[k];
      for (int tr = 1; tr < l.TR; ++tr) {
        const Pair q = parts[tr * wide + k];
        sum.a += q.a;
        sum.b += q.b;
      }
      parts[k] = sum;
    }
    __syncthreads();
    Pair* out = slice_pairs(p, f, blockIdx.y, blockIdx.x);
    each_part_group(p, l, W, [&](int q, int e0, int e1, int lane, bool in) {
      float a = 0.0f, c = 0.0f;
      for (int k = e0 + lane; k < e1; k += 1 << p.lanes) a += parts[k].a, c += parts[k].b;
      a = sum_lanes(a, p.lanes);
      c = sum_lanes(c, p.lanes);
      if (in && lane == 0) out[q] = Pair{a, c};
    });
  }
  if (p.partial)
    put_channel_sums<VE>(p, l, ga, be, sums, p.partial + ((long)blockIdx.z * p.slices + blockIdx.y) * 2 * p.channels);
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
      const GroupSums sums(p, q);
      double a = 0.0, b = 0.0;
#pragma unroll 4
      for (unsigned k = threadIdx.x; k < sums.n; k += kThreads) {
        int z, channels;
        const Pair e = sums.get(p, f, q, k, z, channels);
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

template <int KIND, int VE, int GEN, bool KEPT, bool ONCE>
__global__ __launch_bounds__(kThreads) void k_norm_dx(const NormArgs p) {
  const Lay l = lay_of<VE>(p);
  if (!l.in) return;
  float gamma[VE], beta[VE];
  load_affine<KIND, VE, GEN>(p, l.x, gamma, beta);
  for (int f = blockIdx.z; f < p.frames; f += gridDim.z) {
    const Frame w = slice_of(frame_of(p, f), gridDim.y - 1 - blockIdx.y, gridDim.y);
    const long at = 2 * (long)f * p.groups;
    thread_dx<KIND, VE, GEN, KEPT, ONCE>(
        p, w.first, w.count, l, 0, of_groups<VE, GEN>(reinterpret_cast<const Pair*>(p.stats + at), l.x, p.per),
        of_groups<VE, GEN>(reinterpret_cast<const Pair*>(p.sums + at), l.x, p.per), gamma, beta);
  }
}

// ---- launches ---------------------------------------------------------------------------------
// channels of a thread, and whether groups are anything but multiples of them
template <class F>
void by_vec(const NormArgs& p, F&& f) {
  using std::integral_constant;
  constexpr int kMost = ELEM_KIND == kF32 ? 4 : 8;
  if (p.vec == 1)
    f(integral_constant<int, 1>{}, std::false_type{});
  else if (p.general)
    f(integral_constant<int, kMost>{}, std::true_type{});
  else
    f(integral_constant<int, kMost>{}, std::false_type{});
}
template <class F>
void with(bool b, F&& f) {
  if (b)
    f(std::true_type{});
  else
    f(std::false_type{});
}
// threads of a row, vectors of a thread, whether groups are lanes, and what a thread's entries are
// (VE is 1 for rows of less than 16 bytes: seven vectors at most)
template <int VE, int GEN, class F>
void by_row(const NormArgs& p, F&& f) {
  using std::integral_constant;
  auto lanes = [&](auto t, auto c) {
    if constexpr (!GEN) {
      if (p.by_lanes) return f(t, c, std::true_type{}, integral_constant<int, 0>{});
    } else if constexpr (ELEM_KIND != kF32 || decltype(c)::value > 1) {
      if (p.pieces) return f(t, c, std::false_type{}, integral_constant<int, kPieces>{});
    }
    f(t, c, std::false_type{}, integral_constant<int, GEN>{});
  };
  if (p.vecs <= 4)
    return lanes(integral_constant<int, 4>{}, integral_constant<int, 1>{});
  if (p.vecs <= 8)
    return lanes(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  if constexpr (VE == 1)
    return;
  else if (p.vecs <= 16)
    lanes(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (p.vecs <= 32)
    lanes(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  else if (p.vecs <= 64)
    lanes(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  else if (p.vecs <= 128)
    lanes(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  else if (p.vecs <= 256)
    lanes(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  else if (p.vecs <= 512)
    lanes(integral_constant<int, 256>{}, integral_constant<int, 2>{});
  else if constexpr (!GEN || ELEM_KIND == kF32)
    lanes(integral_constant<int, 256>{}, integral_constant<int, 4>{});
}
size_t row_lds(const NormArgs& p, int T, int VE, bool grad, bool lanes) {
  const size_t parts = lanes ? 0 : (size_t)(kThreads / T) * (p.entries + p.groups) * sizeof(Pair);
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
  auto launch = [&](auto ve, auto gen, auto past) {
    constexpr int VE = decltype(ve)::value;
    constexpr int GEN = decltype(gen)::value, ONCE = decltype(past)::value;
    if (p.form == kNormRows) {
      by_row<VE, GEN>(p, [&](auto t, auto c, auto lanes, auto entries) {
        constexpr int T = decltype(t)::value, C = decltype(c)::value;
        constexpr bool LANES = decltype(lanes)::value;
        hipLaunchKernelGGL((k_norm_rows<KIND, VE, decltype(entries)::value, T, C, LANES, ONCE>), dim3(p.blocks), dim3(kThreads),
                           row_lds(p, T, VE, false, LANES), st, p);
      });
    } else if (p.form == kNormFrames) {
      hipLaunchKernelGGL((k_norm_frames<KIND, VE, GEN, ONCE>), frame_grid(p), dim3(kThreads), 0, st, p);
    } else {
      hipLaunchKernelGGL((k_norm_stats<KIND, VE, GEN>), slice_grid(p, kGrid), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
      const long all = (long)p.frames * p.groups;
      hipLaunchKernelGGL(k_norm_stats_join, dim3((unsigned)std::min(all, 1L << 20)), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
      hipLaunchKernelGGL((k_norm_apply<KIND, VE, GEN, ONCE>), out_grid(p), dim3(kThreads), 0, st, p);
    }
  };
  by_vec(p, [&](auto ve, auto gen) { with(p.once, [&](auto past) { launch(ve, gen, past); }); });
  DPAMD_LAUNCH_CHECK();
}

template <>
void norm_grad_launch<ELEM_KIND>(hipStream_t st, const NormArgs& p) {
  constexpr int KIND = ELEM_KIND;
  const int channel_blocks = p.dgamma || p.dbeta ? (p.channels + 15) / 16 : 0;
  auto launch = [&](auto ve, auto gen, auto kept, auto past) {
    constexpr int VE = decltype(ve)::value;
    constexpr int GEN = decltype(gen)::value, KEPT = decltype(kept)::value, ONCE = decltype(past)::value;
    int group_blocks = 0;
    long parts = 0;
    if (p.form == kNormRows) {
      by_row<VE, GEN>(p, [&](auto t, auto c, auto lanes, auto entries) {
        constexpr int T = decltype(t)::value, C = decltype(c)::value;
        constexpr bool LANES = decltype(lanes)::value;
        hipLaunchKernelGGL((k_norm_rows_grad<KIND, VE, decltype(entries)::value, T, C, LANES, KEPT, ONCE>), dim3(p.blocks), dim3(kThreads),
                           row_lds(p, T, VE, true, LANES), st, p);
      });
      parts = p.blocks;
    } else if (p.form == kNormFrames) {
      hipLaunchKernelGGL((k_norm_frames_grad<KIND, VE, GEN, KEPT, ONCE>), frame_grid(p), dim3(kThreads), 0, st, p);
      parts = frame_grid(p).y;
    } else {
      hipLaunchKernelGGL((k_norm_sums<KIND, VE, GEN, KEPT>), slice_grid(p, p.blocks), dim3(kThreads), 0, st, p);
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
      hipLaunchKernelGGL((k_norm_dx<KIND, VE, GEN, KEPT, ONCE>), out_grid(p), dim3(kThreads), 0, st, p);
      DPAMD_LAUNCH_CHECK();
    }
  };
  by_vec(p, [&](auto ve, auto gen) {
    with(p.kept != nullptr, [&](auto kept) { with(p.once, [&](auto past) { launch(ve, gen, kept, past); }); });
  });
}

}  // namespace dpamd
