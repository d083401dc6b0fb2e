// groupnorm.hip -- group norm with an activation over rows of channels (channels last), for the graphs of a batch (ragged segments of
// rows, graph_ptr) and for dense samples of equal length (dgcnn_group_norm_fwd, dgcnn_group_norm_bwd).
//
//   per segment and group of D = C / G channels, n rows:   mu = mean x   var = mean (x - mu)^2   r = 1 / sqrt(var + eps)
//   h = (x - mu) r     z = h w + b     y = act(z)
//   q = dy act'(z)     db = sum q      dw = sum q h     a = mean(q w)    c = mean(q w h)     dx = r (q w - a - h c)
//
// Bound: HBM (forward x in, y out; backward x and dy in, dx out).  The tensor is cut into CHUNKS of R rows, R such that a workgroup holds a
// chunk in registers (NV vectors a thread), and every row is read once into registers, whatever the segments' lengths:
//   * a segment of at most R rows belongs to one workgroup: read once, statistics over the registers, written once (a form of the kernel for
//     small tensors streams any length: L, not R, is where a segment counts as long);
//   * a longer segment is the business of the chunks it spans: each leaves its partial (mean, M2) per group -- slot = chunk + segment, unique
//     because (chunk, segment) pairs form a staircase -- and a second launch combines the partials of the segment (a few KB, from L2) and
//     reads its chunk once more (from the last-level cache when the tensor fits it).
// Lengths are known on the device alone, so both run in ONE launch (the workgroups of whole segments and, behind them, those of the chunks), and the second launch
// is left out when the host knows that no segment can be longer than L (few rows, or equal lengths).  Nothing is summed by atomics: every
// sum has one order.
// A thread keeps one column (VEC channels of one group) and every RY-th row; sums over a group go through one LDS slot a thread.
// Statistics, partials and dw / db sums are fp32; y and dx are rounded once.
// Mean and M2 = sum (x - mean)^2 take two sums: m = sum x / n, off by up to K 2^-24 mean|x| after K rounded additions in a row; then, over t = x - m (exact
// where x is near m), S1 = sum t and S2 = sum t^2:  mean = m + S1 / n,  M2 = S2 - S1^2 / n.  What m was off by is in S1, so the mean is left with its
// own rounding: a constant segment's mean is the constant, and small noise on a large offset keeps its variance.  K stays below 200
// forward, 280 backward: a thread sums its 64 (backward 8 a channel) elements of a piece, then the pieces' sums, LDS adds up to 32 and 6 more.  Most pieces: 512 KB of
// 129 16-bit channels, one a thread, 127 of 16 rows forward and 254 of 8 backward.
// Measured (MI355X; a 1 GiB copy reaches 5.2 TB/s): 16 maps of 64 x 64 x 512 bf16, 32 groups, silu, 67 MB a tensor: forward 16 us (reads x, 4.2 TB/s) + 4.5 (join) + 25
// (reads x, writes y, 5.4 TB/s), backward 35 (3.8 TB/s) + 5 + 37 (5.4 TB/s).  2048 graphs of 74 rows on average, 128 bf16 channels, 8 groups, silu, 39 MB a tensor:
// forward 26 + 5 + 11, backward 41 + 6.5 + 22: short segments leave a workgroup's loads and its sums one after the other, three or four workgroups a
// compute unit hide part of it.  3725 rows of 32 fp32 channels, 50 graphs: 8.5 us, one launch.
#include "dg_half.h"

#define GN_T 256             // threads of a workgroup, at least
// ... and at most, which is also how many vectors a group may be wide: 1024 threads leave 128 registers each, which wide vectors' arithmetic
// (w, b, the sums of dw and db) spills
static constexpr int gn_most(int vec) { return vec >= 4 ? 512 : 1024; }
#define GN_CUS 256           // compute units
#define GN_MAX_D 2048        // channels of a group

struct DgGn {
  const void *x, *dy, *w, *b;
  void* out;                     // y or dx
  const int64_t* ptr;            // null: B samples of `per` rows
  float *mean, *rstd;            // [B][G]
  float *part;                   // [chunks + B][G][2]
  float *wpart;                  // [wrows][2][C]
  float *ac;                     // backward, long segments: [B][G][2], the two means
  int64_t N, per, L;             // a segment of more than L rows is split over the workgroups of its chunks
  int B, C, G, D, DV, Gt, CVt, RY, R, P;      // D channels = DV vectors a group; Gt groups (CVt vectors) a workgroup; R = RY * NV rows a chunk; P lanes sum a group
  int nseg;                      // workgroups that own whole segments
  int nchunk, cgrid;             // chunks; workgroups that walk them (0: no segment is split)
  int wdt, act;                  // type of w and b; activation
  float eps;
};

// one vector's arithmetic at a time (one element's where it is an erf): interleaved by the scheduler they spill
#define GN_FENCE() __builtin_amdgcn_sched_barrier(0)

// ---- activation ------------------------------------------------------------------------------------------------------------------
// v_exp_f32 and v_rcp_f32 are good to 1 ulp: exp(-z) carries |z| * 2^-24 * 1.44 of relative error, which the sigmoid's own decay outruns
__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z)); }
__device__ __forceinline__ float gn_tanh(float z) {
  // the quotient form loses the value's own scale near 0; there the Taylor series (next term: 0.009 z^11, below 2^-24 of z for |z| < 0.3)
  const float a = fabsf(z), u = z * z;
  const float e = __builtin_amdgcn_exp2f(-2.8853900817779268f * a);
  const float t = copysignf((1.f - e) * __builtin_amdgcn_rcpf(1.f + e), z);
  const float s = z * (1.f + u * (-0.33333334f + u * (0.13333334f + u * (-0.053968254f + u * 0.021869488f))));
  return a < 0.3f ? s : t;      // (NaN takes t)
}
template <int VEC> __device__ __forceinline__ void gn_act(int act, float* z) {
  switch (act) {
    case DGCNN_ACT_RELU:
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[i] = z[i] > 0.f ? z[i] : z[i] != z[i] ? z[i] : 0.f;
      break;
    case DGCNN_ACT_SILU:
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[i] = z[i] * gn_sigmoid(z[i]);
      break;
    case DGCNN_ACT_GELU:
#pragma unroll
      for (int i = 0; i < VEC; ++i) { z[i] = 0.5f * z[i] * (1.f + erff(z[i] * 0.70710678f)); GN_FENCE(); }
      break;
    case DGCNN_ACT_TANH:
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[i] = gn_tanh(z[i]);
      break;
    default: break;
  }
}
// z -> act'(z)
template <int VEC> __device__ __forceinline__ void gn_slope(int act, float* z) {
  switch (act) {
    case DGCNN_ACT_RELU:
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[i] = z[i] > 0.f ? 1.f : z[i] != z[i] ? z[i] : 0.f;
      break;
    case DGCNN_ACT_SILU:
#pragma unroll
      for (int i = 0; i < VEC; ++i) { const float s = gn_sigmoid(z[i]); z[i] = s * (1.f + z[i] * (1.f - s)); }
      break;
    case DGCNN_ACT_GELU:
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        z[i] = 0.5f * (1.f + erff(z[i] * 0.70710678f)) + z[i] * 0.3989422804f * __builtin_amdgcn_exp2f(-0.72134752f * z[i] * z[i]);
        GN_FENCE();
      }
      break;
    case DGCNN_ACT_TANH:
#pragma unroll
      for (int i = 0; i < VEC; ++i) { const float t = gn_tanh(z[i]); z[i] = (1.f - t) * (1.f + t); }
      break;
    default:
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[i] = 1.f;
  }
}

// ---- segments --------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int64_t gn_uniform(int64_t v) {      // (the same in every lane: into scalar registers)
  return (int64_t)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)((uint64_t)v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
// rows of segment s; whatever ptr holds, the range lies inside [0, N]
__device__ __forceinline__ void gn_range(const DgGn& a, int s, int64_t& lo, int64_t& hi) {
  if (a.ptr) {
    lo = min(max(gn_uniform(a.ptr[s]), (int64_t)0), a.N);
    hi = min(max(gn_uniform(a.ptr[s + 1]), lo), a.N);
  } else {
    lo = (int64_t)s * a.per;
    hi = lo + a.per;
  }
}
// the segment that row r lies in (-1: in front of the first; B: behind the last), found by the whole wave: 64 probes a step
__device__ __forceinline__ int gn_find(const DgGn& a, int64_t r) {
  if (!a.ptr) return (r | a.per) >> 31 ? (int)(r / a.per) : (int)((unsigned)r / (unsigned)a.per);
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = a.B + 1;
  while (lo < hi) {
    const int64_t step = (hi - lo + 63) >> 6, at = lo + lane * step;
    const int n = __popcll(__ballot(at < hi && a.ptr[min(at, (int64_t)a.B)] <= r));
    if (n == 0) break;
    hi = min(hi, lo + (int64_t)n * step);
    lo += (int64_t)(n - 1) * step + 1;
  }
  return (int)lo - 1;
}

template <int CTRL> __device__ __forceinline__ float gn_dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
// ---- sums over a group -----------------------------------------------------------------------------------------------------------
struct GnLds { float red[2][1024]; float stat[2][1024]; };
struct GnLane {
  int t, r, c, g, slot;      // row and vector column inside the chunk, group inside the workgroup's, LDS slot (a group's slots are contiguous)
  unsigned off;              // of the thread's vector in row block 0
  bool on;                   // the thread owns a column (else r lies behind every row)
};
// x summed over P = 1, 4, 16 or 64 neighbouring lanes, the sum in all of them
__device__ __forceinline__ float gn_lanes(float x, int P) {
  if (P >= 4) { x += gn_dpp<0xB1>(x); x += gn_dpp<0x4E>(x); }              // quad_perm [1 0 3 2], [2 3 0 1]
  if (P >= 16) { x += gn_dpp<0x124>(x); x += gn_dpp<0x128>(x); }           // row_ror 4, 8
  if (P >= 64) { x += __shfl_xor(x, 16); x += __shfl_xor(x, 32); }
  return x;
}
// every thread's u (and v) summed over its group -> L.stat[0/1][group].  Two barriers a sum; the first one of the next sum is what keeps this one's
// results in place until everyone has read them.  P lanes add a group's slots: few enough that each has several reads in flight.
template <bool TWO> __device__ __forceinline__ void gn_sum(const DgGn& a, GnLds& L, const GnLane& me, int gn, float u, float v) {
  if (me.on) { L.red[0][me.slot] = u; if (TWO) L.red[1][me.slot] = v; }
  __syncthreads();
  const int items = a.RY * a.DV, g = me.t / a.P, l = me.t & (a.P - 1);
  float su = 0.f, sv = 0.f;
  if (g < gn) {
#pragma unroll 4
    for (int j = l; j < items; j += a.P) { su += L.red[0][g * items + j]; if (TWO) sv += L.red[1][g * items + j]; }
  }
  su = gn_lanes(su, a.P);
  if (TWO) sv = gn_lanes(sv, a.P);
  if (g < gn && l == 0) { L.stat[0][g] = su; if (TWO) L.stat[1][g] = sv; }
  __syncthreads();
}

template <class D, int VEC> __device__ __forceinline__ void gn_zero_rows(const DgGn& a, const GnLane& me, int64_t lo, int64_t hi) {
  for (int64_t at = lo; at < hi; at += a.RY)
    if (me.r < hi - at) dg_store<D, VEC>(static_cast<typename D::S*>(a.out) + at * a.C + me.off, dg_zero<D, VEC>());
}

template <int VEC> __device__ __forceinline__ void gn_load_w(const void* p, int dt, bool on, int ch, float absent, float* w) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) w[i] = absent;
  if (!p || !on) return;
  if (dt == DGCNN_F32) {      // (the branch outside the elements: their loads become one)
    const float* const q = static_cast<const float*>(p) + ch;
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] = q[i];
  } else if (dt == DGCNN_BF16) {
    const uint16_t* const q = static_cast<const uint16_t*>(p) + ch;
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] = DgBF16::to(q[i]);
  } else {
    const uint16_t* const q = static_cast<const uint16_t*>(p) + ch;
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] = DgF16::to(q[i]);
  }
}

#define GN_SETUP()                                                                                                     \
  const int g0 = blockIdx.y * a.Gt, gn = min(a.Gt, a.G - g0);                                                          \
  GnLane me;                                                                                                           \
  me.t = threadIdx.x; me.r = me.t / a.CVt; me.c = me.t - me.r * a.CVt; me.g = me.c / a.DV;                             \
  me.on = me.r < a.RY && me.g < gn;                                                                                    \
  me.slot = me.g * (a.RY * a.DV) + me.r * a.DV + (me.c - me.g * a.DV);                                                 \
  const int ch = (g0 * a.DV + me.c) * VEC;      /* first channel of the thread */                                      \
  me.off = (unsigned)me.r * a.C + ch;                                                                                  \
  if (!me.on) me.r = 1 << 30;                                                                                          \
  typedef typename D::S S;                                                                                             \
  const S* const x = static_cast<const S*>(a.x);                                                                       \
  S* const out = static_cast<S*>(a.out);                                                                               \
  float w[VEC], b[VEC];                                                                                                \
  gn_load_w<VEC>(a.w, a.wdt, me.on, ch, 1.f, w);                                                                       \
  gn_load_w<VEC>(a.b, a.wdt, me.on, ch, 0.f, b);                                                                       \
  (void)x; (void)out; (void)b; (void)ch

// Rows are addressed as (uniform base of the row block i RY) + (the thread's own 32-bit offset): a 64-bit address a row and thread would take
// more registers than the rows.  `left` rows are there; a thread without a column has r beyond every `left`.
template <class D, int VEC, int NV> __device__ __forceinline__ void gn_load(const DgGn& a, const GnLane& me, const typename D::S* p, int64_t at, int left, DgRaw<D, VEC>* v) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i] = dg_zero<D, VEC>();
    if (me.r < left - i * a.RY) v[i] = dg_load<D, VEC>(p + (at + (int64_t)i * a.RY) * a.C + me.off);
  }
}
// What does not fit the registers passes through them R rows at a time: f(at, left) for each piece
template <class F> __device__ __forceinline__ void gn_pieces(const DgGn& a, int64_t lo, int64_t hi, F f) {
#pragma unroll 1
  for (int64_t at = lo; at < hi; at += a.R) f(at, (int)min(hi - at, (int64_t)a.R));
}

// x - mu is kept apart from the scale: a constant segment, whose mean is the constant, gives exactly b, and a large mean cancels before anything is
// rounded.  rw = rstd * w.
template <class D, int VEC> __device__ __forceinline__ DgRaw<D, VEC> gn_apply(const DgGn& a, const DgRaw<D, VEC>& v, float mu, const float* rw, const float* b) {
  float z[VEC];
  DgRaw<D, VEC> o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) z[e] = __builtin_fmaf(v.get(e) - mu, rw[e], b[e]);
  gn_act<VEC>(a.act, z);
#pragma unroll
  for (int e = 0; e < VEC; ++e) o.set(e, z[e]);
  return o;
}

// What a workgroup of the first launch works on, one item after the other: segments q, q + 1, ... < end (whole, slot < 0), or the rows of long
// segments inside the chunks k, k + cgrid, ...
struct GnWork {
  int64_t lo, hi;
  int s, slot;
  int next, end, k;
  __device__ __forceinline__ GnWork(const DgGn& a) {
    if ((int)blockIdx.x < a.nseg) {
      next = (int)((int64_t)blockIdx.x * a.B / a.nseg); end = (int)((int64_t)(blockIdx.x + 1) * a.B / a.nseg) - 1; k = -1;
    } else {
      next = 0; end = -1; k = (int)blockIdx.x - a.nseg - a.cgrid;
    }
  }
  // the next item with rows; false: done.  Uniform over the workgroup.  `empty(s)` is called for a segment without rows.
  template <class Z> __device__ __forceinline__ bool fetch(const DgGn& a, Z empty) {
    for (;;) {
      if ((int)blockIdx.x < a.nseg) {
        if (next > end) return false;
        s = next++; slot = -1;
        gn_range(a, s, lo, hi);
        if (lo == hi) { empty(s); continue; }
        if (hi - lo > a.L) continue;
        return true;
      }
      if (next > end) {
        k += a.cgrid;
        if (k >= a.nchunk) return false;
        const int64_t r0 = (int64_t)k * a.R, r1 = min(r0 + a.R, a.N);
        next = max(gn_find(a, r0), 0); end = min(gn_find(a, r1 - 1), a.B - 1);
        continue;
      }
      s = next; slot = k + s;
      next = s < end ? end : end + 1;      // (a segment longer than a chunk is the chunk's first or its last)
      gn_range(a, s, lo, hi);
      if (hi - lo <= a.L) continue;
      lo = max(lo, (int64_t)k * a.R); hi = min(hi, (int64_t)(k + 1) * a.R);
      if (lo < hi) return true;
    }
  }
};
// without a second launch, the rows outside every segment are cleared by the workgroups of the first and the last one
template <class D, int VEC> __device__ __forceinline__ void gn_clear(const DgGn& a, const GnLane& me) {
  if (a.cgrid) return;
  int64_t lo, hi;
  if (blockIdx.x == 0) { gn_range(a, 0, lo, hi); gn_zero_rows<D, VEC>(a, me, 0, lo); }
  if ((int)blockIdx.x == a.nseg - 1) { gn_range(a, a.B - 1, lo, hi); gn_zero_rows<D, VEC>(a, me, hi, a.N); }
}

// forward: whole segments, and the partial moments of the chunks of long ones.  More than R rows (a few long segments, no second launch) pass
// through the registers piece by piece, read again for each of the three passes.
template <class D, int VEC, int NV, bool STREAM>
__global__ void __launch_bounds__(gn_most(VEC))
k_gn_fwd(const DgGn a) {
  __shared__ GnLds L;
  GN_SETUP();
  DgRaw<D, VEC> v[NV];
  gn_clear<D, VEC>(a, me);
  GnWork it(a);
  while (it.fetch(a, [&](int s) {
    if (me.t < gn) { a.mean[(int64_t)s * a.G + g0 + me.t] = 0.f; a.rstd[(int64_t)s * a.G + g0 + me.t] = 0.f; }
  })) {
    const int left = (int)min(it.hi - it.lo, (int64_t)a.R);
    const float n = (float)(it.hi - it.lo) * (float)a.D;
    float sum = 0.f, t1 = 0.f, t2 = 0.f;
    if constexpr (!STREAM) {
      gn_load<D, VEC, NV>(a, me, x, it.lo, left, v);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += v[i].get(e);
    } else {
      gn_pieces(a, it.lo, it.hi, [&](int64_t at, int left) {
        DgRaw<D, VEC> u[NV];
        gn_load<D, VEC, NV>(a, me, x, at, left, u);
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) s += u[i].get(e);
        sum += s;
      });
    }
    gn_sum<false>(a, L, me, gn, sum, 0.f);
    if constexpr (!STREAM) dg_hide<D, VEC, NV>(v);
    float mu = me.on ? L.stat[0][me.g] / n : 0.f;
    if constexpr (!STREAM) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (me.r < left - i * a.RY) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) { const float t = v[i].get(e) - mu; t1 += t; t2 += t * t; }
        }
    } else {
      gn_pieces(a, it.lo, it.hi, [&](int64_t at, int left) {
        DgRaw<D, VEC> u[NV];
        gn_load<D, VEC, NV>(a, me, x, at, left, u);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
          if (me.r < left - i * a.RY) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) { const float t = u[i].get(e) - mu; s1 += t; s2 += t * t; }
          }
        t1 += s1; t2 += s2;
      });
    }
    gn_sum<true>(a, L, me, gn, t1, t2);
    float m2 = 0.f;
    if (me.on) {
      const float off = L.stat[0][me.g] / n;
      mu += off;
      m2 = L.stat[1][me.g] - L.stat[0][me.g] * off;
      m2 = m2 < 0.f ? 0.f : m2;      // (rounding, where all of S2 was m's error; NaN stays)
    }
    if constexpr (!STREAM) dg_hide<D, VEC, NV>(v);
    const bool first = me.r == 0 && me.c == me.g * a.DV;      // one thread of each group
    if (it.slot >= 0) {
      if (first) {
        float* const p = a.part + ((int64_t)it.slot * a.G + g0 + me.g) * 2;
        p[0] = mu; p[1] = m2;
      }
      continue;
    }
    const float rs = me.on ? 1.f / sqrtf(m2 / n + a.eps) : 0.f;
    if (first) { a.mean[(int64_t)it.s * a.G + g0 + me.g] = mu; a.rstd[(int64_t)it.s * a.G + g0 + me.g] = rs; }
    float rw[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) rw[e] = rs * w[e];
    if constexpr (!STREAM) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (me.r < left - i * a.RY) dg_store<D, VEC>(out + (it.lo + (int64_t)i * a.RY) * a.C + me.off, gn_apply<D, VEC>(a, v[i], mu, rw, b));
        GN_FENCE();
      }
    } else {
      gn_pieces(a, it.lo, it.hi, [&](int64_t at, int left) {
        DgRaw<D, VEC> u[NV];
        gn_load<D, VEC, NV>(a, me, x, at, left, u);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (me.r < left - i * a.RY) dg_store<D, VEC>(out + (at + (int64_t)i * a.RY) * a.C + me.off, gn_apply<D, VEC>(a, u[i], mu, rw, b));
          GN_FENCE();
        }
      });
    }
  }
}

// ---- long segments: the partials of a segment's chunks, then its rows once more -----------------------------------------------------
// 64 lanes a (segment, group) where there are at most 4096 of them, else 16 (backward, with the sum of dw and db: 512 of 256 partials 5.2 us, with 16 lanes
// 9.9; 16384, most of them of none, 7.9 and 6.3).  Forward: mean = mean_0 + sum n_i (mean_i - mean_0) / n (equal means stay what they are), M2 = sum M2_i +
// n_i (mean_i - mean)^2 -> mean, rstd.  Backward: the two means -> ac.
__host__ __device__ inline int gn_join_lanes(const DgGn& a) { return (int64_t)a.B * a.G <= 4096 ? 64 : 16; }
template <bool BWD> __device__ __forceinline__ void gn_join(const DgGn& a, int64_t thread) {
  const int lanes = gn_join_lanes(a), l = (int)thread & (lanes - 1);
  const int64_t item = thread / lanes;
  const int s = (int)(item / a.G), g = (int)(item % a.G);
  int64_t lo = 0, hi = 0;
  if (s < a.B) {
    if (a.ptr) { lo = min(max(a.ptr[s], (int64_t)0), a.N); hi = min(max(a.ptr[s + 1], lo), a.N); }
    else { lo = (int64_t)s * a.per; hi = lo + a.per; }
  }
  const bool on = hi - lo > a.L;
  const int k0 = (int)(lo / a.R), n = on ? (int)((hi - 1) / a.R) - k0 + 1 : 0;
  const float* const p = a.part + ((int64_t)(k0 + s) * a.G + g) * 2;
  const float rows = (float)(hi - lo);
  float u = 0.f, v = 0.f;
  if (BWD) {
#pragma unroll 4
    for (int i = l; i < n; i += lanes) { u += p[(int64_t)i * a.G * 2]; v += p[(int64_t)i * a.G * 2 + 1]; }
    u = gn_lanes(u, lanes); v = gn_lanes(v, lanes);
    if (on && l == 0) {
      a.ac[((int64_t)s * a.G + g) * 2] = u / (rows * (float)a.D);
      a.ac[((int64_t)s * a.G + g) * 2 + 1] = v / (rows * (float)a.D);
    }
    return;
  }
  const float m0 = on ? p[0] : 0.f;
#pragma unroll 4
  for (int i = l; i < n; i += lanes)
    u += (p[(int64_t)i * a.G * 2] - m0) * (float)(min((int64_t)(k0 + i + 1) * a.R, hi) - max((int64_t)(k0 + i) * a.R, lo));
  u = gn_lanes(u, lanes);
  const float m = m0 + u / rows;
#pragma unroll 4
  for (int i = l; i < n; i += lanes) {
    const float d = p[(int64_t)i * a.G * 2] - m;
    v += p[(int64_t)i * a.G * 2 + 1] + (float)(min((int64_t)(k0 + i + 1) * a.R, hi) - max((int64_t)(k0 + i) * a.R, lo)) * (float)a.D * d * d;
  }
  v = gn_lanes(v, lanes);
  if (on && l == 0) {
    a.mean[(int64_t)s * a.G + g] = m;
    a.rstd[(int64_t)s * a.G + g] = 1.f / sqrtf(v / rows / (float)a.D + a.eps);
  }
}
__global__ void __launch_bounds__(256) k_gn_join(const DgGn a) { gn_join<false>(a, (int64_t)blockIdx.x * 256 + threadIdx.x); }

// rows [at0, at1) of long segment s; ROWS(at, left) for each R of them
template <class F> __device__ __forceinline__ void gn_long_rows(const DgGn& a, int k, F rows) {
  const int64_t r0 = (int64_t)k * a.R, r1 = min(r0 + a.R, a.N);
  const int s0 = max(gn_find(a, r0), 0), s1 = min(gn_find(a, r1 - 1), a.B - 1);
  for (int s = s0; s <= s1; s = s < s1 ? s1 : s1 + 1) {
    int64_t lo, hi;
    gn_range(a, s, lo, hi);
    if (hi - lo <= a.L) continue;
    lo = max(lo, r0); hi = min(hi, r1);
    if (lo < hi) rows(s, lo, (int)(hi - lo));
  }
}
// the chunk's rows that lie in no segment -> 0
template <class D, int VEC> __device__ __forceinline__ void gn_clear_chunk(const DgGn& a, const GnLane& me, int k) {
  if (!a.ptr) return;
  const int64_t r0 = (int64_t)k * a.R, r1 = min(r0 + a.R, a.N);
  int64_t lo, hi, u;
  gn_range(a, 0, lo, u);
  gn_range(a, a.B - 1, u, hi);
  if (r0 < lo) gn_zero_rows<D, VEC>(a, me, r0, min(lo, r1));
  if (hi < r1) gn_zero_rows<D, VEC>(a, me, max(hi, r0), r1);
}
template <class D, int VEC, int NV>
__global__ void __launch_bounds__(gn_most(VEC))
k_gn_fwd_long(const DgGn a) {
  GN_SETUP();
  gn_clear_chunk<D, VEC>(a, me, blockIdx.x);
  gn_long_rows(a, blockIdx.x, [&](int s, int64_t at, int left) {
    DgRaw<D, VEC> v[NV];
    gn_load<D, VEC, NV>(a, me, x, at, left, v);
    const float mu = me.on ? a.mean[(int64_t)s * a.G + g0 + me.g] : 0.f, rs = me.on ? a.rstd[(int64_t)s * a.G + g0 + me.g] : 0.f;
    float rw[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) rw[e] = rs * w[e];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (me.r < left - i * a.RY) dg_store<D, VEC>(out + (at + (int64_t)i * a.RY) * a.C + me.off, gn_apply<D, VEC>(a, v[i], mu, rw, b));
      GN_FENCE();
    }
  });
}

// ---- backward --------------------------------------------------------------------------------------------------------------------
// With t = x - mu, h = t rstd:  q = dy act'(t rw + b);  over a segment's rows, per channel, sq = sum q and sqt = sum q t give everything: db = sq, dw = rstd sqt,
// and over a group's channels a = sum w sq / n, c = rstd sum w sqt / n.   dx = rw q - rstd a - t (rstd^2 c) = rw q - A - t B
template <class D, int VEC> __device__ __forceinline__ void gn_q(const DgGn& a, const DgRaw<D, VEC>& x, const DgRaw<D, VEC>& dy, float mu, const float* rw, const float* b, float* q) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) q[e] = __builtin_fmaf(x.get(e) - mu, rw[e], b[e]);
  gn_slope<VEC>(a.act, q);
#pragma unroll
  for (int e = 0; e < VEC; ++e) q[e] *= dy.get(e);
}
template <class D, int VEC> __device__ __forceinline__ DgRaw<D, VEC> gn_dx(const DgRaw<D, VEC>& x, float mu, const float* q, const float* rw, float A, float B) {
  DgRaw<D, VEC> o;
#pragma unroll
  for (int e = 0; e < VEC; ++e) o.set(e, __builtin_fmaf(q[e], rw[e], -__builtin_fmaf(x.get(e) - mu, B, A)));
  return o;
}
template <class D, int VEC> __device__ __forceinline__ void gn_add(const DgRaw<D, VEC>& x, float mu, const float* q, float* sq, float* sqt) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) { sq[e] += q[e]; sqt[e] = __builtin_fmaf(q[e], x.get(e) - mu, sqt[e]); }
}
// the workgroup's dw, db sums -> its row of wpart
template <int VEC> __device__ __forceinline__ void gn_put_w(const DgGn& a, GnLds& L, const GnLane& me, int gn, int ch, const float* dw, const float* db) {
  float* const row = a.wpart + (int64_t)blockIdx.x * 2 * a.C;
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    __syncthreads();
    if (me.on) { L.red[0][me.t] = dw[e]; L.red[1][me.t] = db[e]; }
    __syncthreads();
    if (me.on && me.r == 0) {
      float u = 0.f, v = 0.f;
      for (int r = 0; r < a.RY; ++r) { u += L.red[0][r * a.CVt + me.t]; v += L.red[1][r * a.CVt + me.t]; }
      row[ch + e] = u; row[a.C + ch + e] = v;
    }
  }
}

// backward: whole segments (each workgroup walks a contiguous share of them), and the partial sums of the chunks of long ones
template <class D, int VEC, int NV, bool STREAM>
__global__ void __launch_bounds__(gn_most(VEC))
k_gn_bwd(const DgGn a) {
  __shared__ GnLds L;
  GN_SETUP();
  const S* const dy = static_cast<const S*>(a.dy);
  float dw[VEC], db[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) dw[e] = db[e] = 0.f;
  gn_clear<D, VEC>(a, me);
  GnWork it(a);
  while (it.fetch(a, [](int) {})) {
    const int left = (int)min(it.hi - it.lo, (int64_t)a.R);
    const float inv_n = 1.f / ((float)(it.hi - it.lo) * (float)a.D);
    const float mu = me.on ? a.mean[(int64_t)it.s * a.G + g0 + me.g] : 0.f;
    const float rs = me.on ? a.rstd[(int64_t)it.s * a.G + g0 + me.g] : 0.f;
    float rw[VEC], sq[VEC], sqt[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { rw[e] = rs * w[e]; sq[e] = sqt[e] = 0.f; }
    DgRaw<D, VEC> v[NV];
    float q[NV][VEC];      // (kept over the sum: the activation's slope costs more than anything else here)
    if constexpr (!STREAM) {
      DgRaw<D, VEC> d[NV];
      gn_load<D, VEC, NV>(a, me, x, it.lo, left, v);
      gn_load<D, VEC, NV>(a, me, dy, it.lo, left, d);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i * a.RY >= left) continue;      // (uniform: whole row blocks that are not there; a missing row of the last one has dy = 0, q = 0)
        gn_q<D, VEC>(a, v[i], d[i], mu, rw, b, q[i]);
        gn_add<D, VEC>(v[i], mu, q[i], sq, sqt);
        GN_FENCE();
      }
    } else {
      gn_pieces(a, it.lo, it.hi, [&](int64_t at, int left) {
        DgRaw<D, VEC> d[NV];
        gn_load<D, VEC, NV>(a, me, x, at, left, v);
        gn_load<D, VEC, NV>(a, me, dy, at, left, d);
        float pq[VEC], pqt[VEC];      // (the piece's sums apart: fewer additions in a row)
#pragma unroll
        for (int e = 0; e < VEC; ++e) pq[e] = pqt[e] = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (me.r < left - i * a.RY) {
            gn_q<D, VEC>(a, v[i], d[i], mu, rw, b, q[i]);
            gn_add<D, VEC>(v[i], mu, q[i], pq, pqt);
          }
          GN_FENCE();
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) { sq[e] += pq[e]; sqt[e] += pqt[e]; }
      });
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      s1 += w[e] * sq[e]; s2 += rw[e] * sqt[e];
      db[e] += sq[e]; dw[e] += rs * sqt[e];
    }
    gn_sum<true>(a, L, me, gn, s1, s2);
    if (it.slot >= 0) {
      if (me.t < gn) {
        float* const p = a.part + ((int64_t)it.slot * a.G + g0 + me.t) * 2;
        p[0] = L.stat[0][me.t]; p[1] = L.stat[1][me.t];
      }
      continue;
    }
    const float A = me.on ? rs * (L.stat[0][me.g] * inv_n) : 0.f, B = me.on ? rs * rs * (L.stat[1][me.g] * inv_n) : 0.f;
    if constexpr (!STREAM) {
      dg_hide<D, VEC, NV>(v);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (me.r < left - i * a.RY) dg_store<D, VEC>(out + (it.lo + (int64_t)i * a.RY) * a.C + me.off, gn_dx<D, VEC>(v[i], mu, q[i], rw, A, B));
        GN_FENCE();
      }
    } else {
      gn_pieces(a, it.lo, it.hi, [&](int64_t at, int left) {
        DgRaw<D, VEC> d[NV];
        gn_load<D, VEC, NV>(a, me, x, at, left, v);
        gn_load<D, VEC, NV>(a, me, dy, at, left, d);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          if (me.r < left - i * a.RY) {
            gn_q<D, VEC>(a, v[i], d[i], mu, rw, b, q[i]);
            dg_store<D, VEC>(out + (at + (int64_t)i * a.RY) * a.C + me.off, gn_dx<D, VEC>(v[i], mu, q[i], rw, A, B));
          }
          GN_FENCE();
        }
      });
    }
  }
  if (a.wpart) gn_put_w<VEC>(a, L, me, gn, ch, dw, db);
}

template <class D, int VEC, int NV>
__global__ void __launch_bounds__(gn_most(VEC))
k_gn_bwd_long(const DgGn a) {
  GN_SETUP();
  const S* const dy = static_cast<const S*>(a.dy);
  gn_clear_chunk<D, VEC>(a, me, blockIdx.x);
  gn_long_rows(a, blockIdx.x, [&](int s, int64_t at, int left) {
    DgRaw<D, VEC> v[NV], d[NV];
    gn_load<D, VEC, NV>(a, me, x, at, left, v);
    gn_load<D, VEC, NV>(a, me, dy, at, left, d);
    const int64_t sg = (int64_t)s * a.G + g0 + me.g;
    const float mu = me.on ? a.mean[sg] : 0.f, rs = me.on ? a.rstd[sg] : 0.f;
    const float A = me.on ? rs * a.ac[2 * sg] : 0.f, B = me.on ? rs * rs * a.ac[2 * sg + 1] : 0.f;
    float rw[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) rw[e] = rs * w[e];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (me.r < left - i * a.RY) {
        float q[VEC];
        gn_q<D, VEC>(a, v[i], d[i], mu, rw, b, q);
        dg_store<D, VEC>(out + (at + (int64_t)i * a.RY) * a.C + me.off, gn_dx<D, VEC>(v[i], mu, q, rw, A, B));
      }
      GN_FENCE();
    }
  });
}

// dw, db: the workgroups' rows summed column by column, in a fixed order (8 columns x 128 row lanes a workgroup); the workgroups behind those
// combine the partial sums of long segments
__global__ void __launch_bounds__(1024)
k_gn_wsum(const DgGn a, int rows, int wblocks, void* dw, void* db, int dt) {
  __shared__ float red[128][9];
  if ((int)blockIdx.x >= wblocks) {
    gn_join<true>(a, (int64_t)(blockIdx.x - wblocks) * 1024 + threadIdx.x);
    return;
  }
  const int c = threadIdx.x & 7, col = blockIdx.x * 8 + c, lane = threadIdx.x >> 3;
  float s = 0.f;
  if (col < 2 * a.C) {
    const float* const p = a.wpart + col;
#pragma unroll 16
    for (int r = lane; r < rows; r += 128) s += p[(int64_t)r * 2 * a.C];
  }
  red[lane][c] = s;
  __syncthreads();
  for (int o = 64; o; o >>= 1) {
    if (lane < o) red[lane][c] += red[lane + o][c];
    __syncthreads();
  }
  if (lane == 0 && col < 2 * a.C) {
    void* const out = col < a.C ? dw : db;
    if (out) dg_store_as(out, col < a.C ? col : col - a.C, dt, red[0][c]);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
// vectors a thread holds: 8 of x (of up to 16 bytes) forward, 16 where they are one register or half of one; 8 of x and dy (of up to 8 bytes) backward
static constexpr int gn_nv(int vec_bytes, bool bwd) { return bwd ? 8 : vec_bytes <= 4 ? 16 : 8; }

// everything that follows from the shape; false: the shape is outside what this build handles
static bool gn_plan(DgGn* a, int dtype, int vec_cap, bool bwd, int* vec, int* threads, int* tiles) {
  // (backward: 8-byte vectors.  16-byte ones take 171 registers with w, b and the sums of dw and db, two waves a SIMD: 115 us against 49 for the
  // first launch of 2048 graphs of 128 bf16 channels)
  const int full = (dtype == DGCNN_F32 ? 4 : 8) >> bwd;
  int v = full < vec_cap ? full : vec_cap;
  while (a->D % v) v >>= 1;
  a->DV = a->D / v;
  const int most = gn_most(v);
  if (a->DV > most || a->D > GN_MAX_D) return false;
  const int nv = gn_nv(v * dg_dtype_size(dtype), bwd), cols = a->DV * a->G;
  int t = GN_T;
  while (t < most && (a->DV > t || cols > t)) t *= 2;      // one column tile if the threads suffice
  a->Gt = cols <= t ? a->G : t / a->DV;
  // (512 threads, or fewer groups a workgroup, hold segments twice as long: fewer of them are split, but fewer workgroups are resident.  2048 graphs of 74
  // rows on average, 128 bf16 channels: backward 79 us as it is, 89 with half the groups, 160 with both; forward 44, 43, 43)
  a->CVt = a->Gt * a->DV;
  a->RY = t / a->CVt;
  a->R = a->RY * nv;
  const int items = a->RY * a->DV;
  a->P = items <= 64 ? 4 : items <= 512 ? 16 : 64;
  while (a->P > 1 && a->P * a->Gt > t) a->P >>= 2;
  *vec = v; *threads = t; *tiles = (a->G + a->Gt - 1) / a->Gt;
  return true;
}
// which workgroups run: see the head of the file
static void gn_grid(DgGn* a, int es, bool bwd) {
  // Up to 512 KB in all no split is worth its two more launches (4 us each): any segment then passes through its workgroup (STREAM), read again
  // for each sum out of the caches.
  a->L = a->N * a->C * es <= 512 * 1024 && (a->ptr ? a->N : a->per) > a->R ? a->N : a->R;
  const bool one_long = (a->ptr ? a->N : a->per) > a->L;      // can any segment be longer?
  // Workgroups of a role: three of 256 threads fit a compute unit backward (141 registers), four forward.  Up to four each, one item a workgroup; beyond
  // that as many as fit at once, each with a contiguous share or every cgrid-th chunk.  2048 graphs of 128 bf16 channels: backward 41 us with 768, 45 with 1024,
  // 49 with 2048 (and the sum of their partial rows 6, 7, 9); forward 25.6 with 1024, 27.9 with 2048; 16 x 4096 rows of 512: backward 35, 42 with 1024, forward 16.4, 18.7.
  const int all = GN_CUS * 4, most = GN_CUS * (bwd ? 3 : 4);
  a->nseg = one_long && !a->ptr ? 0 : a->B <= all ? a->B : most;      // (dense samples: all or none)
  a->nchunk = one_long ? (int)((a->N + a->R - 1) / a->R) : 0;
  a->cgrid = a->nchunk <= all ? a->nchunk : most;
}
static bool gn_shape(DgGn* a, int64_t rows, int C, int groups, int segments) {
  if (rows < 0 || C < 1 || groups < 1 || C % groups || segments < 0) return false;
  a->N = rows; a->B = segments; a->C = C; a->G = groups; a->D = C / groups;
  return true;
}
// counts of 32 bits: chunks hold at least 2^10 of 2^40 elements, the joins take 16 threads a (segment, group)
static bool gn_fits(const DgGn& a) {
  return a.N <= ((int64_t)1 << 40) / a.C && a.C <= 1 << 24 && (int64_t)a.B * a.G <= 1 << 27;
}
static int64_t gn_part_bytes(const DgGn& a) { return a.nchunk ? dg_align(((int64_t)a.nchunk + a.B) * a.G * 2 * 4, 256) : 0; }
static int64_t gn_ac_bytes(const DgGn& a) { return a.nchunk ? dg_align((int64_t)a.B * a.G * 2 * 4, 256) : 0; }

// the plan of a call; alignment of the tensors (a multiple of the vector's bytes) is known at the call only, so the workspace is for the worst
extern "C" int64_t dgcnn_group_norm_workspace_bytes(int64_t rows, int C, int groups, int segments, int dense, int dtype, int backward) {
  DgGn a = {};
  if (!gn_shape(&a, rows, C, groups, segments) || !dg_dtype_ok(dtype)) return DGCNN_EINVAL;
  if (segments == 0 || rows == 0) return 256;
  if (!gn_fits(a)) return DGCNN_EUNSUPPORTED;
  static const int64_t dummy[2] = {0, 0};
  int64_t most = 256;
  for (int cap = 8; cap >= 1; cap >>= 1) {
    int v, t, n;
    a.ptr = dense ? nullptr : dummy;
    a.per = dense ? rows / segments : 0;
    if (!gn_plan(&a, dtype, cap, backward != 0, &v, &t, &n)) continue;
    gn_grid(&a, dg_dtype_size(dtype), backward != 0);
    const int64_t b = gn_part_bytes(a) + (backward ? gn_ac_bytes(a) + dg_align(((int64_t)a.nseg + a.cgrid) * 2 * C * 4, 256) : 0);
    if (b > most) most = b;
  }
  return most;
}

typedef void (*gn_kernel)(const DgGn);
enum { GN_FWD, GN_FWD_STREAM, GN_FWD_LONG, GN_BWD, GN_BWD_STREAM, GN_BWD_LONG };
template <class D, int VEC> static gn_kernel gn_pick(int which) {
  constexpr int F = gn_nv(VEC * sizeof(typename D::S), false), W = gn_nv(VEC * sizeof(typename D::S), true);
  switch (which) {
    case GN_FWD: return (gn_kernel)k_gn_fwd<D, VEC, F, false>;
    case GN_FWD_STREAM: return (gn_kernel)k_gn_fwd<D, VEC, F, true>;
    case GN_FWD_LONG: return (gn_kernel)k_gn_fwd_long<D, VEC, F>;
  }
  if constexpr (VEC < D::FULL) {      // (backward: vectors of up to 8 bytes)
    switch (which) {
      case GN_BWD: return (gn_kernel)k_gn_bwd<D, VEC, W, false>;
      case GN_BWD_STREAM: return (gn_kernel)k_gn_bwd<D, VEC, W, true>;
      case GN_BWD_LONG: return (gn_kernel)k_gn_bwd_long<D, VEC, W>;
    }
  }
  return nullptr;
}
template <class D> static gn_kernel gn_pick_vec(int vec, int which) {
  if constexpr (D::FULL == 8) { if (vec == 8) return gn_pick<D, 8>(which); }
  return vec == 4 ? gn_pick<D, 4>(which) : vec == 2 ? gn_pick<D, 2>(which) : gn_pick<D, 1>(which);
}
static gn_kernel gn_pick_dtype(int dtype, int vec, int which) {
  return dtype == DGCNN_F32 ? gn_pick_vec<DgF32>(vec, which) : dtype == DGCNN_BF16 ? gn_pick_vec<DgBF16>(vec, which) : gn_pick_vec<DgF16>(vec, which);
}
// largest vector (in elements) that every address in `low` and the row length admit
static int gn_vec_cap(uintptr_t low, int C, int es) {
  int v = 16 / es;
  while (v > 1 && ((low & (uintptr_t)(v * es - 1)) || C % v)) v >>= 1;
  return v;
}
static int gn_check(const dgcnn_group_norm_args* p, DgGn* a) {
  if (!p || !gn_shape(a, p->rows, p->channels, p->groups, p->segments)) return DGCNN_EINVAL;
  if (!dg_dtype_ok(p->dtype) || ((p->weight || p->bias) && !dg_dtype_ok(p->weight_dtype))) return DGCNN_EINVAL;
  if (p->act < DGCNN_ACT_NONE || p->act > DGCNN_ACT_TANH || !(p->eps >= 0.f)) return DGCNN_EINVAL;
  if (p->rows > 0 && p->segments > 0 && (!p->x || !p->mean || !p->rstd)) return DGCNN_EINVAL;
  if (!p->ptr && p->segments > 0 && p->rows % p->segments) return DGCNN_EINVAL;
  if (!p->ptr && p->segments == 0 && p->rows > 0) return DGCNN_EINVAL;
  if (!gn_fits(*a)) return DGCNN_EUNSUPPORTED;
  a->x = p->x; a->w = p->weight; a->b = p->bias; a->ptr = p->ptr; a->mean = p->mean; a->rstd = p->rstd;
  a->per = !p->ptr && p->segments ? p->rows / p->segments : 0;
  a->wdt = p->weight_dtype; a->act = p->act; a->eps = p->eps;
  return DGCNN_OK;
}

extern "C" int dgcnn_group_norm_fwd(const dgcnn_group_norm_args* p, void* y, void* ws, dgcnn_stream_t stream) {
  DgGn a = {};
  const int rc = gn_check(p, &a);
  if (rc != DGCNN_OK) return rc;
  if (p->rows == 0 || p->segments == 0) return DGCNN_OK;      // (no segment: nothing is written)
  if (!y || !ws) return DGCNN_EINVAL;
  a.out = y;
  int vec, threads, tiles;
  const int cap = gn_vec_cap(reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(y), a.C, dg_dtype_size(p->dtype));
  if (!gn_plan(&a, p->dtype, cap, false, &vec, &threads, &tiles)) return DGCNN_EUNSUPPORTED;
  gn_grid(&a, dg_dtype_size(p->dtype), false);
  if ((int64_t)a.nchunk * threads >> 32) return DGCNN_EUNSUPPORTED;
  a.part = static_cast<float*>(ws);
  hipLaunchKernelGGL(gn_pick_dtype(p->dtype, vec, a.L > a.R ? GN_FWD_STREAM : GN_FWD), dim3(a.nseg + a.cgrid, tiles), dim3(threads), 0, (hipStream_t)stream, a);
  DG_CHECK_LAUNCH();
  if (a.cgrid) {
    hipLaunchKernelGGL(k_gn_join, dim3((unsigned)(((int64_t)a.B * a.G * gn_join_lanes(a) + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a);
    DG_CHECK_LAUNCH();
    hipLaunchKernelGGL(gn_pick_dtype(p->dtype, vec, GN_FWD_LONG), dim3(a.nchunk, tiles), dim3(threads), 0, (hipStream_t)stream, a);
    DG_CHECK_LAUNCH();
  }
  return DGCNN_OK;
}

extern "C" int dgcnn_group_norm_bwd(const dgcnn_group_norm_args* p, const void* dy, void* dx, void* dweight, void* dbias, void* ws, dgcnn_stream_t stream) {
  DgGn a = {};
  const int rc = gn_check(p, &a);
  if (rc != DGCNN_OK) return rc;
  if ((dweight || dbias) && !dg_dtype_ok(p->weight_dtype)) return DGCNN_EINVAL;
  const bool none = p->rows == 0 || p->segments == 0;
  if (!none && (!dy || !dx || !ws)) return DGCNN_EINVAL;
  if (none) {      // (empty sums; dx has no row that lies in a segment)
    if (dweight || dbias) {
      hipLaunchKernelGGL(k_gn_wsum, dim3(dg_cdiv(2 * a.C, 8)), dim3(1024), 0, (hipStream_t)stream, a, 0, dg_cdiv(2 * a.C, 8), dweight, dbias, p->weight_dtype);
      DG_CHECK_LAUNCH();
    }
    return DGCNN_OK;
  }
  a.dy = dy; a.out = dx;
  int vec, threads, tiles;
  const int cap = gn_vec_cap(reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx), a.C, dg_dtype_size(p->dtype));
  if (!gn_plan(&a, p->dtype, cap, true, &vec, &threads, &tiles)) return DGCNN_EUNSUPPORTED;
  gn_grid(&a, dg_dtype_size(p->dtype), true);
  if ((int64_t)a.nchunk * threads >> 32) return DGCNN_EUNSUPPORTED;
  a.part = static_cast<float*>(ws);
  char* const after = static_cast<char*>(ws) + gn_part_bytes(a);
  a.ac = reinterpret_cast<float*>(after);
  if (dweight || dbias) a.wpart = reinterpret_cast<float*>(after + gn_ac_bytes(a));
  hipLaunchKernelGGL(gn_pick_dtype(p->dtype, vec, a.L > a.R ? GN_BWD_STREAM : GN_BWD), dim3(a.nseg + a.cgrid, tiles), dim3(threads), 0, (hipStream_t)stream, a);
  DG_CHECK_LAUNCH();
  const int wblocks = a.wpart ? dg_cdiv(2 * a.C, 8) : 0;
  const int64_t jblocks = a.cgrid ? ((int64_t)a.B * a.G * gn_join_lanes(a) + 1023) / 1024 : 0;
  if (wblocks + jblocks) {
    hipLaunchKernelGGL(k_gn_wsum, dim3((unsigned)(wblocks + jblocks)), dim3(1024), 0, (hipStream_t)stream, a, a.nseg + a.cgrid, wblocks, dweight, dbias, p->weight_dtype);
    DG_CHECK_LAUNCH();
  }
  if (a.cgrid) {
    hipLaunchKernelGGL(gn_pick_dtype(p->dtype, vec, GN_BWD_LONG), dim3(a.nchunk, tiles), dim3(threads), 0, (hipStream_t)stream, a);
    DG_CHECK_LAUNCH();
  }
  return DGCNN_OK;
}
