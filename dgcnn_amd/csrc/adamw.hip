// adamw.hip -- AdamW over a list of tensors in one launch (dgcnn_adamw_step).
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bound: HBM.  An element of an fp32 parameter moves 28 bytes with fp32 moments and 16 with 8-bit ones; ~25 operations.  One pass, nothing
// else leaves the registers: every thread owns eight consecutive elements, so the parameter, the gradient and both moments of a
// workgroup's 2048 elements are in flight together as 16-byte accesses, and the addresses of up to 48 tensors travel in the
// kernel's arguments (no table to upload, nothing to invalidate when a gradient moves, valid inside a captured graph).
//
// 8-bit moments: m and r = sqrt(v) are held as e4m3 codes times one fp32 scale for each 256 consecutive elements of a tensor (the block's
// largest magnitude is code 448).  r instead of v: e4m3 spans a factor of 2^17 in r, 2^35 in v.  An element with v > 0 never gets code 0:
// its next update would divide by eps alone.  Codes are rounded STOCHASTICALLY (up with the probability of the distance from the
// lower neighbour): b2 = 0.999 changes r by at most 1/2000 of its value in a step while half a code step is 3..6 %, so rounding to nearest would
// leave r where it is from its tenth step on, a factor of ~10 too small.  The random bits are a hash of (seed, the tensor's index,
// step, element), so a step is reproducible.  The update itself uses m and v before they are rounded.
// NaN and infinities are coded as NaN and leave the block's scale to its finite elements.
//
// Measured (MI355X; a 1 GiB copy reaches 5.2 TB/s): 200 M fp32 elements in 40 tensors 1034 us, 5.4 TB/s; 24 M bf16 ones with fp32 copies and moments in 60 tensors (two
// launches) 140 us, 4.8 TB/s; 200 M bf16 ones with 8-bit moments 490 us (under a profiler 514 to 751), 4.1 TB/s, held back by the arithmetic of decoding, scaling, hashing and encoding
// two codes an element; 16 tensors of 52 K elements together 5.4 us, a launch's own time.
// The operation sequence is fixed (no contraction): a step's result does not depend on alignment, on the list a tensor is in, or on the launch (with 8-bit
// moments: as long as the tensor keeps its index).
#include "dg_half.h"
#include <math.h>

#define AW_TENSORS 48      // tensors a launch: 3.5 KB of kernel arguments (4 KB are allowed)
#define AW_THREADS 256
#define AW_EPT 8           // consecutive elements of a thread
#define AW_SPAN (AW_THREADS * AW_EPT)
#define AW_TINY 7.7037197775489434e-34f      // 2^-110: a block whose largest value is below this is held as zeros (448 times its inverse would overflow)

struct DgAdamwTable {
  void* param[AW_TENSORS];
  const void* grad[AW_TENSORS];
  void* m[AW_TENSORS];
  void* v[AW_TENSORS];
  float* ms[AW_TENSORS];
  float* vs[AW_TENSORS];
  float* master[AW_TENSORS];
  int64_t numel[AW_TENSORS];
  uint32_t first[AW_TENSORS + 1];      // first workgroup of each tensor
  uint32_t key[AW_TENSORS];
  int count;
  int spans;                           // AW_SPAN elements each, per workgroup
};
struct DgAdamwScalars {
  float decay, b1, omb1, b2, omb2, rbc2, eps, ss;
  uint32_t step;
};
static_assert(sizeof(DgAdamwScalars) <= 16 * sizeof(float), "scalars_dev holds 16 floats");

static __host__ __device__ inline DgAdamwScalars aw_scalars(double lr, double b1, double b2, double eps, double wd, int64_t step) {
  DgAdamwScalars s;
  s.decay = (float)(1.0 - lr * wd);
  s.b1 = (float)b1; s.omb1 = (float)(1.0 - b1);
  s.b2 = (float)b2; s.omb2 = (float)(1.0 - b2);
  s.rbc2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)step)));
  s.eps = (float)eps;
  s.ss = (float)(lr / (1.0 - pow(b1, (double)step)));
  s.step = (uint32_t)step;
  return s;
}

// the step counter lives on the device (captured training steps): count, and leave this step's factors for the launches behind
__global__ void k_adamw_tick(int64_t* step, const float* lr_dev, double lr, double b1, double b2, double eps, double wd, DgAdamwScalars* out) {
  if (threadIdx.x) return;      // (one wave, one lane of it)
  const int64_t t = *step + 1;
  *step = t;
  *out = aw_scalars(lr_dev ? (double)*lr_dev : lr, b1, b2, eps, wd, t);
}

#ifdef DG_EMU
static inline float aw_e4m3(uint32_t code) {
  const uint32_t c = code & 0x7f;
  const float f = c == 0x7f ? NAN : c < 8 ? (float)c * 0x1p-9f : ldexpf((float)(8 + (c & 7)), (int)(c >> 3) - 10);
  return (code & 0x80) ? -f : f;
}
static inline void aw_decode4(uint32_t w, float* f) { for (int i = 0; i < 4; ++i) f[i] = aw_e4m3(w >> (8 * i)); }
#else
__device__ __forceinline__ void aw_decode4(uint32_t w, float* f) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  f[0] = a[0]; f[1] = a[1]; f[2] = b[0]; f[3] = b[1];
}
#endif

// e4m3 code of t (|t| <= 448 up to rounding): with e = max(floor(log2 |t|), -6) the grid is 2^(e-3), and the code of q grid steps is 8 (e + 6) + q
__device__ __forceinline__ uint32_t aw_encode(float t, uint32_t noise16) {
  const float a = fabsf(t);
  const uint32_t e = max(__float_as_uint(a), 0x3c800000u) >> 23;      // biased exponent, at least that of 2^-6
  const float q = floorf(a * __uint_as_float((257u - e) << 23) + (float)noise16 * 0x1p-16f);
  uint32_t code = min((e - 121u) * 8u + (uint32_t)q, 126u);
  code = a < 512.f ? code : 127u;                                     // (NaN)
  return code | ((__float_as_uint(t) >> 24) & 0x80u);
}
__device__ __forceinline__ uint32_t aw_hash(uint32_t h) {             // a bijective 32-bit mixer of xor-shifts and odd multipliers (constants in the public domain)
  h = (h ^ (h >> 16)) * 0x85EBCA6Bu;
  h = (h ^ (h >> 13)) * 0xC2B2AE35u;
  return h ^ (h >> 16);
}

// largest finite magnitude over the 32 lanes that hold one block of 256 elements (the maximum passes over NaN; infinities are looked for where it is one)
__device__ __forceinline__ float aw_block_max(const float* x) {
  float a = 0.f;
#pragma unroll
  for (int i = 0; i < AW_EPT; ++i) a = fmaxf(a, fabsf(x[i]));
  if (a > 3.4028235e38f) {
    a = 0.f;
#pragma unroll
    for (int i = 0; i < AW_EPT; ++i) a = fmaxf(a, fabsf(x[i]) <= 3.4028235e38f ? fabsf(x[i]) : 0.f);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) a = fmaxf(a, __shfl_xor(a, o));
  return a >= AW_TINY ? a : 0.f;
}

// n of the eight elements at p (all of them as vectors where `wide`)
template <class D> __device__ __forceinline__ void aw_load(const typename D::S* p, int n, bool wide, float* f) {
  if (wide && n == AW_EPT) {
#pragma unroll
    for (int h = 0; h < AW_EPT; h += D::FULL) {
      const DgRaw<D, D::FULL> r = dg_load<D, D::FULL>(p + h);
#pragma unroll
      for (int i = 0; i < D::FULL; ++i) f[h + i] = r.get(i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < AW_EPT; ++i) f[i] = i < n ? D::to(p[i]) : 0.f;
  }
}
template <class D> __device__ __forceinline__ void aw_store(typename D::S* p, int n, bool wide, const float* f) {
  if (wide && n == AW_EPT) {
#pragma unroll
    for (int h = 0; h < AW_EPT; h += D::FULL) {
      DgRaw<D, D::FULL> r;
#pragma unroll
      for (int i = 0; i < D::FULL; ++i) r.set(i, f[h + i]);
      dg_store<D, D::FULL>(p + h, r);
    }
  } else {
#pragma unroll
    for (int i = 0; i < AW_EPT; ++i) if (i < n) p[i] = D::from(f[i]);
  }
}

template <class P, class G, bool MASTER, int BITS>
__global__ void __launch_bounds__(AW_THREADS)
k_adamw(const DgAdamwTable t, const DgAdamwScalars byval, const DgAdamwScalars* dev) {
#pragma clang fp contract(off)
  const DgAdamwScalars s = dev ? *dev : byval;
  int k = 0;
  for (int hi = t.count; hi - k > 1;) {
    const int mid = (k + hi) >> 1;
    if (blockIdx.x >= t.first[mid]) k = mid; else hi = mid;
  }
  const int64_t numel = t.numel[k];
  typename P::S* const param = static_cast<typename P::S*>(t.param[k]);
  const typename G::S* const grad = static_cast<const typename G::S*>(t.grad[k]);
  float* const master = t.master[k];
  const uintptr_t low = reinterpret_cast<uintptr_t>(param) | reinterpret_cast<uintptr_t>(grad) | (MASTER ? reinterpret_cast<uintptr_t>(master) : 0);
  const uintptr_t slow = reinterpret_cast<uintptr_t>(t.m[k]) | reinterpret_cast<uintptr_t>(t.v[k]);
  const bool wide = (low & 15) == 0 && (slow & (BITS == 32 ? 15 : 7)) == 0;
  const int64_t base = (int64_t)(blockIdx.x - t.first[k]) * t.spans * AW_SPAN;

  for (int it = 0; it < t.spans; ++it) {
    const int64_t at = base + (int64_t)it * AW_SPAN + threadIdx.x * AW_EPT;
    if (base + (int64_t)it * AW_SPAN >= numel) break;                  // (the whole workgroup)
    const int n = at >= numel ? 0 : numel - at < AW_EPT ? (int)(numel - at) : AW_EPT;
    float p[AW_EPT], g[AW_EPT], m[AW_EPT], v[AW_EPT], r[AW_EPT];
    if (MASTER) aw_load<DgF32>(master + at, n, wide, p); else aw_load<P>(param + at, n, wide, p);
    aw_load<G>(grad + at, n, wide, g);
    if (BITS == 32) {
      aw_load<DgF32>(static_cast<const float*>(t.m[k]) + at, n, wide, m);
      aw_load<DgF32>(static_cast<const float*>(t.v[k]) + at, n, wide, v);
    } else {
      const uint8_t* const mq = static_cast<const uint8_t*>(t.m[k]) + at;
      const uint8_t* const vq = static_cast<const uint8_t*>(t.v[k]) + at;
      uint32_t wm[2] = {0, 0}, wv[2] = {0, 0};
      if (wide && n == AW_EPT) {
        const uint2 a = *reinterpret_cast<const uint2*>(mq), b = *reinterpret_cast<const uint2*>(vq);
        wm[0] = a.x; wm[1] = a.y; wv[0] = b.x; wv[1] = b.y;
      } else {
#pragma unroll
        for (int i = 0; i < AW_EPT; ++i)
          if (i < n) { wm[i >> 2] |= (uint32_t)mq[i] << (8 * (i & 3)); wv[i >> 2] |= (uint32_t)vq[i] << (8 * (i & 3)); }
      }
      const float ms = n ? t.ms[k][at >> 8] : 0.f, vs = n ? t.vs[k][at >> 8] : 0.f;
      aw_decode4(wm[0], m); aw_decode4(wm[1], m + 4);
      aw_decode4(wv[0], v); aw_decode4(wv[1], v + 4);
#pragma unroll
      for (int i = 0; i < AW_EPT; ++i) { m[i] = m[i] * ms; v[i] = v[i] * vs; v[i] = v[i] * v[i]; }
    }
#pragma unroll
    for (int i = 0; i < AW_EPT; ++i) {
      m[i] = m[i] * s.b1 + g[i] * s.omb1;
      v[i] = v[i] * s.b2 + (g[i] * g[i]) * s.omb2;
      r[i] = sqrtf(v[i]);
      const float den = r[i] * s.rbc2 + s.eps;
      // (8 bits: bound by arithmetic, and v_rcp_f32's 1 ulp of an update is far below its parameter's rounding)
      const float u = BITS == 32 ? m[i] / den : m[i] * __builtin_amdgcn_rcpf(den);
      p[i] = p[i] * s.decay - u * s.ss;
    }
    if (MASTER) aw_store<DgF32>(master + at, n, wide, p);
    aw_store<P>(param + at, n, wide, p);
    if (BITS == 32) {
      aw_store<DgF32>(static_cast<float*>(t.m[k]) + at, n, wide, m);
      aw_store<DgF32>(static_cast<float*>(t.v[k]) + at, n, wide, v);
    } else {
      const float mtop = aw_block_max(m), rtop = aw_block_max(r);      // (elements behind the tensor's end are zeros)
      const float minv = mtop > 0.f ? 1.f / mtop * 448.f : 0.f, rinv = rtop > 0.f ? 1.f / rtop * 448.f : 0.f;
      uint32_t wm[2] = {0, 0}, wv[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < AW_EPT; ++i) {
        const uint32_t h = aw_hash((uint32_t)(at + i) * 0x9E3779B1u + t.key[k] + s.step * 0x632BE5ABu);
        wm[i >> 2] |= aw_encode(m[i] * minv, h & 0xffffu) << (8 * (i & 3));
        const float x = r[i] * rinv;
        const uint32_t c = aw_encode(x, h >> 16);
        wv[i >> 2] |= (x > 0.f ? max(c, 1u) : c) << (8 * (i & 3));
      }
      uint8_t* const mq = static_cast<uint8_t*>(t.m[k]) + at;
      uint8_t* const vq = static_cast<uint8_t*>(t.v[k]) + at;
      if (wide && n == AW_EPT) {
        *reinterpret_cast<uint2*>(mq) = make_uint2(wm[0], wm[1]);
        *reinterpret_cast<uint2*>(vq) = make_uint2(wv[0], wv[1]);
      } else {
#pragma unroll
        for (int i = 0; i < AW_EPT; ++i)
          if (i < n) { mq[i] = (uint8_t)(wm[i >> 2] >> (8 * (i & 3))); vq[i] = (uint8_t)(wv[i >> 2] >> (8 * (i & 3))); }
      }
      if (n && (threadIdx.x & 31) == 0) { t.ms[k][at >> 8] = mtop * (1.f / 448.f); t.vs[k][at >> 8] = rtop * (1.f / 448.f); }
    }
  }
}

typedef void (*aw_kernel)(const DgAdamwTable, const DgAdamwScalars, const DgAdamwScalars*);
template <class P, class G> static aw_kernel aw_pick(bool master, int bits) {
  if (master) return bits == 32 ? (aw_kernel)k_adamw<P, G, true, 32> : (aw_kernel)k_adamw<P, G, true, 8>;
  return bits == 32 ? (aw_kernel)k_adamw<P, G, false, 32> : (aw_kernel)k_adamw<P, G, false, 8>;
}

extern "C" int dgcnn_adamw_step(const dgcnn_adamw_args* a, dgcnn_stream_t stream) {
  if (!a || a->count < 0 || (a->count > 0 && !a->tensors)) return DGCNN_EINVAL;
  if (!dg_dtype_ok(a->param_dtype) || (a->grad_dtype != a->param_dtype && a->grad_dtype != DGCNN_F32)) return DGCNN_EINVAL;
  if (a->state_bits != 32 && a->state_bits != 8) return DGCNN_EINVAL;
  if (a->step_dev ? !a->scalars_dev : a->step < 1) return DGCNN_EINVAL;
  if (!(a->beta1 >= 0.0 && a->beta1 < 1.0) || !(a->beta2 >= 0.0 && a->beta2 < 1.0) || !(a->eps >= 0.0)) return DGCNN_EINVAL;
  int masters = 0, live = 0;
  int64_t total = 0;
  for (int i = 0; i < a->count; ++i) {
    const dgcnn_adamw_tensor* t = &a->tensors[i];
    if (t->numel < 0) return DGCNN_EINVAL;
    if (t->numel == 0) continue;
    if (!t->param || !t->grad || !t->exp_avg || !t->exp_avg_sq) return DGCNN_EINVAL;
    if (a->state_bits == 8 && (!t->exp_avg_scale || !t->exp_avg_sq_scale)) return DGCNN_EINVAL;
    if (t->numel > ((int64_t)1 << 40)) return DGCNN_EUNSUPPORTED;
    masters += t->master != nullptr;
    ++live;
    total += t->numel;
  }
  if (masters != 0 && (masters != live || a->param_dtype == DGCNN_F32)) return DGCNN_EINVAL;

  hipStream_t st = (hipStream_t)stream;
  DgAdamwScalars sc = {};
  DgAdamwScalars* const dev = a->step_dev ? reinterpret_cast<DgAdamwScalars*>(a->scalars_dev) : nullptr;
  if (dev) {
    hipLaunchKernelGGL(k_adamw_tick, dim3(1), dim3(64), 0, st, a->step_dev, a->lr_dev, a->lr, a->beta1, a->beta2, a->eps, a->weight_decay, dev);
    DG_CHECK_LAUNCH();
  } else {
    sc = aw_scalars(a->lr, a->beta1, a->beta2, a->eps, a->weight_decay, a->step);
  }
  aw_kernel kern = nullptr;
  if (a->param_dtype == DGCNN_F32) kern = aw_pick<DgF32, DgF32>(false, a->state_bits);
  else if (a->param_dtype == DGCNN_BF16)
    kern = a->grad_dtype == DGCNN_F32 ? aw_pick<DgBF16, DgF32>(masters != 0, a->state_bits) : aw_pick<DgBF16, DgBF16>(masters != 0, a->state_bits);
  else
    kern = a->grad_dtype == DGCNN_F32 ? aw_pick<DgF16, DgF32>(masters != 0, a->state_bits) : aw_pick<DgF16, DgF16>(masters != 0, a->state_bits);

  DgAdamwTable tab;
  tab.spans = 1;
  while (total / ((int64_t)tab.spans * AW_SPAN) > ((int64_t)1 << 20)) tab.spans *= 2;      // at most 2^20 workgroups and one a tensor
  int k = 0;
  uint64_t blocks = 0;
  for (int i = 0; i <= a->count; ++i) {
    const bool end = i == a->count;
    if (!end && a->tensors[i].numel > 0) {
      const dgcnn_adamw_tensor* t = &a->tensors[i];
      uint64_t z = a->seed + 0x9E3779B97F4A7C15ull * ((uint64_t)(a->indices ? a->indices[i] : a->first_index + i) + 1);      // (splitmix64, as the dropout mask's)
      z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
      z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
      tab.param[k] = t->param; tab.grad[k] = t->grad; tab.m[k] = t->exp_avg; tab.v[k] = t->exp_avg_sq;
      tab.ms[k] = t->exp_avg_scale; tab.vs[k] = t->exp_avg_sq_scale; tab.master[k] = t->master;
      tab.numel[k] = t->numel; tab.key[k] = (uint32_t)(z ^ (z >> 31));
      tab.first[k] = (uint32_t)blocks;
      const int64_t per = (int64_t)tab.spans * AW_SPAN;
      blocks += (uint64_t)((t->numel + per - 1) / per);
      ++k;
    }
    if (k == AW_TENSORS || (end && k > 0)) {
      tab.first[k] = (uint32_t)blocks;
      tab.count = k;
      hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(AW_THREADS), 0, st, tab, sc, (const DgAdamwScalars*)dev);
      DG_CHECK_LAUNCH();
      k = 0; blocks = 0;
    }
  }
  return DGCNN_OK;
}
