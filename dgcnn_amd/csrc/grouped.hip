// grouped.hip -- matrix products grouped by type over ragged runs of rows (dgcnn_grouped_linear_fwd, dgcnn_grouped_linear_bwd).
//
//   rows ptr[e] .. ptr[e+1]-1 of x belong to group e:   y_i = W_e x_i + b_e     dx_i = W_e^T dy_i     dW_e = sum_i dy_i x_i^T     db_e = sum_i dy_i
//
// One tile kernel computes C[i][j] = sum_r P[i][r] Q[j][r] for all three products:
//              i          j         r          P                    Q
//   y          rows       out       in         x   (r contiguous)   W_e (r contiguous)
//   dx         rows       in        out        dy  (r contiguous)   W_e (j contiguous)
//   dW_e       out        in        rows       dy  (i contiguous)   x   (j contiguous)
// Tiles of P and Q lie in LDS as they lie in memory, 128 bytes of r a row (or all columns of an r), in 16-byte chunks whose place is swizzled so that a
// wave's reads spread over the banks.  An operand that is contiguous in r is read as the matrix instruction wants it (16 bytes = the lane's r
// values); one that is not goes through the transposing LDS read (16-bit types) or element by element (fp32).  The instruction's A
// operand is Q: a lane then holds four consecutive columns of one row of C, which it stores at once.
//
// Group boundaries are known on the device alone: the grid is the largest number of tiles that any split of the rows into groups can need, and every
// workgroup finds its tile by a prefix sum over the groups' tile counts.  Rows outside every group form two more groups, which are cleared.
// dW: a group's rows are cut into slices where there are too few tiles for the chip; slices leave fp32 partial tiles, summed in a fixed order.
// db rides on the dW product as a column of ones.
#include "dg_half.h"

#define GL_ROWB 128      // bytes of r in a row of an r-contiguous tile

struct DgGl {
  const void *p, *q;             // operands (see above); q of group e begins at e * qstride
  const void* bias;              // y only: [groups][nj]
  void* c;                       // y, dx or dW
  float* part;                   // dW in slices: [slots][ni * nj + ni] partial sums
  void* db;                      // dW: [groups][ni], or null
  const int64_t* ptr;
  int64_t M;                     // rows
  int64_t ldp, ldq, ldc, qstride;
  int ni, nj, nr;                // extents of C and of the sum (ni: -1 where i runs over rows; nr: -1 where r does)
  int E;
  int tj, ti;                    // tiles along j (and, dW, along i)
  int64_t slice;                 // dW: rows a slice (a multiple of the tile's r)
  int split;                     // dW: 1: partial tiles
  int64_t slots;                 // ... that there is room for: enough for every ascending ptr
};

__device__ __forceinline__ void gl_range(const DgGl& a, int e, int64_t& lo, int64_t& hi) {      // inside [0, M] whatever ptr holds
  if (e < a.E) {
    lo = min(max(a.ptr[e], (int64_t)0), a.M);
    hi = min(max(a.ptr[e + 1], lo), a.M);
  } else if (e == a.E) {         // in front of the first group
    lo = 0; hi = a.E ? min(max(a.ptr[0], (int64_t)0), a.M) : a.M;
  } else {                       // behind the last one
    hi = a.M; lo = a.E ? min(max(a.ptr[a.E], (int64_t)0), a.M) : a.M;
  }
}
// Work item t -> the group it lies in and its index there; every group has ceil(rows / per) items.  The whole wave searches: 64 groups a step.
// total: all items.  false: no such item.
__device__ __forceinline__ bool gl_find(const DgGl& a, int groups, int64_t per, int64_t t, int& e, int64_t& in, int64_t& total) {
  const int lane = threadIdx.x & 63;
  int64_t base = 0;
  bool found = false;
  for (int e0 = 0; e0 < groups; e0 += 64) {
    int64_t n = 0;
    if (e0 + lane < groups) {
      int64_t lo, hi;
      gl_range(a, e0 + lane, lo, hi);
      n = (hi - lo + per - 1) / per;
    }
    int64_t upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t u = __shfl_up(upto, o);
      if (lane >= o) upto += u;
    }
    const uint64_t m = __ballot(base + upto > t);
    if (!found && m) {
      const int k = __ffsll((long long)m) - 1;
      e = e0 + k;
      in = t - base - (__shfl(upto, k) - __shfl(n, k));
      found = true;
    }
    base += __shfl(upto, 63);
  }
  total = base;
  return found;
}

__device__ __attribute__((aligned(16))) uint32_t gl_zero[4];      // what chunks behind an operand's end are loaded from

#ifdef DG_EMU
typedef dg_emu_bf16x8 gl_bf16x8;
typedef dg_emu_f16x8 gl_f16x8;
typedef dg_emu_s16x4 gl_s16x4;
#define GL_LDS_PTR(p) (p)
#else
typedef __bf16 gl_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 gl_f16x8 __attribute__((ext_vector_type(8)));
typedef short gl_s16x4 __attribute__((ext_vector_type(4)));
#endif
typedef uint32_t gl_u32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of every lane to LDS at (uniform) dst + 16 * lane, without passing through registers
__device__ __forceinline__ void gl_to_lds(const char* src, char* dst) {
#ifdef DG_EMU
  *reinterpret_cast<gl_u32x4*>(dst + 16 * (threadIdx.x & 63)) = *reinterpret_cast<const gl_u32x4*>(src);
#else
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
#endif
}
__device__ __forceinline__ gl_s16x4 gl_read_tr(const char* p) {
#ifdef DG_EMU
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<const gl_s16x4*>(p));
#else
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) gl_s16x4*)p);
#endif
}
template <class D> __device__ __forceinline__ f32x4 gl_mfma(const gl_u32x4& a, const gl_u32x4& b, f32x4 c) {
  if constexpr (sizeof(typename D::S) == 4) {      // the lane's four r values one after the other: the same ones on both sides
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[s]), __uint_as_float(b[s]), c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(D, DgBF16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gl_bf16x8, a), __builtin_bit_cast(gl_bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gl_f16x8, a), __builtin_bit_cast(gl_f16x8, b), c, 0, 0, 0);
  }
}

// One operand's tile: W indices (i or j) x R = 128 / sizeof r values
//   T = false: memory and LDS [index][r]; 8 chunks an index, chunk c at place c ^ (index & 7): 8 lanes of a fragment read 8 different places
//   T = true : memory and LDS [r][index]; chunk c at place c ^ swizzle(r).  16-bit: a transposing read takes 32 bytes of r = 8g + j (j < 4, g < 4): j and one
//              bit of g pick the 32-byte piece.  fp32: 64 bytes of r = 4g + s: g picks it.
template <class D, int W, bool T> struct GlTile {
  typedef typename D::S S;
  static constexpr int ES = sizeof(S), CE = 16 / ES, R = GL_ROWB / ES, BYTES = W * GL_ROWB, CPR = W * ES / 16;
  static __device__ __forceinline__ int swizzle(int r) {
    if (ES == 4) return (((r >> 2) & 3) << 2) & (CPR - 1);
    return (((r & 3) | (((r >> 3) & 1) << 2)) << 1) & (CPR - 1);
  }
  // chunk q of the tile in LDS order: which index and r it begins at
  static __device__ __forceinline__ void place(int q, int& w, int& r) {
    if (T) { r = q / CPR; w = ((q % CPR) ^ swizzle(r)) * CE; }
    else { w = q >> 3; r = ((q & 7) ^ (w & 7)) * CE; }
  }
  // the tile at (w0, r0) of an operand with nw indices and r values up to rend
  template <bool ALIGNED, int THREADS>
  static __device__ __forceinline__ void load(char* lds, const S* base, int64_t ld, int64_t w0, int64_t r0, int64_t nw, int64_t rend) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < BYTES / 16 / THREADS; ++k) {
      const int q0 = (k * (THREADS / 64) + wave) * 64;
      int w, r;
      place(q0 + lane, w, r);
      const S* const src = T ? base + (r0 + r) * ld + (w0 + w) : base + (w0 + w) * ld + (r0 + r);
      if (ALIGNED) {      // (a chunk lies inside the operand or outside: extents and strides are multiples of it)
        const bool in = w0 + w < nw && r0 + r < rend;
        gl_to_lds(in ? reinterpret_cast<const char*>(src) : reinterpret_cast<const char*>(gl_zero), lds + q0 * 16);
      } else {
        DgRaw<D, CE> v = dg_zero<D, CE>();
#pragma unroll
        for (int i = 0; i < CE; ++i)
          if (T ? w0 + w + i < nw && r0 + r < rend : w0 + w < nw && r0 + r + i < rend) v.v[i] = src[i];
        dg_store<D, CE>(reinterpret_cast<S*>(lds + (q0 + lane) * 16), v);
      }
    }
  }
  // the lane's r values of index w0 + lane % 16 in half s of the tile: r = R/2 s + CE (lane / 16) + 0 .. CE-1
  static __device__ __forceinline__ gl_u32x4 fragment(const char* lds, int w0, int s) {
    const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
    if constexpr (!T) {
      const int w = w0 + l;
      return *reinterpret_cast<const gl_u32x4*>(lds + w * GL_ROWB + (((s * 4 + g) ^ (w & 7)) << 4));
    } else if constexpr (ES == 2) {
      gl_s16x4 v[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = s * 32 + g * 8 + h * 4 + (l >> 2), c = w0 / 8 + ((l & 3) >> 1);
        v[h] = gl_read_tr(lds + r * (W * ES) + ((c ^ swizzle(r)) << 4) + ((l & 1) << 3));
      }
      struct { gl_s16x4 a, b; } two = {v[0], v[1]};
      return __builtin_bit_cast(gl_u32x4, two);
    } else {
      gl_u32x4 v;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = s * 16 + g * 4 + k, w = w0 + l;
        v[k] = *reinterpret_cast<const uint32_t*>(lds + r * (W * ES) + (((w >> 2) ^ swizzle(r)) << 4) + ((w & 3) << 2));
      }
      return v;
    }
  }
};

template <class D> __device__ __forceinline__ uint32_t gl_ones() { return sizeof(typename D::S) == 4 ? 0x3f800000u : __is_same(D, DgBF16) ? 0x3f803f80u : 0x3c003c00u; }

// WI x WJ waves of (16 FI) x (16 FJ) tiles of C
template <class D, int WI, int WJ, int FI, int FJ, bool PT, bool QT, bool ALIGNED>
__global__ void __launch_bounds__(64 * WI * WJ)
k_gl(const DgGl a) {
  constexpr int BI = WI * FI * 16, BJ = WJ * FJ * 16, THREADS = 64 * WI * WJ;
  constexpr bool GRAD = PT;                                   // the product over rows
  typedef typename D::S S;
  typedef GlTile<D, BI, PT> TP;
  typedef GlTile<D, BJ, QT> TQ;
  constexpr int R = TP::R;
  DG_DYN_SMEM(char, smem);                                    // two stages of P and Q
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const int wi = wave / WJ, wj = wave - wi * WJ;

  // ---- which tile
  int e = 0, i0, j0;
  int64_t lo, hi, r0, rend, in = 0, total;
  const S *p = static_cast<const S*>(a.p), *q = static_cast<const S*>(a.q);
  int64_t nw_i;
  int slot = 0;
  if (!GRAD) {
    // consecutive tiles (the columns of one run of rows first) on one XCD: workgroups go to the eight in turn
    if (!gl_find(a, a.E + 2, BI, -1, e, in, total)) {}
    const int64_t tiles = total * a.tj, share = (tiles + 7) >> 3;
    const int64_t t = (int64_t)(blockIdx.x & 7) * share + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= share || t >= tiles) return;
    gl_find(a, a.E + 2, BI, t / a.tj, e, in, total);
    gl_range(a, e, lo, hi);
    j0 = (int)(t % a.tj) * BJ;
    i0 = 0;
    lo += in * BI;
    nw_i = hi;                                                // row index
    r0 = 0; rend = a.nr;
    if (e >= a.E) {                                           // rows of no group
      S* const c = static_cast<S*>(a.c);
      for (int64_t k = threadIdx.x; k < BI * BJ; k += THREADS) {
        const int64_t i = lo + k / BJ, j = j0 + k % BJ;
        if (i < hi && j < a.nj) c[i * a.ldc + j] = D::from(0.f);
      }
      return;
    }
    q += (int64_t)e * a.qstride;
  } else {
    const int tile = blockIdx.x % (a.ti * a.tj);
    const int64_t t = blockIdx.x / (a.ti * a.tj);
    if (a.split) {
      if (!gl_find(a, a.E, a.slice, t, e, in, total)) return;
      slot = (int)t;
      gl_range(a, e, lo, hi);
    } else {
      e = (int)t;
      gl_range(a, e, lo, hi);
    }
    i0 = (tile / a.tj) * BI; j0 = (tile % a.tj) * BJ;
    r0 = lo + in * a.slice;
    rend = a.split ? min(r0 + a.slice, hi) : hi;
    nw_i = a.ni;
    lo = i0;
  }

  f32x4 acc[FI][FJ], sum[FI];
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    sum[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < FJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const bool sums = GRAD && a.db && j0 == 0 && wj == 0;
  gl_u32x4 ones;
#pragma unroll
  for (int i = 0; i < 4; ++i) ones[i] = gl_ones<D>();

  // ---- two stages: the next tiles are on their way while the present ones are multiplied
  const int steps = (int)((rend - r0 + R - 1) / R);
  if (steps > 0) {
    TP::template load<ALIGNED, THREADS>(smem, p, a.ldp, lo, r0, nw_i, rend);
    TQ::template load<ALIGNED, THREADS>(smem + TP::BYTES, q, a.ldq, j0, r0, a.nj, rend);
  }
  __syncthreads();
  for (int k = 0; k < steps; ++k) {
    char* const now = smem + (k & 1) * (TP::BYTES + TQ::BYTES);
    char* const next = smem + ((k + 1) & 1) * (TP::BYTES + TQ::BYTES);
    if (k + 1 < steps) {
      TP::template load<ALIGNED, THREADS>(next, p, a.ldp, lo, r0 + (int64_t)(k + 1) * R, nw_i, rend);
      TQ::template load<ALIGNED, THREADS>(next + TP::BYTES, q, a.ldq, j0, r0 + (int64_t)(k + 1) * R, a.nj, rend);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      gl_u32x4 fp[FI], fq[FJ];
#pragma unroll
      for (int i = 0; i < FI; ++i) fp[i] = TP::fragment(now, (wi * FI + i) * 16, s);
#pragma unroll
      for (int j = 0; j < FJ; ++j) fq[j] = TQ::fragment(now + TP::BYTES, (wj * FJ + j) * 16, s);
#pragma unroll
      for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = gl_mfma<D>(fq[j], fp[i], acc[i][j]);
      if (GRAD && sums) {
#pragma unroll
        for (int i = 0; i < FI; ++i) sum[i] = gl_mfma<D>(ones, fp[i], sum[i]);
      }
    }
    __syncthreads();
  }

  // ---- C: the lane holds row l and columns 4g .. 4g+3 of every 16 x 16 tile
#pragma unroll
  for (int i = 0; i < FI; ++i) {
    const int64_t row = lo + (wi * FI + i) * 16 + l;
    if (row >= nw_i) continue;
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int col = j0 + (wj * FJ + j) * 16 + 4 * g;
      if (col >= a.nj) continue;
      f32x4 v = acc[i][j];
      if (GRAD && a.split) {
        float* const c = a.part + (int64_t)slot * ((int64_t)a.ni * a.nj + a.ni) + row * a.nj + col;
#pragma unroll
        for (int k = 0; k < 4; ++k) if (col + k < a.nj) c[k] = v[k];
        continue;
      }
      S* const c = static_cast<S*>(a.c) + (GRAD ? (int64_t)e * a.ni * a.nj : 0) + row * a.ldc + col;
      if (!GRAD && a.bias) {
        const S* const b = static_cast<const S*>(a.bias) + (int64_t)e * a.nj + col;
#pragma unroll
        for (int k = 0; k < 4; ++k) if (col + k < a.nj) v[k] += D::to(b[k]);
      }
      if (ALIGNED || (col + 4 <= a.nj && (reinterpret_cast<uintptr_t>(c) & (4 * sizeof(S) - 1)) == 0)) {
        DgRaw<D, 4> o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o.set(k, v[k]);
        dg_store<D, 4>(c, o);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) if (col + k < a.nj) c[k] = D::from(v[k]);
      }
    }
    if (GRAD && sums && g == 0) {
      if (a.split) a.part[(int64_t)slot * ((int64_t)a.ni * a.nj + a.ni) + (int64_t)a.ni * a.nj + row] = sum[i][0];
      else static_cast<S*>(a.db)[(int64_t)e * a.ni + row] = D::from(sum[i][0]);
    }
  }
}

// dW and db from the slices' partial tiles, slice after slice; a group without rows gets zeros
template <class D>
__global__ void __launch_bounds__(256)
k_gl_join(const DgGl a) {
  typedef typename D::S S;
  const int64_t each = (int64_t)a.ni * a.nj + a.ni;
  const int e = blockIdx.y;
  int64_t first = 0, slices = 0;
  {      // slots in front of group e's
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 <= e; e0 += 64) {
      int64_t n = 0;
      if (e0 + lane <= e) {
        int64_t lo, hi;
        gl_range(a, e0 + lane, lo, hi);
        n = (hi - lo + a.slice - 1) / a.slice;
      }
      const int64_t last = __shfl(n, (e - e0) & 63);
      for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
      first += n;
      if (e - e0 < 64) { slices = last; first -= last; }
    }
  }
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < each; k += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    const float* const p = a.part + first * each + k;
    for (int64_t i = 0; i < slices && first + i < a.slots; ++i) s += p[i * each];
    if (k < (int64_t)a.ni * a.nj) static_cast<S*>(a.c)[(int64_t)e * a.ni * a.nj + k] = D::from(s);
    else if (a.db) static_cast<S*>(a.db)[(int64_t)e * a.ni + (k - (int64_t)a.ni * a.nj)] = D::from(s);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
typedef void (*gl_kernel)(const DgGl);
struct GlForm { gl_kernel k; int bi, bj, threads, lds, r; };
template <class D, int WI, int WJ, int FI, int FJ, bool PT, bool QT> static GlForm gl_form(bool aligned) {
  GlForm f;
  f.k = aligned ? (gl_kernel)k_gl<D, WI, WJ, FI, FJ, PT, QT, true> : (gl_kernel)k_gl<D, WI, WJ, FI, FJ, PT, QT, false>;
  f.bi = WI * FI * 16; f.bj = WJ * FJ * 16; f.threads = 64 * WI * WJ;
  f.lds = 2 * (f.bi + f.bj) * GL_ROWB;
  f.r = GL_ROWB / (int)sizeof(typename D::S);
  return f;
}
template <class D, bool PT, bool QT> static GlForm gl_pick(int nj, bool aligned) {
  if (nj <= 32) return gl_form<D, 4, 1, 2, 2, PT, QT>(aligned);
  return gl_form<D, 2, 2, 4, 4, PT, QT>(aligned);
}
template <bool PT, bool QT> static GlForm gl_pick_dtype(int dtype, int nj, bool aligned) {
  return dtype == DGCNN_F32 ? gl_pick<DgF32, PT, QT>(nj, aligned) : dtype == DGCNN_BF16 ? gl_pick<DgBF16, PT, QT>(nj, aligned) : gl_pick<DgF16, PT, QT>(nj, aligned);
}
static int gl_launch(const GlForm& f, int64_t blocks, const DgGl& a, hipStream_t s) {
  if (blocks <= 0) return DGCNN_OK;
  if (blocks > 0x7fffffff) return DGCNN_EUNSUPPORTED;
  if (f.lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(f.k), hipFuncAttributeMaxDynamicSharedMemorySize, f.lds) != hipSuccess) return DGCNN_ELAUNCH;
  hipLaunchKernelGGL(f.k, dim3((unsigned)blocks), dim3(f.threads), f.lds, s, a);
  DG_CHECK_LAUNCH();
  return DGCNN_OK;
}
// dW: rows a slice, or 0 for one slice a group.  As many slices as fill the chip twice over (512 workgroups), each at least 512 rows.
static int64_t gl_slice(int64_t rows, int E, int64_t tiles) {
  if (tiles * E >= 512) return 0;
  const int64_t want = (512 + tiles - 1) / tiles;
  int64_t s = (rows + want - 1) / want;
  s = dg_align(s < 512 ? 512 : s, 64);
  return s;
}
static int gl_check(const dgcnn_grouped_linear_args* p) {
  if (!p || p->rows < 0 || p->in_features < 1 || p->out_features < 1 || p->groups < 0 || !dg_dtype_ok(p->dtype) || !p->ptr) return DGCNN_EINVAL;
  if (p->ldx < p->in_features) return DGCNN_EINVAL;
  if (p->rows > 0 && !p->x) return DGCNN_EINVAL;
  if (p->groups > 0 && !p->weight) return DGCNN_EINVAL;
  if (p->rows > ((int64_t)1 << 40) / p->ldx || p->rows > ((int64_t)1 << 40) / p->out_features ||
      (int64_t)p->in_features * p->out_features > ((int64_t)1 << 40) / (p->groups ? p->groups : 1) || p->groups > (1 << 20)) return DGCNN_EUNSUPPORTED;
  return DGCNN_OK;
}

extern "C" int64_t dgcnn_grouped_linear_workspace_bytes(int64_t rows, int in_features, int out_features, int groups, int dtype) {
  if (rows < 0 || in_features < 1 || out_features < 1 || groups < 0 || !dg_dtype_ok(dtype)) return DGCNN_EINVAL;
  const GlForm f = gl_pick_dtype<true, true>(dtype, in_features, true);
  const int64_t tiles = (int64_t)dg_cdiv(out_features, f.bi) * dg_cdiv(in_features, f.bj), slice = gl_slice(rows, groups, tiles);
  if (!slice) return 256;
  return dg_align((rows / slice + groups) * ((int64_t)in_features * out_features + out_features) * 4, 256);
}

extern "C" int dgcnn_grouped_linear_fwd(const dgcnn_grouped_linear_args* p, void* y, dgcnn_stream_t stream) {
  const int rc = gl_check(p);
  if (rc != DGCNN_OK) return rc;
  if (p->rows == 0) return DGCNN_OK;
  if (!y) return DGCNN_EINVAL;
  const int es = dg_dtype_size(p->dtype), ce = 16 / es;
  DgGl a = {};
  a.p = p->x; a.q = p->weight; a.bias = p->bias; a.c = y; a.ptr = p->ptr; a.M = p->rows;
  a.ldp = p->ldx; a.ldq = p->in_features; a.ldc = p->out_features; a.qstride = (int64_t)p->in_features * p->out_features;
  a.ni = -1; a.nj = p->out_features; a.nr = p->in_features; a.E = p->groups;
  const bool aligned = !((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->weight) | reinterpret_cast<uintptr_t>(y)) & 15) &&
                       p->in_features % ce == 0 && p->ldx % ce == 0 && p->out_features % ce == 0;
  const GlForm f = gl_pick_dtype<false, false>(p->dtype, a.nj, aligned);
  a.tj = dg_cdiv(a.nj, f.bj);
  return gl_launch(f, dg_align((p->rows / f.bi + p->groups + 2) * a.tj, 8), a, (hipStream_t)stream);
}

extern "C" int dgcnn_grouped_linear_bwd(const dgcnn_grouped_linear_args* p, const void* dy, void* dx, void* dweight, void* dbias, void* ws, dgcnn_stream_t stream) {
  const int rc = gl_check(p);
  if (rc != DGCNN_OK) return rc;
  if (p->rows > 0 && !dy) return DGCNN_EINVAL;
  if ((dweight || dbias) && !ws) return DGCNN_EINVAL;
  if (dbias && !dweight) return DGCNN_EINVAL;
  const int es = dg_dtype_size(p->dtype), ce = 16 / es;
  const bool wide = p->in_features % ce == 0 && p->out_features % ce == 0;
  if (dx && p->rows > 0) {
    DgGl a = {};
    a.p = dy; a.q = p->weight; a.c = dx; a.ptr = p->ptr; a.M = p->rows;
    a.ldp = p->out_features; a.ldq = p->in_features; a.ldc = p->in_features; a.qstride = (int64_t)p->in_features * p->out_features;
    a.ni = -1; a.nj = p->in_features; a.nr = p->out_features; a.E = p->groups;
    const bool aligned = wide && !((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(p->weight) | reinterpret_cast<uintptr_t>(dx)) & 15);
    const GlForm f = gl_pick_dtype<false, true>(p->dtype, a.nj, aligned);
    a.tj = dg_cdiv(a.nj, f.bj);
    const int r2 = gl_launch(f, dg_align((p->rows / f.bi + p->groups + 2) * a.tj, 8), a, (hipStream_t)stream);
    if (r2 != DGCNN_OK) return r2;
  }
  if (dweight && p->groups > 0) {
    DgGl a = {};
    a.p = dy; a.q = p->x; a.c = dweight; a.db = dbias; a.ptr = p->ptr; a.M = p->rows;
    a.ldp = p->out_features; a.ldq = p->ldx; a.ldc = p->in_features;
    a.ni = p->out_features; a.nj = p->in_features; a.nr = -1; a.E = p->groups;
    const bool aligned = wide && p->ldx % ce == 0 && !((reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(dweight)) & 15);
    const GlForm f = gl_pick_dtype<true, true>(p->dtype, a.nj, aligned);
    a.ti = dg_cdiv(a.ni, f.bi); a.tj = dg_cdiv(a.nj, f.bj);
    const int64_t tiles = (int64_t)a.ti * a.tj;
    a.slice = gl_slice(p->rows, p->groups, tiles);
    a.split = a.slice != 0;
    a.part = static_cast<float*>(ws);
    if (a.split && p->groups > 65535) return DGCNN_EUNSUPPORTED;
    a.slots = a.split ? p->rows / a.slice + p->groups : 0;
    const int r2 = gl_launch(f, (a.split ? a.slots : p->groups) * tiles, a, (hipStream_t)stream);
    if (r2 != DGCNN_OK) return r2;
    if (a.split) {
      const int64_t each = (int64_t)a.ni * a.nj + a.ni;
      const int64_t bx = (each + 255) / 256;
      const dim3 grid((unsigned)(bx < 4096 ? bx : 4096), p->groups);
      if (p->dtype == DGCNN_F32) hipLaunchKernelGGL(k_gl_join<DgF32>, grid, dim3(256), 0, (hipStream_t)stream, a);
      else if (p->dtype == DGCNN_BF16) hipLaunchKernelGGL(k_gl_join<DgBF16>, grid, dim3(256), 0, (hipStream_t)stream, a);
      else hipLaunchKernelGGL(k_gl_join<DgF16>, grid, dim3(256), 0, (hipStream_t)stream, a);
      DG_CHECK_LAUNCH();
    }
  }
  return DGCNN_OK;
}
