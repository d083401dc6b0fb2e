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
// Bound: the matrix units where rows a group are many, the weights' bytes where they are few.  Measured (MI355X; an 8192^3 library product reaches 1.4 PFLOP/s
// in bf16, a 1 GiB copy 5.2 TB/s): 131072 rows, 16 groups, 512 -> 512 bf16: y 131 us, dx 134, dW 143 + 12 (join) in a training pass, 116 for y alone, 590
// TFLOP/s (one library product of the same size, which knows no groups: 97 to 101 us); 48 rows, 8 groups, 1024 -> 1024 bf16: 7.3 us, of which 3.3 are the weights' 17 MB; 152576 rows,
// 3 groups, 97 -> 128 fp32: y 63 us, dx 72, dW 86 + 14.
#include "dg_half.h"

struct DgGl {
  const void *p, *q;             // operands (see above); q of group e begins at e * qstride
  const void* bias;              // y only: [groups][nj]
  void* c;                       // y, dx or dW
  float* part;                   // dW in slices: [slots] partial sums of dW, rows padded to 16 bytes, and of db
  void* db;                      // dW: [groups][ni], or null
  const int64_t* ptr;
  int64_t M;                     // rows
  int64_t ldp, ldq, ldc, qstride;
  int ni, nj, nr;                // extents of C and of the sum (ni: -1 where i runs over rows; nr: -1 where r does)
  int E;
  int tj, ti;                    // tiles along j (and, dW, along i)
  int shift;                     // dW: 2^shift rows a slice
  int split;                     // dW: 1: partial tiles
  int64_t slots;                 // ... that there is room for: enough for every ascending ptr
};

__host__ __device__ inline int gl_ld4(const DgGl& a) { return (a.nj + 3) & ~3; }
__host__ __device__ inline int64_t gl_each(const DgGl& a) { return (int64_t)a.ni * gl_ld4(a) + ((a.ni + 3) & ~3); }      // floats of a slot

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
// Every group has ceil(rows / 2^shift) work items.  The whole wave counts them, 64 groups at a time.
__device__ __forceinline__ int gl_scan(int x) {      // inclusive sum over the wave's lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);      // row_shr 1, 2, 4, 8: inside each 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);     // row_bcast 15, 31: the sums in front
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);
  return x;
}
struct GlItems {
  int n, upto;      // of this lane's group; up to and with it
  __device__ __forceinline__ void count(const DgGl& a, int groups, int shift, int e0) {
    const int lane = threadIdx.x & 63;
    n = 0;
    if (e0 + lane < groups) {
      int64_t lo, hi;
      gl_range(a, e0 + lane, lo, hi);
      n = (int)((hi - lo + ((int64_t)1 << shift) - 1) >> shift);
    }
    upto = gl_scan(n);
  }
};
__device__ __forceinline__ int gl_total(const DgGl& a, int groups, int shift, GlItems& c) {
  int total = 0;
  for (int e0 = 0; e0 < groups; e0 += 64) {
    c.count(a, groups, shift, e0);
    total += __builtin_amdgcn_readlane(c.upto, 63);
  }
  return total;
}
// item t -> its group and its index there (c: gl_total's counts, which are those of all groups if there are at most 64).  false: no such item, or -- a ptr
// that does not ascend -- none that lies in its group.
__device__ __forceinline__ bool gl_find(const DgGl& a, int groups, int shift, int t, GlItems c, int& e, int64_t& lo, int64_t& hi) {
  int base = 0;
  for (int e0 = 0; e0 < groups; e0 += 64) {
    if (groups > 64) c.count(a, groups, shift, e0);
    const uint64_t m = __ballot(base + c.upto > t);
    if (m) {
      const int k = __ffsll((long long)m) - 1;
      const int in = t - base - (__builtin_amdgcn_readlane(c.upto, k) - __builtin_amdgcn_readlane(c.n, k));
      e = e0 + k;
      gl_range(a, e, lo, hi);
      lo += (int64_t)in << shift;
      return in >= 0 && lo < hi;
    }
    base += __builtin_amdgcn_readlane(c.upto, 63);
  }
  return false;
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

// G = 16 or 4 bytes of every lane, from base (uniform) + off, to LDS at (uniform) dst + G * lane, without passing through registers.  In assembly because the
// compiler would wait for every such load before the next LDS read of any kind, i.e. never have one in flight; the LDS address is an
// operand in m0, so that the compiler knows of it (one wait state lies between a write of m0 and such a load); no register is written, the waits are gl_barrier's.
template <int G> __device__ __forceinline__ void gl_to_lds(const char* base, uint32_t off, char* dst) {
#ifdef DG_EMU
  for (int i = 0; i < G / 4; ++i) reinterpret_cast<uint32_t*>(dst + G * (threadIdx.x & 63))[i] = reinterpret_cast<const uint32_t*>(base + off)[i];
#else
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst);
  if constexpr (G == 16) asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" :: "{m0}"(at), "v"(off), "s"(base) : "memory");
  else asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, %2" :: "{m0}"(at), "v"(off), "s"(base) : "memory");
#endif
}
// the same from an address of each lane's own
template <int G> __device__ __forceinline__ void gl_to_lds(const char* src, char* dst) {
#ifdef DG_EMU
  gl_to_lds<G>(src, 0, dst);
#else
  const uint32_t at = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)dst);
  if constexpr (G == 16) asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "{m0}"(at), "v"(src) : "memory");
  else asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" :: "{m0}"(at), "v"(src) : "memory");
#endif
}
template <class T> __device__ __forceinline__ T* gl_uniform(T* p) {      // (the same in every lane: into scalar registers)
  const uint64_t v = (uint64_t)p;
  return (T*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
// all but the newest N of the wave's direct loads are in LDS, its LDS accesses are done, and so are the other waves'
template <int N> __device__ __forceinline__ void gl_barrier() {
#ifdef DG_EMU
  __syncthreads();
#else
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" :: "n"(N) : "memory");
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

__device__ __forceinline__ int gl_wave() { return __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }      // (scalar)

// One operand's tile: W indices (i or j) x R r values, ROWB = 64 or 128 bytes of them
//   T = false: memory and LDS [index][r]; chunk c of an index at place c ^ (index / (256 / ROWB)): 16 lanes read one chunk of 16 indices, which are then 16
//              different 16-byte pieces of the 256 bytes that the banks are wide
//   T = true : memory and LDS [r][index]; chunk c at place c ^ swizzle(r).  16-bit: a transposing read takes 32 bytes of r = 8g + j (j < 4, g < 4): j and one
//              bit of g pick the 32-byte piece.  fp32: 64 bytes of r = 4g + s: g picks it.
template <class D, int W, bool T, int ROWB> struct GlTile {
  typedef typename D::S S;
  static constexpr int ES = sizeof(S), CE = 16 / ES, R = ROWB / ES, BYTES = W * ROWB, CPR = W * ES / 16, CPI = ROWB / 16;
  static __device__ __forceinline__ int turn(int w) { return (w / (256 / ROWB)) & (CPI - 1); }
  static __device__ __forceinline__ int swizzle(int r) {
    if (ES == 4) return (((r >> 2) & 3) << 2) & (CPR - 1);
    return (((r & 3) | (((r >> 3) & 1) << 2)) << 1) & (CPR - 1);
  }
  // chunk q of the tile in LDS order: which index and r it begins at
  static __device__ __forceinline__ void place(int q, int& w, int& r) {
    if (T) { r = q / CPR; w = ((q % CPR) ^ swizzle(r)) * CE; }
    else { w = q / CPI; r = ((q % CPI) ^ turn(w)) * CE; }
  }
  // A direct load brings G bytes a lane: 16 where extents, strides and addresses are multiples of it, else 4 (fp32); 16-bit elements in odd places (G = 2)
  // come through registers.
  template <int G, int THREADS> static constexpr int loads() { return BYTES / (G < 4 ? 16 : G) / THREADS; }
  // Whole tiles: the lane's offsets from the tile's first element (indices behind the operand's last one read that one: they end in rows and columns of
  // C that are not stored), the same for every step.
  template <int G, int THREADS> static __device__ __forceinline__ void offsets(int64_t ld, int64_t left, uint32_t* off) {
    const int wave = gl_wave(), lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < loads<G, THREADS>(); ++k) {
      const int u = (k * (THREADS / 64) + wave) * 64 + lane;      // unit of G bytes
      int w, r;
      place(u / (16 / G), w, r);
      if (T) w += u % (16 / G); else r += u % (16 / G);
      const int last = (int)min(left, (int64_t)W) - (T ? 16 / (int)sizeof(S) / (16 / G) : 1);
      w = min(w, last);
      off[k] = (uint32_t)((T ? r * ld + w : w * ld + r) * ES);
    }
  }
  template <int G, int THREADS> static __device__ __forceinline__ void load(char* lds, const S* base, const uint32_t* off) {
    const int wave = gl_wave();
    const char* const at = gl_uniform(reinterpret_cast<const char*>(base));
#pragma unroll
    for (int k = 0; k < loads<G, THREADS>(); ++k) gl_to_lds<G>(at, off[k], lds + (k * (THREADS / 64) + wave) * 64 * G);
  }
  // the tile at (w0, r0) of an operand with nw indices and r values up to rend, zeros behind them
  template <int G, int THREADS>
  static __device__ __forceinline__ void load_part(char* lds, const S* base, int64_t ld, int64_t w0, int64_t r0, int64_t nw, int64_t rend) {
    const int wave = gl_wave(), lane = threadIdx.x & 63;
    if constexpr (G >= 4) {
#pragma unroll 4
      for (int k = 0; k < loads<G, THREADS>(); ++k) {
        const int u0 = (k * (THREADS / 64) + wave) * 64, u = u0 + lane;
        int w, r;
        place(u / (16 / G), w, r);
        if (T) w += u % (16 / G); else r += u % (16 / G);
        const S* const src = T ? base + (r0 + r) * ld + (w0 + w) : base + (w0 + w) * ld + (r0 + r);
        gl_to_lds<G>(w0 + w < nw && r0 + r < rend ? reinterpret_cast<const char*>(src) : reinterpret_cast<const char*>(gl_zero), lds + u0 * G);
      }
    } else {
#pragma unroll 2
      for (int k = 0; k < loads<G, THREADS>(); ++k) {
        const int q = (k * (THREADS / 64) + wave) * 64 + lane;
        int w, r;
        place(q, w, r);
        const S* const src = T ? base + (r0 + r) * ld + (w0 + w) : base + (w0 + w) * ld + (r0 + r);
        DgRaw<D, CE> v = dg_zero<D, CE>();
#pragma unroll
        for (int i = 0; i < CE; ++i)
          if (T ? w0 + w + i < nw && r0 + r < rend : w0 + w < nw && r0 + r + i < rend) v.v[i] = src[i];
        dg_store<D, CE>(reinterpret_cast<S*>(lds + q * 16), v);
      }
    }
  }
  // the lane's r values of index w0 + lane % 16 in the s-th 64 bytes of r: CE (4 s + lane / 16) + 0 .. CE-1
  static __device__ __forceinline__ gl_u32x4 fragment(const char* lds, int w0, int s) {
    const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
    if constexpr (!T) {
      const int w = w0 + l;
      return *reinterpret_cast<const gl_u32x4*>(lds + w * ROWB + (((s * 4 + g) ^ turn(w)) << 4));
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

// WI x WJ waves of (16 FI) x (16 FJ) tiles of C, ST stages of ROWB bytes of r
template <class D, int WI, int WJ, int FI, int FJ, int ST, int ROWB, bool PT, bool QT, int G>
__global__ void __launch_bounds__(64 * WI * WJ) __attribute__((amdgpu_waves_per_eu(2)))
k_gl(const DgGl a) {
  constexpr int BI = WI * FI * 16, BJ = WJ * FJ * 16, THREADS = 64 * WI * WJ;
  constexpr bool GRAD = PT;                                   // the product over rows
  typedef typename D::S S;
  typedef GlTile<D, BI, PT, ROWB> TP;
  typedef GlTile<D, BJ, QT, ROWB> TQ;
  constexpr int R = TP::R;
  constexpr int STAGE = TP::BYTES + TQ::BYTES, LP = TP::template loads<G, THREADS>(), LQ = TQ::template loads<G, THREADS>();      // (loads of a wave and stage)
  DG_DYN_SMEM(char, smem);                                    // ST stages of P and Q
  const int wave = gl_wave(), lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
  const int wi = wave / WJ, wj = wave - wi * WJ;

  // ---- which tile: C's rows lo .. (fewer than nw_i) and columns j0 .., the sum over r0 .. rend - 1
  int e = 0, j0, slot = 0;
  int64_t lo, hi, r0, rend, nw_i;
  const S *p = static_cast<const S*>(a.p), *q = static_cast<const S*>(a.q);
  GlItems items;
  if (!GRAD) {
    // consecutive tiles (the columns of one run of rows first) on one XCD: workgroups go to the eight in turn
    constexpr int SHIFT = BI == 16 ? 4 : BI == 32 ? 5 : BI == 64 ? 6 : BI == 128 ? 7 : 8;
    static_assert(BI == 1 << SHIFT, "rows a tile");
    const unsigned tiles = (unsigned)gl_total(a, a.E + 2, SHIFT, items) * a.tj, share = (tiles + 7) >> 3, t = (blockIdx.x & 7) * share + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= share || t >= tiles) return;
    if (!gl_find(a, a.E + 2, SHIFT, (int)(t / (unsigned)a.tj), items, e, lo, hi)) return;
    j0 = (int)(t % (unsigned)a.tj) * BJ;
    nw_i = hi;
    r0 = 0; rend = a.nr;
    if (e >= a.E) {                                           // rows of no group
      S* const c = static_cast<S*>(a.c);
      for (int k = threadIdx.x; k < BI * BJ; k += THREADS) {
        const int64_t i = lo + k / BJ;
        const int j = j0 + k % BJ;
        if (i < hi && j < a.nj) c[i * a.ldc + j] = D::from(0.f);
      }
      return;
    }
    q += (int64_t)e * a.qstride;
  } else {
    // the tiles of a slice (or group), which read the same rows, on one XCD
    const unsigned per = a.ti * a.tj, on = blockIdx.x >> 3, tile = on % per, t = on / per * 8 + (blockIdx.x & 7);
    if (t >= (a.split ? (unsigned)a.slots : (unsigned)a.E)) return;
    if (a.split) {
      gl_total(a, a.E, a.shift, items);
      if (!gl_find(a, a.E, a.shift, (int)t, items, e, lo, hi)) return;
      slot = (int)t;
      r0 = lo;
      rend = min(r0 + ((int64_t)1 << a.shift), hi);
    } else {
      e = (int)t;
      gl_range(a, e, r0, rend);
    }
    lo = (int)(tile / (unsigned)a.tj) * BI; j0 = (int)(tile % (unsigned)a.tj) * BJ;
    nw_i = a.ni;
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

  const bool whole4 = G == 16 || ((reinterpret_cast<uintptr_t>(a.c) & (4 * sizeof(S) - 1)) == 0 && (a.nj & 3) == 0);      // every four columns are one access
  float b[GRAD ? 1 : FJ][4];      // the bias of the lane's columns: asked for here, long before it is added
  if constexpr (!GRAD) {
#pragma unroll
    for (int j = 0; j < FJ; ++j) {
      const int col = j0 + (wj * FJ + j) * 16 + 4 * g;
#pragma unroll
      for (int k = 0; k < 4; ++k) b[j][k] = 0.f;
      if (a.bias && col < a.nj) {
        const S* const bias = static_cast<const S*>(a.bias) + (int64_t)e * a.nj;
        if (G == 16) {
          const DgRaw<D, 4> v = dg_load<D, 4>(bias + col);
#pragma unroll
          for (int k = 0; k < 4; ++k) b[j][k] = v.get(k);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) b[j][k] = D::to(bias[min(col + k, a.nj - 1)]);
        }
      }
    }
  }

  // ---- ST stages: ST - 1 of them are on their way or being multiplied, the one that was multiplied last is loaded anew.  One barrier a step: it
  // says that this step's stage has arrived (all but the ST - 2 newer ones' loads are done) and that everyone is through with the last one.
  const int whole = (int)((rend - r0) / R), steps = (int)((rend - r0 + R - 1) / R);
  uint32_t op[G >= 4 ? LP : 1], oq[G >= 4 ? LQ : 1];
  const S *bp = nullptr, *bq = nullptr;
  if constexpr (G >= 4) {
    TP::template offsets<G, THREADS>(a.ldp, nw_i - lo, op);
    TQ::template offsets<G, THREADS>(a.ldq, a.nj - j0, oq);
    bp = PT ? p + r0 * a.ldp + lo : p + lo * a.ldp + r0;
    bq = QT ? q + r0 * a.ldq + j0 : q + j0 * a.ldq + r0;
  }
  auto load = [&](int k) {      // (steps are loaded one after the other)
    char* const at = smem + (k % ST) * STAGE;
    if (G >= 4 && k < whole) {
      TP::template load<G, THREADS>(at, bp, op);
      TQ::template load<G, THREADS>(at + TP::BYTES, bq, oq);
      bp += PT ? R * a.ldp : R;
      bq += QT ? R * a.ldq : R;
    } else {
      TP::template load_part<G, THREADS>(at, p, a.ldp, lo, r0 + (int64_t)k * R, nw_i, rend);
      TQ::template load_part<G, THREADS>(at + TP::BYTES, q, a.ldq, j0, r0 + (int64_t)k * R, a.nj, rend);
    }
  };
#pragma unroll
  for (int k = 0; k < ST - 1; ++k) if (k < steps) load(k);
  for (int k = 0; k < steps; ++k) {
    if (G >= 4 && k + ST - 2 < steps) gl_barrier<G >= 4 ? (LP + LQ) * (ST - 2) : 0>(); else gl_barrier<0>();
    if (k + ST - 1 < steps) load(k + ST - 1);
    char* const now = smem + (k % ST) * STAGE;
#pragma unroll
    for (int s = 0; s < ROWB / 64; ++s) {
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
  }
  gl_barrier<0>();      // (nothing may be on its way to LDS when the workgroup ends)

  // ---- C: the lane holds row l and columns 4g .. 4g+3 of every 16 x 16 tile
  const int left = (int)min(nw_i - lo, (int64_t)BI), wide = min(a.nj - j0, BJ);      // rows and columns of C in this tile
  const int row = wi * FI * 16 + l, col = wj * FJ * 16 + 4 * g;
  if (GRAD && a.split) {
    float* const c = a.part + (int64_t)slot * gl_each(a) + lo * gl_ld4(a) + j0;      // (rows of 16-byte multiples)
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j)
        if (row + 16 * i < left && col + 16 * j < wide) *reinterpret_cast<f32x4*>(c + (row + 16 * i) * gl_ld4(a) + col + 16 * j) = acc[i][j];
    if (sums && g == 0) {
      float* const d = a.part + (int64_t)slot * gl_each(a) + (int64_t)a.ni * gl_ld4(a) + lo;
#pragma unroll
      for (int i = 0; i < FI; ++i) if (row + 16 * i < left) d[row + 16 * i] = sum[i][0];
    }
    return;
  }
  S* const c = static_cast<S*>(a.c) + (GRAD ? (int64_t)e * a.ni * a.nj : 0) + lo * a.ldc + j0;
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    const int n = wide - (col + 16 * j);      // columns that are there
#pragma unroll
    for (int i = 0; i < FI; ++i) {
      if (row + 16 * i >= left || n <= 0) continue;
      S* const at = c + (uint32_t)(row + 16 * i) * (uint32_t)a.ldc + (uint32_t)(col + 16 * j);
      if (whole4) {
        DgRaw<D, 4> o;
#pragma unroll
        for (int k = 0; k < 4; ++k) o.set(k, GRAD ? acc[i][j][k] : acc[i][j][k] + b[GRAD ? 0 : j][k]);
        dg_store<D, 4>(at, o);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) if (k < n) at[k] = D::from(GRAD ? acc[i][j][k] : acc[i][j][k] + b[GRAD ? 0 : j][k]);
      }
    }
  }
  if (GRAD && sums && g == 0) {
    S* const d = static_cast<S*>(a.db) + (int64_t)e * a.ni + lo;
#pragma unroll
    for (int i = 0; i < FI; ++i) if (row + 16 * i < left) d[row + 16 * i] = D::from(sum[i][0]);
  }
}

// dW and db from the slices' partial tiles, slice after slice; a group without rows gets zeros.  Four columns (or four of db) a thread.
template <class D>
__global__ void __launch_bounds__(256)
k_gl_join(const DgGl a) {
  typedef typename D::S S;
  const int64_t each = gl_each(a);
  const int e = blockIdx.y;
  int64_t first = 0, slices = 0;      // slots in front of group e's; its own
  for (int e0 = 0; e0 <= e; e0 += 64) {
    GlItems c;
    c.count(a, e + 1, a.shift, e0);
    first += __builtin_amdgcn_readlane(c.upto, 63);
    if (e - e0 < 64) slices = __builtin_amdgcn_readlane(c.n, e - e0);
  }
  first -= slices;
  const int quads = gl_ld4(a) / 4;
  for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; 4 * k < each; k += (int64_t)gridDim.x * 256) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    const float* const p = a.part + first * each + 4 * k;
    const int n = (int)min(slices, max(a.slots - first, (int64_t)0));
#pragma unroll 4
    for (int i = 0; i < n; ++i) s += *reinterpret_cast<const f32x4*>(p + i * each);
    const int64_t row = k / quads;
    if (row < a.ni) {
      const int col = (int)(k % quads) * 4;
      S* const c = static_cast<S*>(a.c) + ((int64_t)e * a.ni + row) * a.nj + col;
      if ((a.nj & 3) == 0 && (reinterpret_cast<uintptr_t>(a.c) & (4 * sizeof(S) - 1)) == 0) {
        DgRaw<D, 4> o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o.set(i, s[i]);
        dg_store<D, 4>(c, o);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) if (col + i < a.nj) c[i] = D::from(s[i]);
      }
    } else if (a.db) {
      const int64_t i0 = 4 * k - (int64_t)a.ni * gl_ld4(a);
#pragma unroll
      for (int i = 0; i < 4; ++i) if (i0 + i < a.ni) static_cast<S*>(a.db)[(int64_t)e * a.ni + i0 + i] = D::from(s[i]);
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
typedef void (*gl_kernel)(const DgGl);
struct GlForm { gl_kernel k; int bi, bj, threads, lds; };
template <class D, int WI, int WJ, int FI, int FJ, int ST, int ROWB, bool PT, bool QT> static GlForm gl_form(bool aligned) {
  GlForm f;
  f.k = aligned ? (gl_kernel)k_gl<D, WI, WJ, FI, FJ, ST, ROWB, PT, QT, 16> : (gl_kernel)k_gl<D, WI, WJ, FI, FJ, ST, ROWB, PT, QT, sizeof(typename D::S)>;
  f.bi = WI * FI * 16; f.bj = WJ * FJ * 16; f.threads = 64 * WI * WJ;
  f.lds = ST * (f.bi + f.bj) * ROWB;
  return f;
}
// The tile for a shape (rows: of the whole call; nj: columns of C).  Measured, us, forward unless said:
//   16 x 32, six stages: few rows, where the weights are the work and every workgroup has to stream its own share.  bf16, 8 groups, 1024 -> 1024: 48 rows 6.9 (128 x
//     128: 12.9), 256 rows 8.4 (13.1), 512 rows 10.0 (13.3), 1024 rows 18.6 (14.5): up to 1024 tiles.  4096 -> 4096, 256 rows, 2048 tiles: 78 (60).  fp32, whose larger
//     tiles multiply rows that are not there: 1024 rows 41 (78), 2048 rows 77 (79), 4096 -> 4096 256 rows 203 (295): up to 2048 tiles.
//   128 x 32: narrow results.
//   256 x 256, one workgroup a CU: 131072 rows 512 -> 512 bf16 116 (130), 1024 -> 512 178 (208), 8192 rows 4096 -> 4096 240 (294); but 16384 rows 4096 -> 512, 128 tiles
//     of it, 108 (70): from two tiles a CU on.
//   128 x 128 otherwise; 64 bytes of r in three stages (three workgroups a CU) for fp32 (97 -> 128 forward 63, 128 bytes in two stages 77) and dW (131, 138), 128 bytes in
//     two for the others (16384 rows 4096 -> 512: 70, 87).
template <class D, bool PT, bool QT> static GlForm gl_pick(int64_t rows, int E, int nj, bool aligned) {
  constexpr bool WIDE = sizeof(typename D::S) == 4;
  if constexpr (!PT) {
    if (rows <= 16 * (int64_t)E || (rows + 15) / 16 * ((nj + 31) / 32) <= (WIDE ? 2048 : 1024)) return gl_form<D, 1, 2, 1, 1, 6, 128, PT, QT>(aligned);
  }
  if (nj <= 32) return gl_form<D, 4, 1, 2, 2, 2, 128, PT, QT>(aligned);
  if constexpr (!PT && !WIDE) {
    if (nj >= 256 && rows / 256 * ((nj + 255) / 256) >= 512) return gl_form<D, 2, 4, 8, 4, 2, 128, PT, QT>(aligned);
    return gl_form<D, 2, 2, 4, 4, 2, 128, PT, QT>(aligned);
  }
  return gl_form<D, 2, 2, 4, 4, 3, 64, PT, QT>(aligned);
}
template <bool PT, bool QT> static GlForm gl_pick_dtype(int dtype, int64_t rows, int E, int nj, bool aligned) {
  return dtype == DGCNN_F32 ? gl_pick<DgF32, PT, QT>(rows, E, nj, aligned) : dtype == DGCNN_BF16 ? gl_pick<DgBF16, PT, QT>(rows, E, nj, aligned) : gl_pick<DgF16, PT, QT>(rows, E, nj, aligned);
}
static int gl_launch(const GlForm& f, int64_t blocks, const DgGl& a, hipStream_t s) {
  if (blocks <= 0) return DGCNN_OK;
  if (blocks > 0xffffffffll / f.threads) return DGCNN_EUNSUPPORTED;      // (a grid holds fewer than 2^32 threads)
  if (f.lds > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(f.k), hipFuncAttributeMaxDynamicSharedMemorySize, f.lds) != hipSuccess) return DGCNN_ELAUNCH;
  hipLaunchKernelGGL(f.k, dim3((unsigned)blocks), dim3(f.threads), f.lds, s, a);
  DG_CHECK_LAUNCH();
  return DGCNN_OK;
}
// dW: log2 of the rows a slice, or 0 for one slice a group.  As many slices as fill the chip twice over (512 workgroups), each of at least 512 rows.
static int gl_slice(int64_t rows, int E, int64_t tiles) {
  if (tiles * E >= 512) return 0;
  const int64_t want = (512 + tiles - 1) / tiles;
  int shift = 9;
  while (((int64_t)1 << shift) * want < rows) ++shift;
  return shift;
}
static int gl_check(const dgcnn_grouped_linear_args* p) {
  if (!p || p->rows < 0 || p->in_features < 1 || p->out_features < 1 || p->groups < 0 || !dg_dtype_ok(p->dtype) || !p->ptr) return DGCNN_EINVAL;
  if (p->ldx < p->in_features) return DGCNN_EINVAL;
  if (p->rows > 0 && !p->x) return DGCNN_EINVAL;
  if (p->groups > 0 && !p->weight) return DGCNN_EINVAL;
  if (p->rows > ((int64_t)1 << 40) / p->ldx || p->rows > ((int64_t)1 << 40) / p->out_features ||
      (int64_t)p->in_features * p->out_features > ((int64_t)1 << 40) / (p->groups ? p->groups : 1) || p->groups > (1 << 20)) return DGCNN_EUNSUPPORTED;
  if (p->ldx > (1 << 21) || p->out_features > (1 << 21)) return DGCNN_EUNSUPPORTED;      // (offsets inside a tile's 256 rows are 32-bit)
  return DGCNN_OK;
}

extern "C" int64_t dgcnn_grouped_linear_workspace_bytes(int64_t rows, int in_features, int out_features, int groups, int dtype) {
  if (rows < 0 || in_features < 1 || out_features < 1 || groups < 0 || !dg_dtype_ok(dtype)) return DGCNN_EINVAL;
  const GlForm f = gl_pick_dtype<true, true>(dtype, rows, groups, in_features, true);
  const int64_t tiles = (int64_t)dg_cdiv(out_features, f.bi) * dg_cdiv(in_features, f.bj);
  const int shift = gl_slice(rows, groups, tiles);
  if (!shift) return 256;
  DgGl a = {};
  a.ni = out_features; a.nj = in_features;
  return dg_align(((rows >> shift) + groups) * gl_each(a) * 4, 256);
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
  const bool aligned = !((reinterpret_cast<uintptr_t>(p->x) | reinterpret_cast<uintptr_t>(p->weight) | reinterpret_cast<uintptr_t>(p->bias) | reinterpret_cast<uintptr_t>(y)) & 15) &&
                       p->in_features % ce == 0 && p->ldx % ce == 0 && p->out_features % ce == 0;
  const GlForm f = gl_pick_dtype<false, false>(p->dtype, p->rows, p->groups, a.nj, aligned);
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
    const GlForm f = gl_pick_dtype<false, true>(p->dtype, p->rows, p->groups, a.nj, aligned);
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
    const GlForm f = gl_pick_dtype<true, true>(p->dtype, p->rows, p->groups, a.nj, aligned);
    a.ti = dg_cdiv(a.ni, f.bi); a.tj = dg_cdiv(a.nj, f.bj);
    const int64_t tiles = (int64_t)a.ti * a.tj;
    a.shift = gl_slice(p->rows, p->groups, tiles);
    a.split = a.shift != 0;
    a.part = static_cast<float*>(ws);
    if (a.split && p->groups > 65535) return DGCNN_EUNSUPPORTED;
    a.slots = a.split ? (p->rows >> a.shift) + p->groups : 0;
    const int r2 = gl_launch(f, dg_align(a.split ? a.slots : p->groups, 8) * tiles, a, (hipStream_t)stream);
    if (r2 != DGCNN_OK) return r2;
    if (a.split) {
      const int64_t bx = (gl_each(a) / 4 + 255) / 256;
      const dim3 grid((unsigned)(bx < 4096 ? bx : 4096), p->groups);
      if (p->dtype == DGCNN_F32) hipLaunchKernelGGL(k_gl_join<DgF32>, grid, dim3(256), 0, (hipStream_t)stream, a);
      else if (p->dtype == DGCNN_BF16) hipLaunchKernelGGL(k_gl_join<DgBF16>, grid, dim3(256), 0, (hipStream_t)stream, a);
      else hipLaunchKernelGGL(k_gl_join<DgF16>, grid, dim3(256), 0, (hipStream_t)stream, a);
      DG_CHECK_LAUNCH();
    }
  }
  return DGCNN_OK;
}
