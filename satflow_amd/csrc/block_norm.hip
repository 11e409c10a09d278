// Token norms around a residual block, fused with the block's gate, residual scale and residual sum, forward and backward:
//   h = (u - mean) * rstd  over each group of C / groups channels   (SF_NORM_RMS: mean = 0, rstd = 1 / sqrt(mean(u^2) + eps))
//   n = h * w + b ,  z = s * silu(gate) * n ,  r = residual + z ,  y = the same norm of r over all channels with the next block's nw, nb
// Backward, D = dr + (dh' - h' <dh', h'> - <dh'>) * rstd'  with dh' = dy * nw, h' the normalised r, <.> the mean over the row (its second use only for
// SF_NORM_LAYER):   d residual = D ,  ds = sum_rows D silu(gate) n ,  dgate = D s n silu'(gate) ,  dn = D s silu(gate) ,  dw = sum_rows dn h ,
//   db = sum_rows dn ,  du = (dn w - h <dn w h> - <dn w>) * rstd ,  dnw = sum_rows dy h' ,  dnb = sum_rows dy.
// Everything is fp32 in registers: a row is read once, rounded once per output.  The backward pass takes r again from its inputs in fp32 instead of reading
// the stored r: the same bytes (residual instead of r), and the normalised r does not carry r's rounding to 16 bits into dnw (which is an fp32 sum).
#include "sf_common.h"

namespace {

struct NormP {
  const void *u, *gate, *res;
  const float *w, *b, *s, *nw, *nb;
  void *r, *y;
  float *stats, *nstats;   // [rows][groups][2], [rows][2]: mean, rstd
  int64_t ldu, ldg, ldx, ldr, ldy;
  int64_t rows;
  int cg, groups, tpr, layer;
  float eps;
  // backward
  const void *dr, *dy;
  void *du, *dgate, *dres;
  int64_t lddr, lddy, lddu, lddg, lddx;
  int aligned;             // parameters on 16 bytes
  float* partial[5];       // [gridDim.x][C] of dw, db, ds, dnw, dnb; null where the sum is not wanted
};

// A barrier for LDS alone: its writes are waited for, reads and writes of memory in flight are not (__syncthreads() waits for those too).
__device__ __forceinline__ void block_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One step of a sum over neighbouring lanes without LDS: quad, half-row and row patterns (the values of a quad / half-row are equal when its step comes).
template <int CTRL> __device__ __forceinline__ float add_dpp(float a) {
  return a + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, a), CTRL, 0xf, 0xf, true));
}

// Sums of two values over the `tpr` threads that hold a row.  red: 2 x 2 x 16 floats, the halves used in turn, so that one barrier per call is enough
// (a wave can be at most one call behind another).
struct RowSum {
  float* red;
  int tpr, phase;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    a = add_dpp<0xB1>(a); b = add_dpp<0xB1>(b);        // lanes 1 apart
    a = add_dpp<0x4E>(a); b = add_dpp<0x4E>(b);        // 2 apart
    a = add_dpp<0x141>(a); b = add_dpp<0x141>(b);      // the other quad of eight lanes
    if (tpr >= 16) { a = add_dpp<0x140>(a); b = add_dpp<0x140>(b); }   // the other half of sixteen
    if (tpr >= 32) { a += __shfl_xor(a, 16); b += __shfl_xor(b, 16); }
    if (tpr >= 64) { a += __shfl_xor(a, 32); b += __shfl_xor(b, 32); }
    if (tpr <= 64) return;
    float* half = red + phase * 32;
    phase ^= 1;
    const int wave = threadIdx.x >> 6, nw = tpr >> 6, first = wave / nw * nw;
    if ((threadIdx.x & 63) == 0) { half[2 * wave] = a; half[2 * wave + 1] = b; }
    block_sync();
    a = 0.f; b = 0.f;
    for (int i = 0; i < nw; i++) { a += half[2 * (first + i)]; b += half[2 * (first + i) + 1]; }
  }
};

// The NE channels of a thread, as stored: vectors of 8 when VEC (rows 16-byte aligned, C / groups a multiple of 8), single channels tpr apart otherwise.
template <typename T, int NE> struct Raw {
  typedef T vec __attribute__((ext_vector_type(8)));
  vec v[NE / 8];
  __device__ __forceinline__ float operator[](int j) const { return (float)v[j >> 3][j & 7]; }
};
template <int NE, bool VEC> struct Cols {
  int lane, tpr, n;
  __device__ __forceinline__ int at(int j) const { return VEC ? (lane + (j >> 3) * tpr) * 8 + (j & 7) : lane + j * tpr; }
  template <typename T> __device__ __forceinline__ void load(const void* base, int64_t off, bool live, Raw<T, NE>& r) const {
    const T* p = (const T*)base + off;
#pragma unroll
    for (int i = 0; i < NE / 8; i++) {
      r.v[i] = {};
      if constexpr (VEC) {
        const int c = (lane + i * tpr) * 8;
        if (live && c < n) r.v[i] = *reinterpret_cast<const typename Raw<T, NE>::vec*>(p + c);
      } else {
#pragma unroll
        for (int k = 0; k < 8; k++) {
          const int c = at(8 * i + k);
          if (live && c < n) r.v[i][k] = p[c];
        }
      }
    }
  }
  template <typename T> __device__ __forceinline__ void store(void* base, int64_t off, bool live, const float (&v)[NE]) const {
    T* p = (T*)base + off;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NE / 8; i++) {
        const int c = (lane + i * tpr) * 8;
        f32x8_t x;
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = v[8 * i + k];
        if (live && c < n) stv8<T>(p + c, x);
      }
    } else {
#pragma unroll
      for (int j = 0; j < NE; j++) {
        const int c = at(j);
        if (live && c < n) p[c] = (T)v[j];
      }
    }
  }
  // a parameter row (fp32; `fill` where there is none and in the columns behind the row)
  __device__ __forceinline__ void param(const float* p, int off, float fill, float (&v)[NE]) const {
#pragma unroll
    for (int j = 0; j < NE; j++) {
      const int c = at(j);
      v[j] = p && c < n ? p[off + c] : fill;
    }
  }
};

__device__ __forceinline__ float silu(float g, float& sig) {
  sig = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * g));
  return g * sig;
}

// mean and 1 / sqrt(var + eps) of a row held in registers; the variance from the centred values.
template <int NE, bool VEC>
__device__ __forceinline__ void row_stats(const Cols<NE, VEC>& cols, RowSum& sum, const float (&v)[NE], int n, bool layer, float eps, float& mean, float& rstd) {
  float a = 0.f, b = 0.f;
  mean = 0.f;
  if (layer) {
#pragma unroll
    for (int j = 0; j < NE; j++) a += v[j];   // (zeros behind the row)
    sum(a, b);
    mean = a / n;
  }
  a = 0.f; b = 0.f;
#pragma unroll
  for (int j = 0; j < NE; j++) {
    const float d = cols.at(j) < n ? v[j] - mean : 0.f;
    a = __builtin_fmaf(d, d, a);
  }
  sum(a, b);
  rstd = 1.0f / sqrtf(a / n + eps);
}

// Both kernels read the next row of a slot while they work on one, and keep the parameters of their columns in registers over the rows.  Bound by memory: 16384
// rows of 4096 bf16 channels with gate, fp32 residual and the next norm: 184 us a call for 940 MB, 5.1 TB/s, the rate of a copy; 8192 rows of 2048 in training: 47
// us forward (168 MB, 3.6 TB/s) and 67 backward (235 MB, 3.5 TB/s) + 4.5 for the column sums.  That is no bound of memory - copies of 168 and 235 MB, which the last
// cache holds, take 20 and 28 us -: the backward kernel has 208 registers, two waves a SIMD, and carries five column sums whether they are asked for or not.  96 rows of
// 256 fp32: 5.0 us, a launch.
template <typename A, typename R, int NE, bool VEC, bool NEXT, int BLOCK> __global__ void __launch_bounds__(BLOCK) norm_fwd_kernel(NormP p) {
  __shared__ float red[64];
  const int slots = blockDim.x / p.tpr, slot = threadIdx.x / p.tpr;
  Cols<NE, VEC> cols{(int)(threadIdx.x % p.tpr), p.tpr, p.cg};
  RowSum sum{red, p.tpr, 0};
  const int g = blockIdx.y, goff = g * p.cg;
  const int64_t step = (int64_t)gridDim.x * slots;
  Raw<A, NE> ru, rg;
  Raw<R, NE> rx;
  auto fetch = [&](int64_t row) {
    const bool live = row < p.rows;
    cols.template load<A>(p.u, row * p.ldu + goff, live, ru);
    if (p.gate) cols.template load<A>(p.gate, row * p.ldg + goff, live, rg);
    if (p.res) cols.template load<R>(p.res, row * p.ldx + goff, live, rx);
  };
  int64_t base = (int64_t)blockIdx.x * slots;
  if (base < p.rows) fetch(base + slot);
  float w[NE], b[NE], s[NE], nw[NE], nb[NE];
  cols.param(p.w, goff, 1.f, w); cols.param(p.b, goff, 0.f, b); cols.param(p.s, goff, 1.f, s);
  if (NEXT) { cols.param(p.nw, goff, 0.f, nw); cols.param(p.nb, goff, 0.f, nb); }
  for (; base < p.rows; base += step) {
    const int64_t row = base + slot;
    const bool live = row < p.rows;
    const Raw<A, NE> cg = rg;
    const Raw<R, NE> cx = rx;
    float u[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) u[j] = ru[j];
    if (base + step < p.rows) fetch(row + step);
    float mean, rstd;
    row_stats(cols, sum, u, p.cg, p.layer, p.eps, mean, rstd);
    if (p.stats && live && cols.lane == 0) { float* st = p.stats + (row * p.groups + g) * 2; st[0] = mean; st[1] = rstd; }
#pragma unroll
    for (int j = 0; j < NE; j++) {
      float z = s[j] * __builtin_fmaf((u[j] - mean) * rstd, w[j], b[j]), sig;
      if (p.gate) z *= silu(cg[j], sig);
      u[j] = p.res ? cx[j] + z : z;
      if (cols.at(j) >= p.cg) u[j] = 0.f;
    }
    cols.template store<R>(p.r, row * p.ldr + goff, live, u);
    if constexpr (NEXT) {
      row_stats(cols, sum, u, p.cg, p.layer, p.eps, mean, rstd);
      if (p.nstats && live && cols.lane == 0) { p.nstats[row * 2] = mean; p.nstats[row * 2 + 1] = rstd; }
#pragma unroll
      for (int j = 0; j < NE; j++) u[j] = __builtin_fmaf((u[j] - mean) * rstd, nw[j], nb[j]);
      cols.template store<A>(p.y, row * p.ldy, live, u);
    }
  }
}

// Column sums: a thread keeps the sums of its columns in registers over the rows of its slot; the block's slots are added through LDS, the blocks by
// norm_reduce_kernel in block order (no atomics: the result does not depend on timing).  NEXT: there is a gradient of y.
template <typename A, typename R, int NE, bool VEC, bool NEXT, int BLOCK> __global__ void __launch_bounds__(BLOCK) norm_bwd_kernel(NormP p) {
  extern __shared__ float lds[];
  float* red = lds;            // 64 floats
  float* acc = lds + 64;       // [slots][cg] (slots > 1)
  const int slots = blockDim.x / p.tpr, slot = threadIdx.x / p.tpr;
  Cols<NE, VEC> cols{(int)(threadIdx.x % p.tpr), p.tpr, p.cg};
  RowSum sum{red, p.tpr, 0};
  const int g = blockIdx.y, goff = g * p.cg;
  const int64_t step = (int64_t)gridDim.x * slots;
  Raw<A, NE> ru, rg, ry;
  Raw<R, NE> rx, rr;
  float st[2], nst[2];
  auto fetch = [&](int64_t row) {
    const bool live = row < p.rows;
    cols.template load<A>(p.u, row * p.ldu + goff, live, ru);
    if (p.gate) cols.template load<A>(p.gate, row * p.ldg + goff, live, rg);
    if (p.dr) cols.template load<R>(p.dr, row * p.lddr + goff, live, rr);
    if (NEXT) {
      if (p.res) cols.template load<R>(p.res, row * p.ldx + goff, live, rx);
      cols.template load<A>(p.dy, row * p.lddy, live, ry);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
      st[i] = live ? p.stats[(row * p.groups + g) * 2 + i] : 0.f;
      if (NEXT) nst[i] = live ? p.nstats[row * 2 + i] : 0.f;
    }
  };
  int64_t base = (int64_t)blockIdx.x * slots;
  if (base < p.rows) fetch(base + slot);
  float w[NE], b[NE], s[NE], nw[NE];
  cols.param(p.w, goff, 1.f, w); cols.param(p.b, goff, 0.f, b); cols.param(p.s, goff, 1.f, s);
  if (NEXT) cols.param(p.nw, goff, 1.f, nw);
  float gw[NE] = {}, gb[NE] = {}, gs[NE] = {}, gnw[NE] = {}, gnb[NE] = {};
  const float inv = 1.0f / p.cg;
  for (; base < p.rows; base += step) {
    const int64_t row = base + slot;
    const bool live = row < p.rows;
    const float mean = st[0], rstd = st[1], nmean = nst[0], nrstd = nst[1];
    const Raw<A, NE> cg = rg, cy = ry;
    const Raw<R, NE> cx = rx;
    float h[NE], d[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) { h[j] = (ru[j] - mean) * rstd; d[j] = p.dr ? rr[j] : 0.f; }
    if (base + step < p.rows) fetch(row + step);
    float c1 = 0.f, c2 = 0.f;
    if constexpr (NEXT) {
      float x[NE];
#pragma unroll
      for (int j = 0; j < NE; j++) {   // x: the normalised r
        float z = s[j] * __builtin_fmaf(h[j], w[j], b[j]), sig;
        if (p.gate) z *= silu(cg[j], sig);
        x[j] = ((p.res ? cx[j] + z : z) - nmean) * nrstd;
        if (cols.at(j) >= p.cg) x[j] = 0.f;
        const float dy = cy[j], t = dy * nw[j];
        gnw[j] = __builtin_fmaf(dy, x[j], gnw[j]); gnb[j] += dy;
        c1 = __builtin_fmaf(t, x[j], c1); c2 += t;
      }
      sum(c1, c2);
      c1 *= inv; c2 = p.layer ? c2 * inv : 0.f;
#pragma unroll
      for (int j = 0; j < NE; j++) d[j] += (cy[j] * nw[j] - x[j] * c1 - c2) * nrstd;
    }
    if (p.dres) cols.template store<R>(p.dres, row * p.lddx + goff, live, d);
    c1 = 0.f; c2 = 0.f;
    float dg[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) {
      if (cols.at(j) >= p.cg) d[j] = 0.f;
      const float n = __builtin_fmaf(h[j], w[j], b[j]);
      float sig = 0.f, a = 1.f;
      if (p.gate) {
        const float gt = cg[j];
        a = silu(gt, sig);
        dg[j] = d[j] * s[j] * n * (sig * (1.0f + gt * (1.0f - sig)));
      }
      gs[j] = __builtin_fmaf(d[j] * a, n, gs[j]);
      const float dn = d[j] * s[j] * a;
      gw[j] = __builtin_fmaf(dn, h[j], gw[j]); gb[j] += dn;
      d[j] = dn * w[j];
      c1 = __builtin_fmaf(d[j], h[j], c1); c2 += d[j];
    }
    if (p.dgate) cols.template store<A>(p.dgate, row * p.lddg + goff, live, dg);
    if (p.du) {
      sum(c1, c2);
      c1 *= inv; c2 = p.layer ? c2 * inv : 0.f;
#pragma unroll
      for (int j = 0; j < NE; j++) d[j] = (d[j] - h[j] * c1 - c2) * rstd;
      cols.template store<A>(p.du, row * p.lddu + goff, live, d);
    }
  }
  const int C = p.cg * p.groups;
  auto flush = [&](int which, const float (&v)[NE]) {
    float* out = p.partial[which];
    if (!out) return;
    out += (int64_t)blockIdx.x * C + goff;
    if (slots == 1) {
#pragma unroll
      for (int j = 0; j < NE; j++) if (cols.at(j) < p.cg) out[cols.at(j)] = v[j];
      return;
    }
    block_sync();
#pragma unroll
    for (int j = 0; j < NE; j++) if (cols.at(j) < p.cg) acc[slot * p.cg + cols.at(j)] = v[j];
    block_sync();
    for (int c = threadIdx.x; c < p.cg; c += blockDim.x) {
      float t = 0.f;
      for (int i = 0; i < slots; i++) t += acc[i * p.cg + c];
      out[c] = t;
    }
  };
  flush(0, gw); flush(1, gb); flush(2, gs);
  flush(3, gnw); flush(4, gnb);
}

// The same for rows of more than 4096 channels, where tokens, parameters and sums do not fit in registers together.  A workgroup takes a row at a time in pieces of
// 8 channels a thread, up to three times over (the row is in the cache): the next norm's sums, then everything but du, then du.  Only the column sums and dn w stay
// in registers (beyond 8192 channels not all of them).  Gate, scale, residual and next norm, against the kernel above with 16 channels a thread: 4096 rows of 8192
// fp32: 366 us and 1158 (2.9 TB/s), bf16 219 and 759; 2048 rows of 16384 fp32: 978 and 2831.  Spilled registers bound it beyond 8192 channels (476 - 1236 bytes a lane; up to
// 128 below), and the forward kernel of 16 channels a thread too (20 - 420): forward 8192 fp32 192 us, 3.5 TB/s, bf16 161, 2.1; 16384 fp32 467, 1.4, bf16 307, 1.1.
template <bool VEC> __device__ __forceinline__ void piece_param(const Cols<8, VEC>& cols, const float* p, int off, float fill, bool aligned, float (&v)[8]) {
  if constexpr (VEC) {
    const int c = cols.at(0);
    if (p && aligned) {
      f32x4 a = {}, b = {};
      if (c < cols.n) { a = *reinterpret_cast<const f32x4*>(p + off + c); b = *reinterpret_cast<const f32x4*>(p + off + c + 4); }
#pragma unroll
      for (int k = 0; k < 4; k++) { v[k] = a[k]; v[4 + k] = b[k]; }
      return;
    }
  }
  cols.param(p, off, fill, v);
}
template <typename A, typename R, int NE, bool VEC, bool NEXT> __global__ void __launch_bounds__(512) norm_bwd_wide_kernel(NormP p) {
  __shared__ float red[64];
  const int lane = threadIdx.x, tpr = 512;
  RowSum sum{red, tpr, 0};
  const int g = blockIdx.y, goff = g * p.cg;
  float gw[NE] = {}, gb[NE] = {}, gs[NE] = {}, gnw[NE] = {}, gnb[NE] = {};
  const float inv = 1.0f / p.cg;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float mean = p.stats[(row * p.groups + g) * 2], rstd = p.stats[(row * p.groups + g) * 2 + 1];
    const float nmean = NEXT ? p.nstats[row * 2] : 0.f, nrstd = NEXT ? p.nstats[row * 2 + 1] : 0.f;
    int at = lane;
    auto again = [&]() { asm volatile("" : "+v"(at)); };   // (what a pass reads is read in it: kept from one to the next, or over the rows, it would be spilled)
    // a piece: h and n of u, the gate's factors, and (NEXT) the normalised r and dy * nw
    auto piece = [&](int i, float (&h)[8], float (&n)[8], float (&s)[8], float (&a)[8], float (&da)[8], float (&x)[8], float (&dy)[8], float (&t)[8], float (&w)[8]) {
      const Cols<8, VEC> cols{at + (VEC ? i : 8 * i) * tpr, tpr, p.cg};
      Raw<A, 8> ru, rg, ry;
      Raw<R, 8> rx;
      cols.template load<A>(p.u, row * p.ldu + goff, true, ru);
      if (p.gate) cols.template load<A>(p.gate, row * p.ldg + goff, true, rg);
      if (NEXT) {
        if (p.res) cols.template load<R>(p.res, row * p.ldx + goff, true, rx);
        cols.template load<A>(p.dy, row * p.lddy, true, ry);
      }
      float b[8], nw[8];
      piece_param(cols, p.w, goff, 1.f, p.aligned, w); piece_param(cols, p.b, goff, 0.f, p.aligned, b); piece_param(cols, p.s, goff, 1.f, p.aligned, s);
      if (NEXT) piece_param(cols, p.nw, goff, 1.f, p.aligned, nw);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        h[j] = (ru[j] - mean) * rstd;
        n[j] = __builtin_fmaf(h[j], w[j], b[j]);
        a[j] = 1.f; da[j] = 0.f;
        if (p.gate) {
          const float gt = rg[j];
          float sig;
          a[j] = silu(gt, sig);
          da[j] = sig * (1.0f + gt * (1.0f - sig));
        }
        if (NEXT) {
          const float z = s[j] * n[j] * a[j];
          x[j] = cols.at(j) < p.cg ? ((p.res ? rx[j] + z : z) - nmean) * nrstd : 0.f;
          dy[j] = ry[j]; t[j] = dy[j] * nw[j];
        }
      }
    };
    float h[8], n[8], s[8], a[8], da[8], x[8], dy[8], t[8], w[8];
    float c1 = 0.f, c2 = 0.f;
    if constexpr (NEXT) {
#pragma unroll
      for (int i = 0; i < NE / 8; i++) {
        again();
        piece(i, h, n, s, a, da, x, dy, t, w);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          gnw[8 * i + j] = __builtin_fmaf(dy[j], x[j], gnw[8 * i + j]); gnb[8 * i + j] += dy[j];
          c1 = __builtin_fmaf(t[j], x[j], c1); c2 += t[j];
        }
        __builtin_amdgcn_sched_barrier(0);   // (pieces one after the other: the next ones' reads would take the registers)
      }
      sum(c1, c2);
      c1 *= inv; c2 = p.layer ? c2 * inv : 0.f;
    }
    float e[NE], d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int i = 0; i < NE / 8; i++) {
      again();
      const Cols<8, VEC> cols{at + (VEC ? i : 8 * i) * tpr, tpr, p.cg};
      Raw<R, 8> rr;
      if (p.dr) cols.template load<R>(p.dr, row * p.lddr + goff, true, rr);
      piece(i, h, n, s, a, da, x, dy, t, w);
      float d[8], dg[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        d[j] = p.dr ? rr[j] : 0.f;
        if (NEXT) d[j] += (t[j] - x[j] * c1 - c2) * nrstd;
        if (cols.at(j) >= p.cg) d[j] = 0.f;
        dg[j] = d[j] * s[j] * n[j] * da[j];
        gs[8 * i + j] = __builtin_fmaf(d[j] * a[j], n[j], gs[8 * i + j]);
        const float dn = d[j] * s[j] * a[j];
        gw[8 * i + j] = __builtin_fmaf(dn, h[j], gw[8 * i + j]); gb[8 * i + j] += dn;
        e[8 * i + j] = dn * w[j];
        d1 = __builtin_fmaf(e[8 * i + j], h[j], d1); d2 += e[8 * i + j];
      }
      if (p.dres) cols.template store<R>(p.dres, row * p.lddx + goff, true, d);
      if (p.dgate) cols.template store<A>(p.dgate, row * p.lddg + goff, true, dg);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (p.du) {
      sum(d1, d2);
      d1 *= inv; d2 = p.layer ? d2 * inv : 0.f;
#pragma unroll
      for (int i = 0; i < NE / 8; i++) {
        again();
        const Cols<8, VEC> cols{at + (VEC ? i : 8 * i) * tpr, tpr, p.cg};
        Raw<A, 8> ru;
        cols.template load<A>(p.u, row * p.ldu + goff, true, ru);
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; j++) d[j] = (e[8 * i + j] - (ru[j] - mean) * rstd * d1 - d2) * rstd;
        cols.template store<A>(p.du, row * p.lddu + goff, true, d);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  const int C = p.cg * p.groups;
  auto flush = [&](int which, const float (&v)[NE]) {
    float* out = p.partial[which];
    if (!out) return;
    out += (int64_t)blockIdx.x * C + goff;
#pragma unroll
    for (int j = 0; j < NE; j++) {
      const Cols<8, VEC> cols{lane + (VEC ? j / 8 : j / 8 * 8) * tpr, tpr, p.cg};
      if (cols.at(j & 7) < p.cg) out[cols.at(j & 7)] = v[j];
    }
  };
  flush(0, gw); flush(1, gb); flush(2, gs);
  flush(3, gnw); flush(4, gnb);
}

struct ReduceP { const float* partial[5]; float* out[5]; int blocks, C; };
// 64 columns a workgroup, 16 threads for each: every thread adds a sixteenth of the blocks, then the sixteen are added in order.
__global__ void __launch_bounds__(1024) norm_reduce_kernel(ReduceP p) {
  __shared__ float part[16][64];
  float* out = p.out[blockIdx.y];
  if (!out) return;
  const int lane = threadIdx.x & 63, q = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
  const float* src = p.partial[blockIdx.y];
  float t = 0.f;
  if (c < p.C) {
    int i = q;
    for (; i + 48 < p.blocks; i += 64) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; k++) v[k] = src[(int64_t)(i + 16 * k) * p.C + c];
      t += (v[0] + v[1]) + (v[2] + v[3]);
    }
    for (; i < p.blocks; i += 16) t += src[(int64_t)i * p.C + c];
  }
  part[q][lane] = t;
  block_sync();
  if (q == 0 && c < p.C) {
    t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) t += part[i][lane];
    out[c] = t;
  }
}

struct Plan { int tpr, ne, block, slots; };
// Threads of a row: the smallest power of two (8 .. 1024) that holds it at 8 channels a thread, 16 a thread beyond 8192 channels.
inline Plan make_plan(int cg) {
  Plan q;
  q.tpr = 8; q.ne = 8;
  while (q.tpr * 8 < cg && q.tpr < 1024) q.tpr *= 2;
  if (q.tpr * 8 < cg) q.ne = 16;
  q.block = q.tpr < 256 ? 256 : q.tpr;
  q.slots = q.block / q.tpr;
  return q;
}
// Backward: rows of more than 4096 channels go to the kernel that takes them in pieces (slots and threads are then its own).
inline Plan make_bwd_plan(int cg) {
  if (cg <= 4096) return make_plan(cg);
  return {512, cg <= 8192 ? 16 : 32, 512, 1};
}
// Workgroups for each group of channels; they go round over the rows.
inline int64_t fwd_blocks(int64_t rows, const Plan& q, int groups) {
  const int64_t want = (rows + q.slots - 1) / q.slots, most = (2048 + groups - 1) / groups;
  return want < most ? want : most;
}
inline int64_t bwd_blocks(int64_t rows, const Plan& q, int groups) {
  const int64_t want = (rows + q.slots - 1) / q.slots, most = (512 * 256 / q.block + groups - 1) / groups;
  return want < most ? want : most;
}
bool aligned16(const void* p, int64_t ld, int64_t esize) { return p == nullptr || (((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0); }

template <bool BWD, typename A, typename R, bool NEXT> void launch_next(const NormP& p, const Plan& q, bool vec, dim3 grid, size_t lds, hipStream_t st) {
  if constexpr (BWD) {
#define SF_NORM_GO(NE, V) hipLaunchKernelGGL((norm_bwd_wide_kernel<A, R, NE, V, NEXT>), grid, dim3(512), 0, st, p)
    if (p.cg > 4096) {
      if (q.ne == 16) { if (vec) SF_NORM_GO(16, true); else SF_NORM_GO(16, false); }
      else { if (vec) SF_NORM_GO(32, true); else SF_NORM_GO(32, false); }
      return;
    }
#undef SF_NORM_GO
#define SF_NORM_GO(V, BLOCK) hipLaunchKernelGGL((norm_bwd_kernel<A, R, 8, V, NEXT, BLOCK>), grid, dim3(q.block), lds, st, p)
    if (q.block == 256) { if (vec) SF_NORM_GO(true, 256); else SF_NORM_GO(false, 256); }
    else { if (vec) SF_NORM_GO(true, 512); else SF_NORM_GO(false, 512); }
#undef SF_NORM_GO
  } else {
#define SF_NORM_GO(NE, V, BLOCK) hipLaunchKernelGGL((norm_fwd_kernel<A, R, NE, V, NEXT, BLOCK>), grid, dim3(q.block), 0, st, p)
    if (q.ne == 16) { if (vec) SF_NORM_GO(16, true, 1024); else SF_NORM_GO(16, false, 1024); }
    else if (q.block == 256) { if (vec) SF_NORM_GO(8, true, 256); else SF_NORM_GO(8, false, 256); }
    else if (q.block == 512) { if (vec) SF_NORM_GO(8, true, 512); else SF_NORM_GO(8, false, 512); }
    else { if (vec) SF_NORM_GO(8, true, 1024); else SF_NORM_GO(8, false, 1024); }
  }
#undef SF_NORM_GO
}
template <bool BWD, typename A, typename R> void launch(const NormP& p, const Plan& q, bool vec, dim3 grid, size_t lds, hipStream_t st) {
  if (BWD ? p.dy != nullptr : p.y != nullptr) launch_next<BWD, A, R, true>(p, q, vec, grid, lds, st);
  else launch_next<BWD, A, R, false>(p, q, vec, grid, lds, st);
}

}  // namespace

extern "C" {

static int norm_check(const char* name, const sfRows& u, int64_t rows, int32_t C, int32_t groups, int32_t kind, int32_t dtype, int32_t res_dtype, float eps) {
  SF_REQUIRE(rows >= 0 && C > 0 && groups > 0 && C % groups == 0 && C / groups <= 16384, "%s: rows %lld, C %d in %d groups (at most 16384 channels each)", name,
             (long long)rows, C, groups);
  SF_REQUIRE(groups <= 65535, "%s: %d groups (at most 65535)", name, groups);
  SF_REQUIRE(kind == SF_NORM_RMS || kind == SF_NORM_LAYER, "%s: unknown norm %d", name, kind);
  SF_REQUIRE((dtype == SF_BF16 && (res_dtype == SF_BF16 || res_dtype == SF_F32)) || (dtype == SF_F32 && res_dtype == SF_F32),
             "%s: unsupported storage types %d / %d", name, dtype, res_dtype);
  SF_REQUIRE(rows == 0 || u.ptr != nullptr, "%s: no input", name);
  SF_REQUIRE(eps >= 0.f, "%s: eps %g", name, eps);
  return 0;
}
#define SF_ROWS_OK(t, name, what) SF_REQUIRE((t).ptr == nullptr || (t).ld >= C || rows <= 1, "%s: rows of `%s` overlap (ld %lld < %d)", name, what, (long long)(t).ld, C)

int sf_block_norm_fwd(sfRows u, const float* w, const float* b, sfRows gate, const float* scale, sfRows residual, sfRows r, const float* next_w,
                      const float* next_b, sfRows y, float* stats, float* next_stats, int64_t rows, int32_t C, int32_t groups, int32_t kind, float eps,
                      int32_t dtype, int32_t res_dtype, sfStream stream) {
  const char* name = "sf_block_norm_fwd";
  if (int rc = norm_check(name, u, rows, C, groups, kind, dtype, res_dtype, eps)) return rc;
  if (rows == 0) return 0;
  SF_REQUIRE(r.ptr != nullptr, "%s: no output", name);
  SF_REQUIRE((y.ptr != nullptr) == (next_w != nullptr) && (y.ptr == nullptr || groups == 1), "%s: the next norm takes a weight, an output and one group", name);
  SF_REQUIRE(next_b == nullptr || next_w != nullptr, "%s: next bias without next weight", name);
  SF_ROWS_OK(r, name, "r"); SF_ROWS_OK(y, name, "y");
  const Plan q = make_plan(C / groups);
  const int es = dtype == SF_BF16 ? 2 : 4, rs = res_dtype == SF_BF16 ? 2 : 4;
  const bool vec = (C / groups) % 8 == 0 && aligned16(u.ptr, u.ld, es) && aligned16(gate.ptr, gate.ld, es) && aligned16(residual.ptr, residual.ld, rs) &&
                   aligned16(r.ptr, r.ld, rs) && aligned16(y.ptr, y.ld, es);
  NormP p = {};
  p.u = u.ptr; p.gate = gate.ptr; p.res = residual.ptr; p.w = w; p.b = b; p.s = scale; p.nw = next_w; p.nb = next_b; p.r = r.ptr; p.y = y.ptr;
  p.stats = stats; p.nstats = next_stats; p.ldu = u.ld; p.ldg = gate.ld; p.ldx = residual.ld; p.ldr = r.ld; p.ldy = y.ld; p.rows = rows;
  p.cg = C / groups; p.groups = groups; p.tpr = q.tpr; p.layer = kind == SF_NORM_LAYER; p.eps = eps;
  const dim3 grid((unsigned)fwd_blocks(rows, q, groups), groups);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SF_F32) launch<false, float, float>(p, q, vec, grid, 0, st);
  else if (res_dtype == SF_F32) launch<false, __bf16, float>(p, q, vec, grid, 0, st);
  else launch<false, __bf16, __bf16>(p, q, vec, grid, 0, st);
  SF_CHECK_LAUNCH(name);
  return 0;
}

size_t sf_block_norm_bwd_workspace_floats(int64_t rows, int32_t C, int32_t groups) {
  if (rows <= 0 || C <= 0 || groups <= 0 || C % groups) return 0;
  return (size_t)5 * (size_t)bwd_blocks(rows, make_bwd_plan(C / groups), groups) * (size_t)C;
}

int sf_block_norm_bwd(sfRows u, const float* w, const float* b, sfRows gate, const float* scale, sfRows residual, const float* next_w, const float* stats,
                      const float* next_stats, sfRows dr, sfRows dy, sfRows du, sfRows dgate, sfRows dresidual, float* dw, float* db, float* dscale,
                      float* dnext_w, float* dnext_b, int64_t rows, int32_t C, int32_t groups, int32_t kind, int32_t dtype, int32_t res_dtype,
                      float* workspace, sfStream stream) {
  const char* name = "sf_block_norm_bwd";
  if (int rc = norm_check(name, u, rows, C, groups, kind, dtype, res_dtype, 0.f)) return rc;
  SF_REQUIRE(rows > 0, "%s: no rows", name);
  SF_REQUIRE(stats != nullptr && workspace != nullptr, "%s: no statistics or workspace", name);
  SF_REQUIRE(dr.ptr != nullptr || dy.ptr != nullptr, "%s: no output gradient", name);
  SF_REQUIRE(dy.ptr == nullptr || (next_w != nullptr && next_stats != nullptr && groups == 1), "%s: a gradient of y without the next norm", name);
  SF_REQUIRE(dgate.ptr == nullptr || gate.ptr != nullptr, "%s: a gate gradient without a gate", name);
  SF_REQUIRE(dresidual.ptr == nullptr || residual.ptr != nullptr, "%s: a residual gradient without a residual", name);
  SF_ROWS_OK(du, name, "du"); SF_ROWS_OK(dgate, name, "dgate"); SF_ROWS_OK(dresidual, name, "dresidual");
  const Plan q = make_bwd_plan(C / groups);
  const int es = dtype == SF_BF16 ? 2 : 4, rs = res_dtype == SF_BF16 ? 2 : 4;
  const bool vec = (C / groups) % 8 == 0 && aligned16(u.ptr, u.ld, es) && aligned16(gate.ptr, gate.ld, es) && aligned16(residual.ptr, residual.ld, rs) &&
                   aligned16(dr.ptr, dr.ld, rs) && aligned16(dy.ptr, dy.ld, es) && aligned16(du.ptr, du.ld, es) && aligned16(dgate.ptr, dgate.ld, es) &&
                   aligned16(dresidual.ptr, dresidual.ld, rs);
  NormP p = {};
  p.u = u.ptr; p.gate = gate.ptr; p.res = residual.ptr; p.w = w; p.b = b; p.s = scale; p.nw = next_w;
  p.stats = const_cast<float*>(stats); p.nstats = const_cast<float*>(next_stats);
  p.ldu = u.ld; p.ldg = gate.ld; p.ldx = residual.ld; p.rows = rows; p.cg = C / groups; p.groups = groups; p.tpr = q.tpr; p.layer = kind == SF_NORM_LAYER;
  p.dr = dr.ptr; p.dy = dy.ptr; p.du = du.ptr; p.dgate = dgate.ptr; p.dres = dresidual.ptr;
  p.lddr = dr.ld; p.lddy = dy.ld; p.lddu = du.ld; p.lddg = dgate.ld; p.lddx = dresidual.ld;
  p.aligned = (((uintptr_t)w | (uintptr_t)b | (uintptr_t)scale | (uintptr_t)next_w) & 15) == 0;
  const int blocks = (int)bwd_blocks(rows, q, groups);
  ReduceP red = {{}, {dw, db, dscale, dnext_w, dnext_b}, blocks, C};
  for (int i = 0; i < 5; i++)
    if (red.out[i]) red.partial[i] = p.partial[i] = workspace + (int64_t)i * blocks * C;
  const dim3 grid(blocks, groups);
  const size_t lds = (64 + (q.slots > 1 ? (size_t)q.slots * (C / groups) : 0)) * sizeof(float)   /* at most 8.25 KB: slots * C / groups <= 2048 */;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SF_F32) launch<true, float, float>(p, q, vec, grid, lds, st);
  else if (res_dtype == SF_F32) launch<true, __bf16, float>(p, q, vec, grid, lds, st);
  else launch<true, __bf16, __bf16>(p, q, vec, grid, lds, st);
  SF_CHECK_LAUNCH(name);
  if (dw || db || dscale || dnext_w || dnext_b) {
    hipLaunchKernelGGL(norm_reduce_kernel, dim3((C + 63) / 64, 5), dim3(1024), 0, st, red);
    SF_CHECK_LAUNCH(name);
  }
  return 0;
}

}  // extern "C"
