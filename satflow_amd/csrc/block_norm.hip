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
  float* partial;          // [5][gridDim.x][C]: dw, db, ds, dnw, dnb
};

// LDS writes are waited for explicitly in front of a barrier: the compiler may drop that wait from __syncthreads().
__device__ __forceinline__ void block_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

// Sums of two values over the `tpr` threads that hold a row.  red: 2 x 2 x 16 floats, the halves used in turn, so that one barrier per call is enough
// (a wave can be at most one call behind another).
struct RowSum {
  float* red;
  int tpr, phase;
  __device__ __forceinline__ void operator()(float& a, float& b) {
    const int w = tpr < 64 ? tpr : 64;
    for (int o = w >> 1; o; o >>= 1) { a += __shfl_xor(a, o); b += __shfl_xor(b, o); }
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

// The NE elements of a thread: vectors of 8 channels when VEC (rows 16-byte aligned, C / groups a multiple of 8), single channels tpr apart otherwise.
template <int NE, bool VEC> struct Cols {
  int lane, tpr, n;
  __device__ __forceinline__ int at(int j) const { return VEC ? (lane + (j >> 3) * tpr) * 8 + (j & 7) : lane + j * tpr; }
  template <typename T> __device__ __forceinline__ void load(const void* base, int64_t off, bool live, float (&v)[NE]) const {
    const T* p = (const T*)base + off;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < NE / 8; i++) {
        const int c = (lane + i * tpr) * 8;
        f32x8_t x = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (live && c < n) x = ldv8<T>(p + c);
#pragma unroll
        for (int k = 0; k < 8; k++) v[8 * i + k] = x[k];
      }
    } else {
#pragma unroll
      for (int j = 0; j < NE; j++) {
        const int c = at(j);
        v[j] = live && c < n ? (float)p[c] : 0.f;
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

template <typename A, typename R, int NE, bool VEC> __global__ void __launch_bounds__(1024) norm_fwd_kernel(NormP p) {
  __shared__ float red[64];
  const int slots = blockDim.x / p.tpr, slot = threadIdx.x / p.tpr;
  Cols<NE, VEC> cols{(int)(threadIdx.x % p.tpr), p.tpr, p.cg};
  RowSum sum{red, p.tpr, 0};
  const int g = blockIdx.y, goff = g * p.cg;
  float w[NE], b[NE], s[NE], nw[NE], nb[NE];
  cols.param(p.w, goff, 1.f, w); cols.param(p.b, goff, 0.f, b); cols.param(p.s, goff, 1.f, s);
  cols.param(p.nw, goff, 0.f, nw); cols.param(p.nb, goff, 0.f, nb);
  for (int64_t base = (int64_t)blockIdx.x * slots; base < p.rows; base += (int64_t)gridDim.x * slots) {
    const int64_t row = base + slot;
    const bool live = row < p.rows;
    float u[NE], x[NE];
    cols.template load<A>(p.u, row * p.ldu + goff, live, u);
    float gt[NE];
    if (p.gate) cols.template load<A>(p.gate, row * p.ldg + goff, live, gt);
    if (p.res) cols.template load<R>(p.res, row * p.ldx + goff, live, x);
    float mean, rstd;
    row_stats(cols, sum, u, p.cg, p.layer, p.eps, mean, rstd);
    if (p.stats && live && cols.lane == 0) { float* st = p.stats + (row * p.groups + g) * 2; st[0] = mean; st[1] = rstd; }
#pragma unroll
    for (int j = 0; j < NE; j++) {
      float z = s[j] * __builtin_fmaf((u[j] - mean) * rstd, w[j], b[j]), sig;
      if (p.gate) z *= silu(gt[j], sig);
      u[j] = p.res ? x[j] + z : z;
      if (cols.at(j) >= p.cg) u[j] = 0.f;
    }
    cols.template store<R>(p.r, row * p.ldr + goff, live, u);
    if (p.y) {
      row_stats(cols, sum, u, p.cg, p.layer, p.eps, mean, rstd);
      if (p.nstats && live && cols.lane == 0) { p.nstats[row * 2] = mean; p.nstats[row * 2 + 1] = rstd; }
#pragma unroll
      for (int j = 0; j < NE; j++) u[j] = __builtin_fmaf((u[j] - mean) * rstd, nw[j], nb[j]);
      cols.template store<A>(p.y, row * p.ldy, live, u);
    }
  }
}

// Column sums: a thread keeps the five sums of its columns in registers over the rows of its slot; the block's slots are added through LDS, the blocks by
// norm_reduce_kernel in block order (no atomics: the result does not depend on timing).
template <typename A, typename R, int NE, bool VEC> __global__ void __launch_bounds__(1024) norm_bwd_kernel(NormP p) {
  extern __shared__ float lds[];
  float* red = lds;            // 64 floats
  float* acc = lds + 64;       // [slots][cg] (slots > 1)
  const int slots = blockDim.x / p.tpr, slot = threadIdx.x / p.tpr;
  Cols<NE, VEC> cols{(int)(threadIdx.x % p.tpr), p.tpr, p.cg};
  RowSum sum{red, p.tpr, 0};
  const int g = blockIdx.y, goff = g * p.cg;
  float w[NE], b[NE], s[NE], nw[NE];
  cols.param(p.w, goff, 1.f, w); cols.param(p.b, goff, 0.f, b); cols.param(p.s, goff, 1.f, s); cols.param(p.nw, goff, 1.f, nw);
  float gw[NE] = {}, gb[NE] = {}, gs[NE] = {}, gnw[NE] = {}, gnb[NE] = {};
  const float inv = 1.0f / p.cg;
  for (int64_t base = (int64_t)blockIdx.x * slots; base < p.rows; base += (int64_t)gridDim.x * slots) {
    const int64_t row = base + slot;
    const bool live = row < p.rows;
    float u[NE], gt[NE], x[NE], d[NE], dy[NE];
    cols.template load<A>(p.u, row * p.ldu + goff, live, u);
    if (p.gate) cols.template load<A>(p.gate, row * p.ldg + goff, live, gt);
    if (p.res && p.dy) cols.template load<R>(p.res, row * p.ldx + goff, live, x);
    if (p.dr) cols.template load<R>(p.dr, row * p.lddr + goff, live, d);
    if (p.dy) cols.template load<A>(p.dy, row * p.lddy, live, dy);
    float mean = 0.f, rstd = 0.f, nmean = 0.f, nrstd = 0.f;
    if (live) {
      const float* st = p.stats + (row * p.groups + g) * 2;
      mean = st[0]; rstd = st[1];
      if (p.dy) { nmean = p.nstats[row * 2]; nrstd = p.nstats[row * 2 + 1]; }
    }
    float c1 = 0.f, c2 = 0.f;
    if (p.dy) {
#pragma unroll
      for (int j = 0; j < NE; j++) {   // x becomes the normalised r
        float z = s[j] * __builtin_fmaf((u[j] - mean) * rstd, w[j], b[j]), sig;
        if (p.gate) z *= silu(gt[j], sig);
        x[j] = ((p.res ? x[j] + z : z) - nmean) * nrstd;
        if (cols.at(j) >= p.cg) x[j] = 0.f;
        const float t = dy[j] * nw[j];
        gnw[j] = __builtin_fmaf(dy[j], x[j], gnw[j]); gnb[j] += dy[j];
        c1 = __builtin_fmaf(t, x[j], c1); c2 += t;
      }
      sum(c1, c2);
      c1 *= inv; c2 = p.layer ? c2 * inv : 0.f;
#pragma unroll
      for (int j = 0; j < NE; j++) {
        const float t = (dy[j] * nw[j] - x[j] * c1 - c2) * nrstd;
        d[j] = p.dr ? d[j] + t : t;
      }
    }
    if (p.dres) cols.template store<R>(p.dres, row * p.lddx + goff, live, d);
    c1 = 0.f; c2 = 0.f;
#pragma unroll
    for (int j = 0; j < NE; j++) {
      if (cols.at(j) >= p.cg) d[j] = 0.f;
      const float h = (u[j] - mean) * rstd, n = __builtin_fmaf(h, w[j], b[j]);
      float sig = 0.f, a = 1.f;
      if (p.gate) {
        a = silu(gt[j], sig);
        gt[j] = d[j] * s[j] * n * (sig * (1.0f + gt[j] * (1.0f - sig)));
      }
      gs[j] = __builtin_fmaf(d[j] * a, n, gs[j]);
      const float dn = d[j] * s[j] * a;
      gw[j] = __builtin_fmaf(dn, h, gw[j]); gb[j] += dn;
      d[j] = dn * w[j];
      c1 = __builtin_fmaf(d[j], h, c1); c2 += d[j];
    }
    if (p.dgate) cols.template store<A>(p.dgate, row * p.lddg + goff, live, gt);
    sum(c1, c2);
    c1 *= inv; c2 = p.layer ? c2 * inv : 0.f;
#pragma unroll
    for (int j = 0; j < NE; j++) d[j] = (d[j] - (u[j] - mean) * rstd * c1 - c2) * rstd;
    if (p.du) cols.template store<A>(p.du, row * p.lddu + goff, live, d);
  }
  const int C = p.cg * p.groups;
  auto flush = [&](int which, const float (&v)[NE]) {
    float* out = p.partial + ((int64_t)which * gridDim.x + blockIdx.x) * C + goff;
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
  flush(0, gw); flush(1, gb); flush(2, gs); flush(3, gnw); flush(4, gnb);
}

__global__ void __launch_bounds__(256) norm_reduce_kernel(const float* partial, int blocks, int C, float* dw, float* db, float* ds, float* dnw, float* dnb) {
  __shared__ float part[4][64];
  float* outs[5] = {dw, db, ds, dnw, dnb};
  float* out = outs[blockIdx.y];
  if (!out) return;
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
  const float* src = partial + (int64_t)blockIdx.y * blocks * C;
  float t = 0.f;
  if (c < C) for (int i = q; i < blocks; i += 4) t += src[(int64_t)i * C + c];
  part[q][threadIdx.x & 63] = t;
  block_sync();
  if (q == 0 && c < C) out[c] = (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
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
inline int64_t fwd_blocks(int64_t rows, const Plan& q) {
  const int64_t want = (rows + q.slots - 1) / q.slots;
  return want < 2048 ? want : 2048;
}
inline int64_t bwd_blocks(int64_t rows, const Plan& q) {
  const int64_t want = (rows + q.slots - 1) / q.slots;
  return want < 512 ? want : 512;
}
bool aligned16(const void* p, int64_t ld, int64_t esize) { return p == nullptr || (((uintptr_t)p & 15) == 0 && (ld * esize) % 16 == 0); }

template <bool BWD, typename A, typename R> void launch(const NormP& p, const Plan& q, bool vec, dim3 grid, size_t lds, hipStream_t st) {
#define SF_NORM_GO(NE, V)                                                                             \
  do {                                                                                                \
    if (BWD) hipLaunchKernelGGL((norm_bwd_kernel<A, R, NE, V>), grid, dim3(q.block), lds, st, p);     \
    else hipLaunchKernelGGL((norm_fwd_kernel<A, R, NE, V>), grid, dim3(q.block), 0, st, p);           \
  } while (0)
  if (q.ne == 8) { if (vec) SF_NORM_GO(8, true); else SF_NORM_GO(8, false); }
  else { if (vec) SF_NORM_GO(16, true); else SF_NORM_GO(16, false); }
#undef SF_NORM_GO
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
  const dim3 grid((unsigned)fwd_blocks(rows, q), groups);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SF_F32) launch<false, float, float>(p, q, vec, grid, 0, st);
  else if (res_dtype == SF_F32) launch<false, __bf16, float>(p, q, vec, grid, 0, st);
  else launch<false, __bf16, __bf16>(p, q, vec, grid, 0, st);
  SF_CHECK_LAUNCH(name);
  return 0;
}

size_t sf_block_norm_bwd_workspace_floats(int64_t rows, int32_t C, int32_t groups) {
  if (rows <= 0 || C <= 0 || groups <= 0 || C % groups) return 0;
  return (size_t)5 * (size_t)bwd_blocks(rows, make_plan(C / groups)) * (size_t)C;
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
  const Plan q = make_plan(C / groups);
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
  p.partial = workspace;
  const int blocks = (int)bwd_blocks(rows, q);
  const dim3 grid(blocks, groups);
  const size_t lds = (64 + (q.slots > 1 ? (size_t)q.slots * (C / groups) : 0)) * sizeof(float)   /* at most 8.25 KB: slots * C / groups <= 2048 */;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == SF_F32) launch<true, float, float>(p, q, vec, grid, lds, st);
  else if (res_dtype == SF_F32) launch<true, __bf16, float>(p, q, vec, grid, lds, st);
  else launch<true, __bf16, __bf16>(p, q, vec, grid, lds, st);
  SF_CHECK_LAUNCH(name);
  if (dw || db || dscale || dnext_w || dnext_b) {
    hipLaunchKernelGGL(norm_reduce_kernel, dim3((C + 63) / 64, 5), dim3(256), 0, st, workspace, blocks, C, dw, db, dscale, dnext_w, dnext_b);
    SF_CHECK_LAUNCH(name);
  }
  return 0;
}

}  // extern "C"
