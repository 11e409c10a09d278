// Linear attention with a decay for each head (see include/satflow_hip.h):  S_t = lambda S_{t-1} + k_t v_t^T ,  o_t = scale * S_t^T q_t.
//
// One sweep kernel serves the forward pass and the three gradients.  With R_t = lambda R_{t+1} + scale q_t do_t^T (R behind the last token: the gradient of
// the state that left), the adjoint is
//   dq_t = scale S_t do_t ,   dk_t = R_t v_t ,   dv_t = R_t^T k_t ,   dS_in = lambda R_0
// so that dq is the sweep on (do, v, k) - state S^T -, dk the sweep in reverse on (v, do, q) - state R^T - and dv the sweep in reverse on (k, q, do).  The
// reverse sweeps take their initial state at the first token without a decay (`plain_init`) and give lambda times their last one (`decay_out`).
#include "sf_common.h"

namespace {

struct Sweep {
  sfSeq q, k, v, o;               // read by q, written k (x) v
  const float* g;
  const float* s_in; int64_t in_d, in_e;   // element strides of the state's two axes (dk, dv of THIS sweep)
  float* s_out;                   // dense, strides out_d / out_e
  int64_t out_d, out_e;
  const int32_t* lengths;
  int B, T, H, dk, dv;
  float kscale, oscale;           // applied to k v^T and to the output
  int reverse, plain_init, decay_out;
};

__device__ __forceinline__ void la_sync() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

// Token by token: a workgroup owns 64 columns of one sequence and head's state, thread (r, e) the rows r, r + 4, ... of column e in registers.
constexpr int TOK = 16;
template <typename T> __global__ void __launch_bounds__(256) la_recurrent_kernel(Sweep p) {
  __shared__ float sq[TOK][128], sk[TOK][128], sv[TOK][64], part[4][TOK][64];
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, e0 = blockIdx.y * 64;
  const int el = threadIdx.x & 63, r = threadIdx.x >> 6, e = e0 + el;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  // lambda in two floats: rounded to one, its error grows with the distance (2^-25 a token, 10^-4 over 5000)
  const double lam2 = exp((double)p.g[h]);
  const float lam = (float)lam2, lam_lo = (float)(lam2 - (double)lam);
  const T* q = (const T*)p.q.ptr + b * p.q.sb + h * p.q.sh;
  const T* k = (const T*)p.k.ptr + b * p.k.sb + h * p.k.sh;
  const T* v = (const T*)p.v.ptr + b * p.v.sb + h * p.v.sh;
  T* o = (T*)p.o.ptr + b * p.o.sb + h * p.o.sh;
  float s[32];
#pragma unroll
  for (int m = 0; m < 32; m++) {
    const int d = r + 4 * m;
    s[m] = p.s_in && d < p.dk && e < p.dv ? p.s_in[(int64_t)bh * p.dk * p.dv + d * p.in_d + e * p.in_e] : 0.f;
  }
  for (int c0 = 0; c0 < p.T; c0 += TOK) {
    la_sync();
    for (int i = threadIdx.x; i < TOK * 128; i += 256) {
      const int tk = i >> 7, d = i & 127, pos = c0 + tk;
      const int64_t t = p.reverse ? len - 1 - pos : pos;
      const bool live = pos < len && d < p.dk;
      sq[tk][d] = live ? (float)q[t * p.q.st + d] : 0.f;
      sk[tk][d] = live ? (float)k[t * p.k.st + d] * p.kscale : 0.f;
    }
    for (int i = threadIdx.x; i < TOK * 64; i += 256) {
      const int tk = i >> 6, c = e0 + (i & 63), pos = c0 + tk;
      const int64_t t = p.reverse ? len - 1 - pos : pos;
      sv[tk][i & 63] = pos < len && c < p.dv ? (float)v[t * p.v.st + c] : 0.f;
    }
    la_sync();
    for (int tk = 0; tk < TOK; tk++) {
      float acc = 0.f;
      if (c0 + tk < len) {
        const bool plain = c0 + tk == 0 && p.plain_init;
        const float l = plain ? 1.f : lam, ll = plain ? 0.f : lam_lo, ve = sv[tk][el];
#pragma unroll
        for (int m = 0; m < 32; m++) {
          if (r + 4 * m >= p.dk) break;   // (a zero row times an infinite value would be NaN)
          s[m] = __builtin_fmaf(l, s[m], __builtin_fmaf(ll, s[m], sk[tk][r + 4 * m] * ve));
          acc = __builtin_fmaf(sq[tk][r + 4 * m], s[m], acc);
        }
      }
      part[r][tk][el] = acc;
    }
    la_sync();
    for (int i = threadIdx.x; i < TOK * 64; i += 256) {
      const int tk = i >> 6, c = e0 + (i & 63), pos = c0 + tk;
      if (pos >= p.T || c >= p.dv) continue;
      const int64_t t = p.reverse && pos < len ? len - 1 - pos : pos;
      o[t * p.o.st + c] = (T)((part[0][tk][i & 63] + part[1][tk][i & 63] + part[2][tk][i & 63] + part[3][tk][i & 63]) * p.oscale);
    }
  }
  if (p.s_out && e < p.dv) {
    const float l = p.decay_out && len > 0 ? lam : 1.f;
#pragma unroll
    for (int m = 0; m < 32; m++) {
      const int d = r + 4 * m;
      if (d < p.dk) p.s_out[(int64_t)bh * p.dk * p.dv + d * p.out_d + e * p.out_e] = s[m] * l;
    }
  }
}

// One token: the state is read and written once.  A workgroup owns `tile` columns of one sequence and head; thread (r, c) the rows r, r + rows, ... of
// VEC neighbouring columns.
template <typename T, int VEC> __global__ void __launch_bounds__(256) la_step_kernel(Sweep p, int tile) {
  __shared__ float sq[128], sk[128], part[16][128];
  const int bh = blockIdx.x, b = bh / p.H, h = bh % p.H, e0 = blockIdx.y * tile;
  const int across = tile / VEC, rows = 256 / across, r = threadIdx.x / across, el = (threadIdx.x % across) * VEC, e = e0 + el;
  const float lam = expf(p.g[h]);
  const T* q = (const T*)p.q.ptr + b * p.q.sb + h * p.q.sh;
  const T* k = (const T*)p.k.ptr + b * p.k.sb + h * p.k.sh;
  const T* v = (const T*)p.v.ptr + b * p.v.sb + h * p.v.sh;
  if ((int)threadIdx.x < p.dk) { sq[threadIdx.x] = (float)q[threadIdx.x]; sk[threadIdx.x] = (float)k[threadIdx.x]; }
  float ve[VEC], acc[VEC] = {};
#pragma unroll
  for (int j = 0; j < VEC; j++) ve[j] = e + j < p.dv ? (float)v[e + j] : 0.f;
  la_sync();
  const float* in = p.s_in + (int64_t)bh * p.dk * p.dv;
  float* out = p.s_out + (int64_t)bh * p.dk * p.dv;
  if (e < p.dv) {
    for (int d = r; d < p.dk; d += rows) {
      float s[VEC];
      if constexpr (VEC == 4) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(in + (int64_t)d * p.dv + e);
#pragma unroll
        for (int j = 0; j < 4; j++) s[j] = x[j];
      } else s[0] = in[(int64_t)d * p.dv + e];
#pragma unroll
      for (int j = 0; j < VEC; j++) {
        s[j] = __builtin_fmaf(lam, s[j], sk[d] * ve[j]);
        acc[j] = __builtin_fmaf(sq[d], s[j], acc[j]);
      }
      if constexpr (VEC == 4) *reinterpret_cast<f32x4*>(out + (int64_t)d * p.dv + e) = f32x4{s[0], s[1], s[2], s[3]};
      else out[(int64_t)d * p.dv + e] = s[0];
    }
  }
  // rows of a wave first (their lanes are `across` apart), then the waves
  for (int m = across; m < 64; m <<= 1)
#pragma unroll
    for (int j = 0; j < VEC; j++) acc[j] += __shfl_xor(acc[j], m);
  const int wave = threadIdx.x >> 6;
  const int groups = across < 64 ? 4 : rows;      // rows of partial sums
  const int slot = across < 64 ? wave : r;
  if (across >= 64 || (int)(threadIdx.x & 63) < across)
#pragma unroll
    for (int j = 0; j < VEC; j++) part[slot][el + j] = acc[j];
  la_sync();
  if ((int)threadIdx.x < tile && e0 + (int)threadIdx.x < p.dv) {
    float t = 0.f;
    for (int i = 0; i < groups; i++) t += part[i][threadIdx.x];
    ((T*)p.o.ptr + b * p.o.sb + h * p.o.sh)[e0 + threadIdx.x] = (T)(t * p.oscale);
  }
}

template <typename F> int by_dtype(int dtype, F f) { return dtype == SF_BF16 ? f((__bf16*)nullptr) : f((float*)nullptr); }

int run_sweep(const Sweep& p, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)(p.B * p.H), (p.dv + 63) / 64);
  if (dtype == SF_BF16) hipLaunchKernelGGL(la_recurrent_kernel<__bf16>, grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL(la_recurrent_kernel<float>, grid, dim3(256), 0, st, p);
  SF_CHECK_LAUNCH("sf_linear_attention");
  return 0;
}

int check_dims(const char* name, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, int32_t dtype) {
  SF_REQUIRE(B >= 0 && T >= 0 && H > 0, "%s: B %d, T %d, H %d", name, B, T, H);
  SF_REQUIRE(dk >= 1 && dk <= 128 && dv >= 1 && dv <= 128, "%s: head widths %d / %d (1 .. 128)", name, dk, dv);
  SF_REQUIRE(dtype == SF_F32 || dtype == SF_BF16, "%s: unsupported storage type %d", name, dtype);
  SF_REQUIRE((int64_t)B * H <= 0x7fffffff, "%s: B * H is too large", name);
  return 0;
}

}  // namespace

extern "C" {

size_t sf_linear_attention_workspace_bytes(int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, int32_t dtype, int32_t backward) {
  (void)B; (void)T; (void)H; (void)dk; (void)dv; (void)dtype; (void)backward;
  return 0;
}

int sf_linear_attention_fwd(sfSeq q, sfSeq k, sfSeq v, sfSeq o, const float* log_decay, const float* s_in, float* s_out, const int32_t* lengths, int32_t B,
                            int32_t T, int32_t H, int32_t dk, int32_t dv, float scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                            sfStream stream) {
  const char* name = "sf_linear_attention_fwd";
  if (int rc = check_dims(name, B, T, H, dk, dv, dtype)) return rc;
  SF_REQUIRE(log_decay != nullptr && (T == 0 || B == 0 || (q.ptr && k.ptr && v.ptr && o.ptr)), "%s: missing tensor", name);
  SF_REQUIRE(workspace_bytes >= sf_linear_attention_workspace_bytes(B, T, H, dk, dv, dtype, 0), "%s: workspace too small", name);
  if (B == 0) return 0;
  Sweep p = {};
  p.q = q; p.k = k; p.v = v; p.o = o; p.g = log_decay; p.s_in = s_in; p.in_d = dv; p.in_e = 1; p.s_out = s_out; p.out_d = dv; p.out_e = 1;
  p.lengths = lengths; p.B = B; p.T = T; p.H = H; p.dk = dk; p.dv = dv; p.kscale = 1.f; p.oscale = scale;
  return run_sweep(p, dtype, (hipStream_t)stream);
}

int sf_linear_attention_bwd(sfSeq q, sfSeq k, sfSeq v, sfSeq dout, const float* log_decay, const float* s_in, const float* ds_out, const int32_t* lengths,
                            sfSeq dq, sfSeq dk_out, sfSeq dv_out, float* ds_in, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, float scale,
                            int32_t dtype, void* workspace, size_t workspace_bytes, sfStream stream) {
  const char* name = "sf_linear_attention_bwd";
  if (int rc = check_dims(name, B, T, H, dk, dv, dtype)) return rc;
  SF_REQUIRE(log_decay != nullptr && (T == 0 || B == 0 || (q.ptr && k.ptr && v.ptr && dout.ptr && dq.ptr && dk_out.ptr && dv_out.ptr)), "%s: missing tensor", name);
  SF_REQUIRE(workspace_bytes >= sf_linear_attention_workspace_bytes(B, T, H, dk, dv, dtype, 1), "%s: workspace too small", name);
  if (B == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  Sweep p = {};
  p.g = log_decay; p.lengths = lengths; p.B = B; p.T = T; p.H = H;
  // dq: state S^T, read by do, written v (x) k
  p.q = dout; p.k = v; p.v = k; p.o = dq; p.dk = dv; p.dv = dk; p.s_in = s_in; p.in_d = 1; p.in_e = dv; p.kscale = 1.f; p.oscale = scale;
  if (int rc = run_sweep(p, dtype, st)) return rc;
  // dk: state R^T, read by v, written do (x) q
  p.reverse = 1; p.plain_init = 1;
  p.q = v; p.k = dout; p.v = q; p.o = dk_out; p.s_in = ds_out; p.kscale = scale; p.oscale = 1.f;
  if (int rc = run_sweep(p, dtype, st)) return rc;
  // dv: state R, read by k, written q (x) do; lambda times its last state is the gradient of s_in
  p.q = k; p.k = q; p.v = dout; p.o = dv_out; p.dk = dk; p.dv = dv; p.in_d = dv; p.in_e = 1; p.s_out = ds_in; p.out_d = dv; p.out_e = 1; p.decay_out = 1;
  return run_sweep(p, dtype, st);
}

int sf_linear_attention_step(sfSeq q, sfSeq k, sfSeq v, sfSeq o, const float* log_decay, const float* s_in, float* s_out, int32_t B, int32_t H, int32_t dk,
                             int32_t dv, float scale, int32_t dtype, sfStream stream) {
  const char* name = "sf_linear_attention_step";
  if (int rc = check_dims(name, B, 1, H, dk, dv, dtype)) return rc;
  SF_REQUIRE(B == 0 || (log_decay && q.ptr && k.ptr && v.ptr && o.ptr && s_in && s_out), "%s: missing tensor", name);
  if (B == 0) return 0;
  Sweep p = {};
  p.q = q; p.k = k; p.v = v; p.o = o; p.g = log_decay; p.s_in = s_in; p.s_out = s_out; p.B = B; p.T = 1; p.H = H; p.dk = dk; p.dv = dv; p.oscale = scale;
  hipStream_t st = (hipStream_t)stream;
  const bool vec = dv % 4 == 0 && (((uintptr_t)s_in | (uintptr_t)s_out) & 15) == 0;
  const int tile = 64;
  const dim3 grid((unsigned)(B * H), (dv + tile - 1) / tile);
#define SF_LA_STEP(T)                                                                                       \
  do {                                                                                                      \
    if (vec) hipLaunchKernelGGL((la_step_kernel<T, 4>), grid, dim3(256), 0, st, p, tile);                   \
    else hipLaunchKernelGGL((la_step_kernel<T, 1>), grid, dim3(256), 0, st, p, tile);                       \
  } while (0)
  if (dtype == SF_BF16) SF_LA_STEP(__bf16); else SF_LA_STEP(float);
#undef SF_LA_STEP
  SF_CHECK_LAUNCH(name);
  return 0;
}

}  // extern "C"
