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
  const float* s_in; int in_d, in_e;   // element strides of the state's two axes (dk, dv of THIS sweep)
  float* s_out;                   // the same strides
  const int32_t* lengths;
  int B, T, H, dk, dv;
  float kscale, oscale;           // applied to k v^T and to the output
  int reverse, plain_init, decay_out;
  // chunked form: the sequence in nseg segments of seg_tokens (a multiple of the chunk).  seg [B * H][nseg] matrices with the strides of s_in: what
  // segment s leaves of a zero state or - joined - the state behind it.
  float* seg;
  int nseg, seg_tokens, joined;
};
// Up to three sweeps of one launch (the gradients): workgroup 8 (g n + r) + x works for sweep r on piece 8 g + x of the sequences, so that the sweeps that read
// the same tokens run side by side on the same die (workgroups go round the eight dies).
struct Sweeps { Sweep s[3]; int n; };

// A barrier for LDS alone: its writes are waited for, reads and writes of memory in flight are not (__syncthreads() waits for those too, the next chunk's
// tokens among them).
__device__ __forceinline__ void la_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// In front of the chunk loop: with nothing in flight there, the wait for the reads at the top of the loop is counted past the writes behind them (vmcnt 0 alone).
__device__ __forceinline__ void la_arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// ---- chunked form ---------------------------------------------------------------------------------------------------------------------------
// A workgroup walks the chunks of C tokens of one (sequence, head, segment); wave w owns value columns 32 w .. 32 w + 31 and holds that part of the state,
// S[d][e], in MFMA accumulators (lane = column e, registers = rows d).  With D_ij = lambda^(i-j) for i >= j, 0 otherwise:
//   P = (Q K^T) o D ,   O = P V + lambda^(i+1) Q S ,   S' = lambda^C S + sum_j k_j (lambda^(C-1-j) v_j)^T
// All three products of a chunk run transposed, so that no value crosses lanes: P^T comes out of K Q^T with lane = token i and registers = tokens j in the
// order {4h, .., 4h + 3, 8 + 4h, ..} (h = lane / 32) of each block of 16, which is the K order of the next product's operand P^T; the matching operand V^T
// is read from the row-major tile by the transposing LDS read in that order.  The state's registers hold rows d in the same order, so S converts in
// place to the operand of Q S, against rows of Q read in that order (two 8-byte reads).  v_j lambda^(C-1-j) reuses the fragments of V^T.
// Precision: operands are sums of bf16 parts (8 bits each) multiplied part by part, fp32 accumulation: bf16 tensors have one part, fp32 ones three (exact);
// the inner operands have two parts where they feed bf16 outputs (P, S: 2^-17, well below the output's rounding; one part, 2^-9 each, would make the error 1.7 times
// that of the one rounding that the output's type asks for) and three where they feed fp32 ones.  The state itself stays fp32; the weighted values added to it have three
// parts where it leaves in fp32 (or goes to a segment's slot), two where only bf16 outputs read it.  Products of parts below 2^-24 are left out.
typedef __bf16 la_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 la_bf16x4 __attribute__((ext_vector_type(4)));

// x as a sum of N bf16 parts, each the rest rounded to nearest (exact for N = 3).  PAIRED: the rest of a pair by dot products with (-1, 0) and (0, -1), one
// instruction instead of two for each value, as exact (the rest is representable) - but a value that is not finite makes its neighbour NaN: for operands whose pairs
// meet in every sum they enter.
template <int N, bool PAIRED = false> __device__ __forceinline__ void split(const f32x8_t& x, la_bf16x8 (&p)[N]) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  unsigned first = 0xbf80u, second = 0xbf800000u;
  if constexpr (PAIRED) asm("" : "+s"(first), "+s"(second));   // (from registers: as a literal the first one is taken for -1.0 in 32 bits, that is the second)
#pragma unroll
  for (int k = 0; k < 4; k++) {
    float a = x[2 * k], b = x[2 * k + 1];
#pragma unroll
    for (int i = 0; i < N; i++) {
      const bf16x2 v = __builtin_convertvector(f32x2{a, b}, bf16x2);
      const unsigned w = __builtin_bit_cast(unsigned, v);
      u4 u = __builtin_bit_cast(u4, p[i]);
      u[k] = w;
      p[i] = __builtin_bit_cast(la_bf16x8, u);
      if (i + 1 < N) {
        if constexpr (PAIRED) {
          a = __builtin_amdgcn_fdot2_f32_bf16(v, __builtin_bit_cast(bf16x2, first), a, false);
          b = __builtin_amdgcn_fdot2_f32_bf16(v, __builtin_bit_cast(bf16x2, second), b, false);
        } else { a -= __builtin_bit_cast(float, w << 16); b -= __builtin_bit_cast(float, w & 0xffff0000u); }
      }
    }
  }
}
// sum of the products of parts, the small ones first; parts whose product falls below 2^-24 are left out
template <int NA, int NB> __device__ __forceinline__ f32x16 mm(const la_bf16x8 (&a)[NA], const la_bf16x8 (&b)[NB], f32x16 c) {
  constexpr int M = NA > NB ? NA : NB;
#pragma unroll
  for (int s = M - 1; s >= 0; s--)
#pragma unroll
    for (int i = 0; i < NA; i++)
      if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[s - i], c, 0, 0, 0);
  return c;
}

template <typename T> struct InParts { static constexpr int N = 1; };
template <> struct InParts<float> { static constexpr int N = 3; };

// Any of eight values infinite or NaN: an exponent of all ones, plus one, carries into the sign bit.
__device__ __forceinline__ bool not_finite(const la_bf16x8& v) {
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  const u4 w = __builtin_bit_cast(u4, v);
  unsigned t = 0;
#pragma unroll
  for (int i = 0; i < 4; i++) t |= (w[i] & 0x7f807f80u) + 0x00800080u;
  return t & 0x80008000u;
}
__device__ __forceinline__ bool not_finite(const f32x8_t& v) {
  typedef unsigned u8 __attribute__((ext_vector_type(8)));
  const u8 w = __builtin_bit_cast(u8, v);
  unsigned t = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) t |= (w[i] & 0x7f800000u) + 0x00800000u;
  return t & 0x80000000u;
}

// base[elems] by a 32-bit byte offset from a base that a wave shares
template <typename T> __device__ __forceinline__ const T* at32(const T* base, unsigned elems) {
  return (const T*)((const char*)base + (size_t)(elems * (unsigned)sizeof(T)));
}

// Reads of a sequence through a buffer descriptor: 32-bit byte offsets from its first token in hand, zeros behind `bytes`.
typedef unsigned la_u32x4 __attribute__((ext_vector_type(4)));
constexpr unsigned LA_NOWHERE = 0xe0000000u;   // behind any descriptor made here, before and after a step of less than 2^29 either way
template <typename T> struct Buf {
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ Buf(const T* base, unsigned bytes)
      : rs(__builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000)) {}
  typedef T vec __attribute__((ext_vector_type(8)));
  __device__ __forceinline__ vec load8(unsigned off) const {
    if constexpr (sizeof(T) == 2) return __builtin_bit_cast(vec, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
    else {
      const f32x4 a = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
      const f32x4 b = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off + 16, 0, 0));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  __device__ __forceinline__ float load1(unsigned off) const {
    if constexpr (sizeof(T) == 2) return __builtin_bit_cast(float, (unsigned)(unsigned short)__builtin_amdgcn_raw_buffer_load_b16(rs, off, 0, 0) << 16);
    else return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, off, 0, 0));
  }
};
// Writes of a chunk's rows, the same way.  (Written under branches, the compiler could not count them, and the wait for the next chunk's reads would be one for
// the writes behind them as well.)
template <typename T> struct OutBuf {
  __amdgpu_buffer_rsrc_t rs;
  __device__ __forceinline__ OutBuf(T* base, unsigned bytes) : rs(__builtin_amdgcn_make_buffer_rsrc(base, 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000)) {}
  // A wave's 32 columns of one row per lane, o[4 m + c] = column 8 m + 4 (lane / 32) + c, d of them wanted; at: byte offset of the row and its first column.  bf16:
  // the half-waves exchange pairs of columns, so that each lane writes 16 bytes.
  __device__ __forceinline__ void row(unsigned at, const f32x16& o, int d, int h5) const {
    if constexpr (sizeof(T) == 2) {
      typedef T t2 __attribute__((ext_vector_type(2)));
      typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int m = 0; m < 4; m += 2) {
        la_u32x4 y;
#pragma unroll
        for (int c = 0; c < 2; c++) {
          const auto x = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, __builtin_convertvector(f2{o[4 * m + 2 * c], o[4 * m + 2 * c + 1]}, t2)),
                                                          __builtin_bit_cast(unsigned, __builtin_convertvector(f2{o[4 * m + 4 + 2 * c], o[4 * m + 5 + 2 * c]}, t2)), false, false);
          y[c] = x[0]; y[2 + c] = x[1];
        }
        __builtin_amdgcn_raw_buffer_store_b128(y, rs, at + (8 * (m + h5) < d ? 8 * (m + h5) * (unsigned)sizeof(T) : LA_NOWHERE), 0, 0);
      }
    } else {
#pragma unroll
      for (int m = 0; m < 4; m++)
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(la_u32x4, f32x4{o[4 * m], o[4 * m + 1], o[4 * m + 2], o[4 * m + 3]}), rs,
                                               at + (8 * m < d ? (8 * m + 4 * h5) * (unsigned)sizeof(T) : LA_NOWHERE), 0, 0);
    }
  }
};
// bytes of n tokens of d channels, st elements apart (st >= d: a row behind them is out of range)
template <typename T> __device__ __forceinline__ unsigned span(int n, int64_t st, int d) { return n > 0 ? (unsigned)(((int64_t)(n - 1) * st + d) * (int)sizeof(T)) : 0u; }

constexpr int C = 32;    // tokens of a chunk
constexpr int CW = 64;   // of a wide one

// A tile's row holds its 16-byte pieces in an order of its own, piece c at place c ^ swz(row): rows read 8 bytes at one channel by 32 lanes (frag_rows) and 64
// bytes of 8 rows read by a transposing load (frag_cols) then both touch every bank equally often.  (Rows padded by 32 bytes instead: row reads 4 on a bank,
// 64 % of the LDS cycles of a sweep at 128 / 128.)
template <int D> __device__ __forceinline__ constexpr int swz(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : D == 64 ? (((row >> 1) & 1) << 2) | ((row >> 2) & 3) : (row >> 2) & 3;
}

// A tile of C tokens x D channels on its way from memory to LDS: 8 channels per piece, L pieces per thread.
template <typename T, int D, int NT, int CT = C> struct Tile {
  static constexpr int NP = InParts<T>::N, PITCH = D * 2, PLANE = CT * PITCH, BYTES = NP * PLANE, L = (CT * D / 8 + NT - 1) / NT;
  typedef T vec __attribute__((ext_vector_type(8)));
  vec r[L];
  unsigned off, step;   // VEC: byte offset of the first piece in a whole chunk, and from one to the next (the same channels, ROWS tokens on)
  static constexpr int ROWS = NT / (D / 8);
  __device__ __forceinline__ void places(int64_t st, int reverse, int d) {
    const int row = threadIdx.x / (D / 8), c = threadIdx.x % (D / 8) * 8;
    off = c < d && row < CT ? ((unsigned)(reverse ? CT - 1 - row : row) * (unsigned)st + c) * (unsigned)sizeof(T) : LA_NOWHERE;
    step = (unsigned)((reverse ? -ROWS : ROWS) * (int)st) * (unsigned)sizeof(T);
  }
  // rows p0 .. p0 + n - 1 of the sequence (position p is token p, or len - 1 - p in reverse), zeros behind; d channels, zeros behind
  template <bool VEC> __device__ __forceinline__ void load(const T* base, int64_t st, int p0, int n, int len, int reverse, int d) {
    if constexpr (VEC) {
      const int64_t first = reverse ? len - p0 - n : p0;
      const Buf<T> buf(base + first * st, span<T>(n, st, d));
      const unsigned short_by = reverse ? (unsigned)(CT - n) * (unsigned)st * (unsigned)sizeof(T) : 0u;   // (rows behind wrap to far offsets)
#pragma unroll
      for (int i = 0; i < L; i++) r[i] = buf.load8(off + i * step - short_by);
    } else {
#pragma unroll
      for (int i = 0; i < L; i++) {
        const int idx = threadIdx.x + i * NT, row = idx / (D / 8), c = idx % (D / 8) * 8;
        vec x = {};
        if (row < n) {
          const int64_t t = reverse ? len - 1 - (p0 + row) : p0 + row;
          const T* src = base + t * st + c;
#pragma unroll
          for (int k = 0; k < 8; k++) if (c + k < d) x[k] = src[k];
        }
        r[i] = x;
      }
    }
  }
  __device__ __forceinline__ void put(char* lds, int i, const vec& v) const {
    const int idx = threadIdx.x + i * NT, row = idx / (D / 8), c = idx % (D / 8) * 8;
    if (CT * D / 8 % NT != 0 && row >= CT) return;
    const int at = row * PITCH + ((c / 8) ^ swz<D>(row)) * 16;
    if constexpr (NP == 1) *reinterpret_cast<vec*>(lds + at) = v;
    else {
      la_bf16x8 p[NP];
      split<NP>(v, p);
#pragma unroll
      for (int k = 0; k < NP; k++) *reinterpret_cast<la_bf16x8*>(lds + k * PLANE + at) = p[k];
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < L; i++) put(lds, i, r[i]);
  }
  // The value tile: a masked P_ij = 0 times a value that is not finite would be NaN in rows in front of it.  Such values go to LDS as 0, bad[e] keeps the
  // first row of column e that has one, and the rows from there on (and the state) become NaN behind the products.
  __device__ __forceinline__ void store_values(char* lds, int* bad, int* any) const {
#pragma unroll
    for (int i = 0; i < L; i++) {
      vec v = r[i];
      const bool off = not_finite(v);
      if (off) {
        const int idx = threadIdx.x + i * NT, row = idx / (D / 8), c = idx % (D / 8) * 8;
#pragma unroll
        for (int k = 0; k < 8; k++)
          if (!(fabsf((float)v[k]) < INFINITY)) { v[k] = (T)0.f; atomicMin(bad + c + k, row); }
        *any = 1;
      }
      put(lds, i, v);
    }
  }
};

// Fragments (8 values of a 16-long K block in the order above).  rows: lane = tile row lane % 32, K = channels d0 ..; cols: lane = channel c0 + lane % 32,
// K = tile rows k0 ..  A lane's addresses differ by constants, added or (within a row's pieces) xor-ed to one base per tile width.
typedef __attribute__((address_space(3))) la_bf16x4* la_p4;
template <int D> struct FragAt {
  unsigned row, lo, hi;
  // base: LDS address of the first tile, a multiple of 256
  __device__ __forceinline__ FragAt(int lane, unsigned base) {
    const int r = lane & 31, t = 4 * (lane >> 5) + ((lane >> 2) & 3), piece = ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1);
    row = base + r * D * 2 + swz<D>(r) * 16 + 8 * (lane >> 5);
    lo = base + t * D * 2 + (piece ^ swz<D>(t)) * 16 + (lane & 1) * 8;
    hi = base + (t + 8) * D * 2 + (piece ^ swz<D>(t + 8)) * 16 + (lane & 1) * 8;
  }
  // keeps the addresses made from it in the loop that calls this (hoisted, they would be spilled)
  __device__ __forceinline__ void again() { asm volatile("" : "+v"(row), "+v"(lo), "+v"(hi)); }
};
// tile: bytes from the first tile, plane: bytes between the parts
template <int NP, int D> __device__ __forceinline__ void frag_rows(const FragAt<D>& at, int tile, int plane, int d0, la_bf16x8 (&f)[NP]) {
#pragma unroll
  for (int k = 0; k < NP; k++) {
    const la_bf16x4 lo = *(la_p4)(uintptr_t)((at.row ^ (d0 * 2)) + (tile + k * plane)), hi = *(la_p4)(uintptr_t)((at.row ^ (d0 * 2 + 16)) + (tile + k * plane));
    f[k] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}
template <int NP, int D> __device__ __forceinline__ void frag_cols(const FragAt<D>& at, unsigned x, int tile, int plane, int k0, int c0, la_bf16x8 (&f)[NP]) {
#pragma unroll
  for (int k = 0; k < NP; k++) {
    const la_bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((la_p4)(uintptr_t)((at.lo ^ x ^ (c0 * 2)) + (tile + k * plane + k0 * D * 2)));
    const la_bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((la_p4)(uintptr_t)((at.hi ^ x ^ (c0 * 2)) + (tile + k * plane + k0 * D * 2)));
    f[k] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// exp(g n) for a distance n >= 0 with the angle in two floats (hardware exp2 of the leading one)
struct Decay {
  float hi, lo;
  __device__ __forceinline__ explicit Decay(float g) {
    hi = g * 1.44269502162933349609f;
    lo = __builtin_fmaf(g, 1.44269502162933349609f, -hi) + g * 1.92596299112661746887e-8f;
  }
  __device__ __forceinline__ float operator()(int n) const {
    if (n == 0) return 1.f;   // (-inf * 0)
    const float f = (float)n, p = hi * f, e = __builtin_fmaf(hi, f, -p) + lo * f;
    const float x = __builtin_amdgcn_exp2f(p);
    return p < -150.f ? 0.f : __builtin_fmaf(x * 0.693147180559945f, e, x);
  }
};
struct Pair { float hi, lo; };
// lambda^n in two floats: as a factor of the state it is applied once for every chunk, and an error of it would grow with their number
__device__ __forceinline__ Pair decay_pair(float g, int n) {
  const double x = n == 0 ? 1.0 : exp((double)g * n);
  const float hi = (float)x;
  return {hi, (float)(x - (double)hi)};
}

// The powers that a workgroup needs in two floats, one lane each (one evaluation of exp for all; in the chunk loop its constants alone would take 40 registers).
enum { POW_CHUNK, POW_TAIL, POW_FIRST, POW_SEG, POW_SEG1, POW_PART, POW_PART1, POW_ONE };
struct Powers {
  float hi, lo;
  // from, to: the workgroup's tokens, chunk: tokens of a whole chunk
  __device__ __forceinline__ Powers(const Sweep& p, float g, int len, int from, int to, int chunk) {
    const int lane = threadIdx.x & 63, mine = max(to - from, 0), part = len % max(p.seg_tokens, 1);
    const int n = lane == POW_CHUNK ? chunk : lane == POW_TAIL ? mine % chunk : lane == POW_FIRST ? min(mine, chunk) - 1 : lane == POW_SEG ? p.seg_tokens
                : lane == POW_SEG1 ? p.seg_tokens - 1 : lane == POW_PART ? part : lane == POW_PART1 ? part - 1 : 1;
    const Pair x = decay_pair(g, max(n, 0));
    hi = x.hi; lo = x.lo;
  }
  __device__ __forceinline__ Pair operator()(int i) const {
    return {__builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, hi), i)), __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, lo), i))};
  }
};

// A state matrix in memory, for the rows 32 t + frag_row(r) and the column of a lane; reads behind it are zero, writes are dropped.
struct StateBuf {
  __amdgpu_buffer_rsrc_t rs;
  unsigned at, step;   // bytes: of the lane's first row, from row to row
  int rows;            // rows there are for this lane
  __device__ __forceinline__ StateBuf(const Sweep& p, const float* m, int e0, int col, int h5)
      : rs(__builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(m), 0, p.dk * p.dv * 4, 0x00020000)), at((4 * h5 * p.in_d + (e0 + col) * p.in_e) * 4),
        step(p.in_d * 4), rows(e0 + col < p.dv ? p.dk - 4 * h5 : 0) {}
  __device__ __forceinline__ unsigned place(int d) const { return d < rows ? at + d * step : LA_NOWHERE; }
  __device__ __forceinline__ float get(int d) const { return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rs, place(d), 0, 0)); }
  __device__ __forceinline__ void put(int d, float x) const { __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), rs, place(d), 0, 0); }
};
// S = S f + m
template <int DK> __device__ __forceinline__ void state_add(const Sweep& p, f32x16 (&S)[DK / 32], const float* m, Pair f, int e0, int col, int h5) {
  const StateBuf buf(p, m, e0, col, h5);
  f32x16 left[DK / 32];   // (all of its reads in flight)
#pragma unroll
  for (int t = 0; t < DK / 32; t++)
#pragma unroll
    for (int r = 0; r < 16; r++) left[t][r] = buf.get(32 * t + frag_row(r, 0));
#pragma unroll
  for (int t = 0; t < DK / 32; t++)
#pragma unroll
    for (int r = 0; r < 16; r++) S[t][r] = __builtin_fmaf(S[t][r], f.hi, __builtin_fmaf(S[t][r], f.lo, left[t][r]));
}
template <int DK> __device__ __forceinline__ void state_put(const Sweep& p, const f32x16 (&S)[DK / 32], float* m, Pair f, int e0, int col, int h5) {
  const StateBuf buf(p, m, e0, col, h5);
#pragma unroll
  for (int t = 0; t < DK / 32; t++)
#pragma unroll
    for (int r = 0; r < 16; r++) buf.put(32 * t + frag_row(r, 0), __builtin_fmaf(S[t][r], f.hi, S[t][r] * f.lo));
}
// lambda^(tokens of segment m), the first one without the decay into its first token for plain_init
__device__ __forceinline__ Pair segment_decay(const Sweep& p, int len, const Powers& pow, int m) {
  const int n = min(max(len - m * p.seg_tokens, 0), p.seg_tokens);
  const bool plain = m == 0 && p.plain_init;
  return n == 0 ? Pair{1.f, 0.f} : n == p.seg_tokens ? pow(plain ? POW_SEG1 : POW_SEG) : pow(plain ? POW_PART1 : POW_PART);
}
// The state in front of a segment.  The last segment's workgroup writes the one that leaves as well (the joining kernel, where there is one), from the segments'
// own states (which are kept to fp32 accuracy, whatever the sweep's outputs need).
template <int DK, bool STATES>
__device__ __forceinline__ void state_in(const Sweep& p, f32x16 (&S)[DK / 32], int bh, int seg, int len, const Powers& pow, int e0, int col, int h5) {
#pragma unroll
  for (int t = 0; t < DK / 32; t++)
#pragma unroll
    for (int r = 0; r < 16; r++) S[t][r] = 0.f;
  if constexpr (!STATES) {
    const int64_t dkdv = p.dk * p.dv;
    const float* slots = p.seg + (int64_t)bh * p.nseg * dkdv;
    const Pair one = {1.f, 0.f};
    if (p.joined && seg > 0) { state_add<DK>(p, S, slots + (seg - 1) * dkdv, one, e0, col, h5); return; }
    if (p.s_in) state_add<DK>(p, S, p.s_in + bh * dkdv, one, e0, col, h5);
    if (p.joined) return;
    for (int m = 0; m < seg; m++) state_add<DK>(p, S, slots + m * dkdv, segment_decay(p, len, pow, m), e0, col, h5);
    if (p.nseg > 1 && seg + 1 == p.nseg && p.s_out) {
      const Pair out = p.decay_out && len > 0 ? pow(POW_ONE) : one, f = segment_decay(p, len, pow, seg);
      const StateBuf mine(p, slots + seg * dkdv, e0, col, h5), dst(p, p.s_out + bh * dkdv, e0, col, h5);
#pragma unroll
      for (int t = 0; t < DK / 32; t++) {
        float left[16];   // (read together: a read behind a write would wait for it)
#pragma unroll
        for (int r = 0; r < 16; r++) left[r] = mine.get(32 * t + frag_row(r, 0));
#pragma unroll
        for (int r = 0; r < 16; r++) {
          const float x = __builtin_fmaf(S[t][r], f.hi, __builtin_fmaf(S[t][r], f.lo, left[r]));
          dst.put(32 * t + frag_row(r, 0), __builtin_fmaf(x, out.hi, x * out.lo));
        }
      }
    }
  }
}
template <int DK, bool STATES>
__device__ __forceinline__ void state_out(const Sweep& p, const f32x16 (&S)[DK / 32], int bh, int seg, int len, const Powers& pow, int e0, int col, int h5) {
  const int64_t dkdv = p.dk * p.dv;
  if constexpr (STATES) state_put<DK>(p, S, p.seg + ((int64_t)bh * p.nseg + seg) * dkdv, Pair{1.f, 0.f}, e0, col, h5);
  else if (p.nseg == 1 && p.s_out) state_put<DK>(p, S, p.s_out + bh * dkdv, p.decay_out && len > 0 ? pow(POW_ONE) : Pair{1.f, 0.f}, e0, col, h5);
}
// where a segment's tokens end (from + seg_tokens itself can pass 2^31 in the last one)
__device__ __forceinline__ int segment_end(const Sweep& p, int len, int from) { return len - from > p.seg_tokens ? from + p.seg_tokens : len; }
template <typename T, int DV> __device__ __forceinline__ void zeros_behind(const Sweep& p, int b, int hd, int seg, int len, int from, int wave, int lane) {
  const int lo = max(len, from), hi = segment_end(p, p.T, from);
  T* o = (T*)p.o.ptr + b * p.o.sb + hd * p.o.sh;
  for (int t = lo + wave; t < hi; t += DV / 32)
    for (int c = lane; c < p.dv; c += 64) o[(int64_t)t * p.o.st + c] = (T)0.f;
}
// which sweep, sequence, head and segment a workgroup works for
struct Place { int role, bh, b, hd, seg; bool live; };
template <bool STATES> __device__ __forceinline__ Place place_of(const Sweeps& all) {
  Place w;
  const int piece = blockIdx.x / (8 * all.n) * 8 + (blockIdx.x & 7);
  w.role = blockIdx.x / 8 % all.n;
  const Sweep& p = all.s[w.role];
  const int pairs = p.B * p.H, nseg = STATES && !p.s_out ? p.nseg - 1 : p.nseg, at = piece / pairs;
  w.live = at < nseg;
  w.bh = piece % pairs; w.b = w.bh / p.H; w.hd = w.bh % p.H;
  w.seg = !STATES && p.reverse ? nseg - 1 - at : at;   // (a reverse sweep counts from the end: the same tokens as its neighbours')
  return w;
}

template <typename T, int DK, int DV, bool STATES> constexpr int chunk_lds() {
  constexpr int NT = DV * 2;
  return (STATES ? 1 : 2) * Tile<T, DK, NT>::BYTES + Tile<T, DV, NT>::BYTES;
}

// STATES: what each segment but the last leaves from a zero state, to p.seg[(bh, segment)]; otherwise the sweep itself, each segment starting from the state
// that came in and what the segments in front of it left.  (Registers: the widths whose tiles leave LDS for one wave per SIMD get all 512.)
template <typename T, int DK, int DV, bool VEC, bool STATES> __global__ void __launch_bounds__(DV * 2, DV == 32 || (DK == 128 && (DV == 64 || sizeof(T) == 4)) ? 1 : 2) la_chunk_kernel(Sweeps all) {
  const Place place = place_of<STATES>(all);
  if (!place.live) return;
  const Sweep& p = all.s[place.role];
  constexpr int NT = DV * 2, NP = InParts<T>::N, PP = NP == 1 ? 2 : 3, NK = C / 16;
  typedef Tile<T, DK, NT> TK;
  typedef Tile<T, DV, NT> TV;
  extern __shared__ __attribute__((aligned(256))) char lds[];
  __shared__ float pw[33 + C];        // pw[32 + n] = lambda^n, 0 for n < 0
  __shared__ __attribute__((aligned(16))) float wt[C];   // kscale * lambda^(n - 1 - j) of the chunk in hand
  __shared__ int bad[DV], any;
  char *lk = lds, *lv = lds + TK::BYTES, *lq = lv + TV::BYTES;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  constexpr int AT_V = TK::BYTES, AT_Q = TK::BYTES + TV::BYTES;
  FragAt<DK> atk(threadIdx.x & 63, lds0);
  FragAt<DV> atv(threadIdx.x & 63, lds0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, h5 = lane >> 5, e0 = wave * 32;
  const int bh = place.bh, b = place.b, hd = place.hd, seg = place.seg;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const int from = seg * p.seg_tokens, to = segment_end(p, len, from);   // (the last segment reaches T)
  const float g = p.g[hd];
  const Decay decay(g);
  const T* q = (const T*)p.q.ptr + b * p.q.sb + hd * p.q.sh;
  const T* k = (const T*)p.k.ptr + b * p.k.sb + hd * p.k.sh;
  const T* v = (const T*)p.v.ptr + b * p.v.sb + hd * p.v.sh;

  TK rk; TV rv; TK rq;
  auto fetch = [&](int c0) {
    const int n = min(C, to - c0);
    rk.template load<VEC>(k, p.k.st, c0, n, len, p.reverse, p.dk);
    rv.template load<VEC>(v, p.v.st, c0, n, len, p.reverse, p.dv);
    if (!STATES) rq.template load<VEC>(q, p.q.st, c0, n, len, p.reverse, p.dk);
  };
  if constexpr (VEC) {
    rk.places(p.k.st, p.reverse, p.dk); rv.places(p.v.st, p.reverse, p.dv);
    if (!STATES) rq.places(p.q.st, p.reverse, p.dk);
  }
  // STATES: from the last chunk to the first (what the sweep that follows reads first is what was read last)
  const int first = STATES ? (from < to ? from + (to - from - 1) / C * C : from - C) : from;
  if (from < to) fetch(first);
  for (int n = tid; n < 33 + C; n += NT) pw[n] = n < 32 ? 0.f : decay(n - 32);
  for (int n = tid; n < C; n += NT) wt[n] = p.kscale * decay(C - 1 - n);
  for (int n = tid; n < DV; n += NT) bad[n] = C;
  if (tid == 0) any = 0;

  f32x16 S[DK / 32];
  const Powers pow(p, g, len, from, to, C);
  state_in<DK, STATES>(p, S, bh, seg, len, pow, e0, col, h5);
  const Pair full = pow(POW_CHUNK);
  float carry = 0.f;   // what the factors applied so far lack of lambda^C each: every factor takes it in, so that their product keeps to lambda^(C m)

  // D^T times the scales (registers: tokens j of P^T)
  float D[16];
  if constexpr (!STATES) {
    la_sync();
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int d = col - frag_row(r, h5);
      D[r] = d >= 0 ? pw[32 + d] * (p.kscale * p.oscale) : 0.f;
    }
  }

  la_arrived();
  for (int c0 = first; STATES ? c0 >= from : c0 < to; c0 += STATES ? -C : C) {
    const int n = min(C, to - c0);
    la_sync();   // the previous chunk has been read
    atk.again(); atv.again();
    rk.store(lk); rv.store_values(lv, bad, &any);
    if (!STATES) rq.store(lq);
    if (STATES) for (int j = tid; j < C; j += NT) wt[j] = j < n ? p.kscale * decay(to - 1 - c0 - j) : 0.f;
    else if (n < C) for (int j = tid; j < C; j += NT) wt[j] = j < n ? p.kscale * decay(n - 1 - j) : 0.f;
    la_sync();
    if (STATES ? c0 > from : c0 + C < to) fetch(c0 + (STATES ? -C : C));
    if (e0 >= p.dv) continue;   // (a wave without columns has only loaded)
    const bool plain = p.plain_init && c0 == 0;   // the state that came in meets the first token without a decay

    la_bf16x8 vf[NK][NP];
    if constexpr (!STATES) {
      f32x16 o = {}, st = {};
#pragma unroll
      for (int s = 0; s < DK / 16; s++) {
        f32x8_t x;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = S[s / 2][8 * (s & 1) + i];
        la_bf16x8 sp[PP], kf[NP], qf[NP];
        split<PP, true>(x, sp);
        frag_rows<NP, DK>(atk, 0, TK::PLANE, 16 * s, kf);
        frag_rows<NP, DK>(atk, AT_Q, TK::PLANE, 16 * s, qf);
        o = mm<PP, NP>(sp, qf, o);
        st = mm<NP, NP>(kf, qf, st);
      }
#pragma unroll
      for (int s = 0; s < NK; s++) frag_cols<NP, DV>(atv, e0 * 2, AT_V, TV::PLANE, 16 * s, 0, vf[s]);
      const float ai = pw[32 + col + (plain ? 0 : 1)] * p.oscale;
#pragma unroll
      for (int r = 0; r < 16; r++) o[r] *= ai;
#pragma unroll
      for (int s = 0; s < NK; s++) {
        f32x8_t x;
#pragma unroll
        for (int r = 0; r < 8; r++) x[r] = col >= frag_row(8 * s + r, h5) ? D[8 * s + r] * st[8 * s + r] : 0.f;   // (a masked score may be NaN)
        la_bf16x8 pp[PP];
        split<PP, true>(x, pp);
        o = mm<NP, PP>(vf[s], pp, o);
      }
      if (any) {
#pragma unroll
        for (int r = 0; r < 16; r++) if (col >= bad[e0 + frag_row(r, h5)]) o[r] = NAN;
      }
      T* out = (T*)p.o.ptr + b * p.o.sb + hd * p.o.sh;
      if constexpr (VEC) {
        const OutBuf<T> buf(out + (int64_t)(p.reverse ? len - c0 - n : c0) * p.o.st, span<T>(n, p.o.st, p.dv));
        buf.row(((unsigned)(p.reverse ? n - 1 - col : col) * (unsigned)p.o.st + e0) * (unsigned)sizeof(T), o, p.dv - e0, h5);
      } else if (col < n) {
        const int64_t t = p.reverse ? len - 1 - (c0 + col) : c0 + col;
        T* dst = out + t * p.o.st + e0 + 4 * h5;
#pragma unroll
        for (int m = 0; m < 4; m++)
#pragma unroll
          for (int c = 0; c < 4; c++) if (e0 + 4 * h5 + 8 * m + c < p.dv) dst[8 * m + c] = (T)o[4 * m + c];
      }
    } else {
#pragma unroll
      for (int s = 0; s < NK; s++) frag_cols<NP, DV>(atv, e0 * 2, AT_V, TV::PLANE, 16 * s, 0, vf[s]);
    }
    if constexpr (!STATES) {   // (there the weights reach to the segment's end)
      float dec;
      if (n == C && !plain) {
        const float want = carry + full.lo;
        dec = full.hi + want;
        carry = want - (dec - full.hi);
      } else dec = pow(plain ? POW_FIRST : POW_TAIL).hi;
#pragma unroll
      for (int t = 0; t < DK / 32; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) S[t][r] *= dec;
    }
#pragma unroll
    for (int s = 0; s < NK; s++) {
      const f32x4 wa = *reinterpret_cast<const f32x4*>(wt + 16 * s + 4 * h5), wb = *reinterpret_cast<const f32x4*>(wt + 16 * s + 8 + 4 * h5);
      f32x8_t x = __builtin_convertvector(vf[s][0], f32x8_t);
#pragma unroll
      for (int i = 1; i < NP; i++) x += __builtin_convertvector(vf[s][i], f32x8_t);
      x *= f32x8_t{wa[0], wa[1], wa[2], wa[3], wb[0], wb[1], wb[2], wb[3]};
      if (s == 0 && any && bad[e0 + col] < C) x[0] = NAN;   // (NaN times any k: the whole column)
      la_bf16x8 vp[3];
      split<3, true>(x, vp);
#pragma unroll
      for (int t = 0; t < DK / 32; t++) {
        la_bf16x8 kt[NP];
        frag_cols<NP, DK>(atk, 0, 0, TK::PLANE, 16 * s, 32 * t, kt);
        if constexpr (NP == 1) {   // (the third part only where the state leaves in fp32)
          if (STATES || (p.s_out && p.nseg == 1)) S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[0], vp[2], S[t], 0, 0, 0);
          S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[0], vp[1], S[t], 0, 0, 0);
          S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[0], vp[0], S[t], 0, 0, 0);
        } else S[t] = mm<NP, 3>(kt, vp, S[t]);
      }
    }
  }

  state_out<DK, STATES>(p, S, bh, seg, len, pow, e0, col, h5);
  if constexpr (!STATES) zeros_behind<T, DV>(p, b, hd, seg, len, from, wave, lane);
}

// The same for bf16 tensors that can be moved 16 bytes at a time, two 32-token tiles at a time: the state is decayed and split into operand parts half as
// often, and a tile of P^T is made by one wave for all (its parts go through LDS, in fragment order).
// Bound, at B 1, T 65536, H 8, 128 / 128 (64 segments, two workgroups on each CU): the main sweep takes 130 - 180 us, 161 in the mean; its 540 MB cost 100 us at the rate of a copy, its
// instructions 105 - two waves a SIMD are too few to cover one with the other, and the matrix instructions (36 us) too few to cover the vector ones that split S, P and
// the values (a state of 128 x 128 takes 64 registers, the next chunk's tokens 48).  The segments' states: 78 us for 268 MB, 50 at the rate of a copy.  256 registers; at 128 / 128 twelve bytes a lane are spilled.
template <int DK, int DV, bool STATES> constexpr int wide_lds() { return (STATES ? 1 : 2) * CW * DK * 2 + CW * DV * 2 + (STATES ? 0 : 3 * 4096); }
// MODE: the sweep, the sweep with a state that leaves it in fp32, the segments' states.
enum { WIDE_SWEEP, WIDE_SWEEP_STATE, WIDE_STATES };
template <int DK, int DV, int MODE> __global__ void __launch_bounds__(DV * 2, DK == 128 && DV == 64 ? 1 : 2) la_wide_kernel(Sweeps all) {
  constexpr bool STATES = MODE == WIDE_STATES, THIRD = MODE != WIDE_SWEEP;
  const Place place = place_of<STATES>(all);
  if (!place.live) return;
  const Sweep& p = all.s[place.role];
  typedef __bf16 T;
  constexpr int NT = DV * 2, NW = DV / 32, NK = CW / 16;
  typedef Tile<T, DK, NT, CW> TK;
  typedef Tile<T, DV, NT, CW> TV;
  extern __shared__ __attribute__((aligned(256))) char lds[];
  __shared__ float pw[33 + CW];
  __shared__ __attribute__((aligned(16))) float wt[CW];
  char *lk = lds, *lv = lds + TK::BYTES, *lq = lv + TV::BYTES, *lp = lq + TK::BYTES;
  const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  constexpr int AT_V = TK::BYTES, AT_Q = TK::BYTES + TV::BYTES;
  FragAt<DK> atk(threadIdx.x & 63, lds0);
  FragAt<DV> atv(threadIdx.x & 63, lds0);
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, h5 = lane >> 5, e0 = wave * 32;
  const int bh = place.bh, b = place.b, hd = place.hd, seg = place.seg;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const int from = seg * p.seg_tokens, to = segment_end(p, len, from);
  const float g = p.g[hd], kscale = p.kscale, oscale = p.oscale;
  const int reverse = p.reverse, dk = p.dk, dv = p.dv;
  const int64_t qst = p.q.st, kst = p.k.st, vst = p.v.st, ost = p.o.st;
  const T* q = (const T*)p.q.ptr + b * p.q.sb + hd * p.q.sh;
  const T* k = (const T*)p.k.ptr + b * p.k.sb + hd * p.k.sh;
  const T* v = (const T*)p.v.ptr + b * p.v.sb + hd * p.v.sh;
  T* out = (T*)p.o.ptr + b * p.o.sb + hd * p.o.sh;
  const Decay decay(g);

  TK rk; TV rv; TK rq;
  rk.places(kst, reverse, dk); rv.places(vst, reverse, dv);
  if (!STATES) rq.places(qst, reverse, dk);
  auto fetch = [&](int c0) {
    const int n = min(CW, to - c0);
    rk.template load<true>(k, kst, c0, n, len, reverse, dk);
    rv.template load<true>(v, vst, c0, n, len, reverse, dv);
    if (!STATES) rq.template load<true>(q, qst, c0, n, len, reverse, dk);
  };
  // STATES: from the last chunk to the first (what the sweep that follows reads first is what was read last)
  const int first = STATES ? (from < to ? from + (to - from - 1) / CW * CW : from - CW) : from;
  if (from < to) fetch(first);
  for (int n = tid; n < 33 + CW; n += NT) pw[n] = n < 32 ? 0.f : decay(n - 32);
  for (int n = tid; n < CW; n += NT) wt[n] = kscale * decay(CW - 1 - n);
  f32x16 S[DK / 32];
  const Powers pow(p, g, len, from, to, CW);
  state_in<DK, STATES>(p, S, bh, seg, len, pow, e0, col, h5);
  const Pair full = pow(POW_CHUNK);
  float carry = 0.f;
  // this wave's tiles of P^T: the two on the diagonal (0, 1) or the one under it (2)
  const bool under = NW == 4 ? wave == 2 : wave == 1;
  const float p_by = kscale * oscale;

  la_arrived();
  for (int c0 = first; STATES ? c0 >= from : c0 < to; c0 += STATES ? -CW : CW) {
    const int n = min(CW, to - c0);
    la_sync();   // the previous chunk has been read
    atk.again(); atv.again();
    rk.store(lk); rv.store(lv);
    if (!STATES) rq.store(lq);
    if (STATES) for (int j = tid; j < CW; j += NT) wt[j] = j < n ? kscale * decay(to - 1 - c0 - j) : 0.f;
    else if (n < CW) for (int j = tid; j < CW; j += NT) wt[j] = j < n ? kscale * decay(n - 1 - j) : 0.f;
    la_sync();
    if (STATES ? c0 > from : c0 + CW < to) fetch(c0 + (STATES ? -CW : CW));
    const bool plain = p.plain_init && c0 == 0;   // the state that came in meets the first token without a decay
    if constexpr (!STATES) {
#pragma unroll 1
      for (int tile = NW == 4 ? wave : 2 * wave; tile < (NW == 4 ? wave + (wave < 3) : wave == 0 ? 2 : 3); tile++) {
        FragAt<DK> ka = atk, qa = atk;
        ka.row += tile == 1 ? 32 * DK * 2 : 0;
        qa.row += tile > 0 ? 32 * DK * 2 : 0;
        f32x16 st = {};
#pragma unroll
        for (int s = 0; s < DK / 16; s++) {
          la_bf16x8 kf[1], qf[1];
          frag_rows<1, DK>(ka, 0, 0, 16 * s, kf);
          frag_rows<1, DK>(qa, AT_Q, 0, 16 * s, qf);
          st = mm<1, 1>(kf, qf, st);
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
          f32x8_t x;
#pragma unroll
          for (int r = 0; r < 8; r++) {
            const int d = col - frag_row(8 * s + r, h5) + (under ? 32 : 0);
            const float w = st[8 * s + r] * (pw[32 + d] * p_by);
            x[r] = d >= 0 ? w : 0.f;   // (a masked score may be NaN)
          }
          la_bf16x8 pp[2];
          split<2, true>(x, pp);
#pragma unroll
          for (int i = 0; i < 2; i++) *reinterpret_cast<la_bf16x8*>(lp + tile * 4096 + (2 * s + i) * 1024 + lane * 16) = pp[i];
        }
      }
      la_sync();   // the tiles of P^T are there
    }
    if (e0 >= dv) continue;   // (a wave without columns has only loaded and made its tile)
    // the values' fragments serve both products; one that is not finite is taken out of them (a masked 0 times it would be NaN), its first row kept: the
    // results from there on, and the state, become NaN
    la_bf16x8 vf[NK];
    bool off = false;
#pragma unroll
    for (int s = 0; s < NK; s++) {
      la_bf16x8 f[1];
      frag_cols<1, DV>(atv, e0 * 2, AT_V, 0, 16 * s, 0, f);
      vf[s] = f[0];
      off |= not_finite(f[0]);
    }
    int bad = CW;
    const bool poison = __any(off);
    if (poison) {
#pragma unroll
      for (int s = 0; s < NK; s++)
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (!(fabsf((float)vf[s][i]) < INFINITY)) { bad = min(bad, 16 * s + (i & 3) + 8 * (i >> 2) + 4 * h5); vf[s][i] = (T)0.f; }
      bad = min(bad, __shfl_xor(bad, 32));
    }
    if constexpr (!STATES) {
      const OutBuf<T> buf(out + (int64_t)(reverse ? len - c0 - n : c0) * ost, span<T>(n, ost, dv));
      f32x16 o[2] = {};
#pragma unroll
      for (int s = 0; s < DK / 16; s++) {
        f32x8_t x;
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = S[s / 2][8 * (s & 1) + i];
        la_bf16x8 sp[2];
        split<2, true>(x, sp);
#pragma unroll
        for (int i = 0; i < 2; i++) {
          la_bf16x8 qf[1];
          frag_rows<1, DK>(atk, AT_Q + i * 32 * DK * 2, 0, 16 * s, qf);
          o[i] = mm<2, 1>(sp, qf, o[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float a = pw[32 + 32 * i + col + (plain ? 0 : 1)] * oscale;
#pragma unroll
        for (int r = 0; r < 16; r++) o[i][r] *= a;
#pragma unroll
        for (int j = 0; j <= i; j++) {
          const char* a = lp + (i == 0 ? 0 : j == 1 ? 1 : 2) * 4096 + lane * 16;
          la_bf16x8 pp[4];
#pragma unroll
          for (int m = 0; m < 4; m++) pp[m] = *reinterpret_cast<const la_bf16x8*>(a + m * 1024);
#pragma unroll
          for (int s = 0; s < 2; s++) {
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[2 * j + s], pp[2 * s + 1], o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[2 * j + s], pp[2 * s], o[i], 0, 0, 0);
          }
        }
        if (poison) {
#pragma unroll
          for (int r = 0; r < 16; r++) if (32 * i + col >= __shfl(bad, frag_row(r, h5))) o[i][r] = NAN;
        }
        buf.row(((unsigned)(reverse ? n - 1 - 32 * i - col : 32 * i + col) * (unsigned)ost + e0) * (unsigned)sizeof(T), o[i], dv - e0, h5);
      }
    }
    if constexpr (!STATES) {   // (there the weights reach to the segment's end)
      float dec;
      if (n == CW && !plain) {
        const float want = carry + full.lo;
        dec = full.hi + want;
        carry = want - (dec - full.hi);
      } else dec = pow(plain ? POW_FIRST : POW_TAIL).hi;
#pragma unroll
      for (int t = 0; t < DK / 32; t++)
#pragma unroll
        for (int r = 0; r < 16; r++) S[t][r] *= dec;
    }
#pragma unroll
    for (int s = 0; s < NK; s++) {
      const f32x4 wa = *reinterpret_cast<const f32x4*>(wt + 16 * s + 4 * h5), wb = *reinterpret_cast<const f32x4*>(wt + 16 * s + 8 + 4 * h5);
      f32x8_t x = __builtin_convertvector(vf[s], f32x8_t);
      x *= f32x8_t{wa[0], wa[1], wa[2], wa[3], wb[0], wb[1], wb[2], wb[3]};
      if (s == 0 && bad < CW) x[0] = NAN;   // (NaN times any k: the whole column)
      la_bf16x8 vp[3];
      split<3, true>(x, vp);
#pragma unroll
      for (int t = 0; t < DK / 32; t++) {
        la_bf16x8 kt[1];
        frag_cols<1, DK>(atk, 0, 0, 0, 16 * s, 32 * t, kt);
        if (THIRD) S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[0], vp[2], S[t], 0, 0, 0);
        S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[0], vp[1], S[t], 0, 0, 0);
        S[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt[0], vp[0], S[t], 0, 0, 0);
      }
    }
  }
  state_out<DK, STATES>(p, S, bh, seg, len, pow, e0, col, h5);
  if constexpr (!STATES) zeros_behind<T, DV>(p, b, hd, seg, len, from, wave, lane);
}

// The states behind the segments from what each leaves: slot s becomes lambda^(tokens of s) (state in front of s) + slot s, in place; the last one leaves.
__global__ void __launch_bounds__(256) la_join_kernel(Sweep p) {
  const int bh = blockIdx.x, b = bh / p.H;
  const int len = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const int64_t dkdv = p.dk * p.dv;
  const int i = blockIdx.y * 256 + threadIdx.x;
  const float g = p.g[bh % p.H];
  const bool in = i < dkdv;
  float s = p.s_in && in ? p.s_in[bh * dkdv + i / p.dv * p.in_d + i % p.dv * p.in_e] : 0.f;
  float* slot = p.seg + (int64_t)bh * p.nseg * dkdv + i;
  const int slots = p.s_out ? p.nseg : p.nseg - 1;
  const Powers pow(p, g, len, 0, 0, 1);
  constexpr int AHEAD = 8;
  for (int m0 = 0; m0 < slots; m0 += AHEAD) {
    float left[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; j++) left[j] = in && m0 + j < slots ? slot[(m0 + j) * dkdv] : 0.f;
#pragma unroll
    for (int j = 0; j < AHEAD; j++) {
      const int m = m0 + j;
      if (m >= slots) break;
      const Pair d = segment_decay(p, len, pow, m);
      s = __builtin_fmaf(s, d.hi, __builtin_fmaf(s, d.lo, left[j]));
      if (in && m + 1 < p.nseg) slot[m * dkdv] = s;
    }
  }
  if (p.s_out && in) {
    const Pair out = p.decay_out && len > 0 ? pow(POW_ONE) : Pair{1.f, 0.f};
    p.s_out[bh * dkdv + i / p.dv * p.in_d + i % p.dv * p.in_e] = __builtin_fmaf(s, out.hi, s * out.lo);
  }
}

// ---- sequences of at most one chunk -----------------------------------------------------------------------------------------------------------
// Many short sequences (the pixels of a map over some frames): one wave per (sequence, head), nothing in LDS but a table of decays.  Operands whose K axis
// is channels are read row by row (lane = token, 8 channels); operands whose K axis is tokens column by column (lane = channel, one row of 32 channels per
// half-wave and load), straight into fragment order, so that nothing is transposed.  Bound by memory: the second reading of a tensor hits the cache.  (8192
// sequences of 24 tokens, 4 heads of 32 / 32, fp32: forward 92 us for 403 MB, 4.4 TB/s; backward 243 us for 705 MB, 2.9 TB/s - 12 of its 28 reads of 16 bytes a
// lane are columns, 4 bytes a lane, and 230 registers leave two waves a SIMD.)
struct Short {
  sfSeq q, k, v, o;          // forward
  sfSeq dout, dq, dk_, dv_;  // backward
  const float* g;
  const float* s_in;         // [B][H][dk][dv]
  float* s_out;
  const float* ds_out;
  float* ds_in;
  const int32_t* lengths;
  int B, T, H, dk, dv;
  float scale;
};

// A sequence's tensor for one wave.  row: lane = token, channels c .. c + 7; col: lane = channel c, tokens k0 + 4 h .. + 3 and k0 + 8 + 4 h .. + 3; zeros
// behind n tokens and d channels.  VEC: through a descriptor; otherwise element by element, unconditionally - of token 0 and channel 0, dropped afterwards,
// where there is nothing to read -, by 32-bit offsets from the wave's own base.
template <typename T, bool VEC> struct Rows {
  const T* base;
  unsigned st;
  int n, d;
  __device__ __forceinline__ Rows(const sfSeq& t, int b, int hd, int n_, int d_) : base((const T*)t.ptr + b * t.sb + hd * t.sh), st((unsigned)t.st), n(n_), d(d_) {}
  __device__ __forceinline__ typename Buf<T>::vec row(int tok, int c) const {
    if constexpr (VEC) return Buf<T>(base, span<T>(n, st, d)).load8(c < d ? ((unsigned)tok * st + c) * (unsigned)sizeof(T) : LA_NOWHERE);
    else {
      const unsigned at = (unsigned)(tok < n ? tok : 0) * st;
      typename Buf<T>::vec x;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const T v = *at32(base, at + (c + i < d ? c + i : 0));
        x[i] = tok < n && c + i < d ? v : (T)0.f;
      }
      return x;
    }
  }
  __device__ __forceinline__ f32x8_t col(int k0, int c, int h5) const {
    f32x8_t x;
    if constexpr (VEC) {
      const Buf<T> buf(base, span<T>(n, st, d));
      const unsigned at = c < d ? ((unsigned)(4 * h5) * st + c) * (unsigned)sizeof(T) : LA_NOWHERE;
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = buf.load1(at + (unsigned)(k0 + (i & 3) + 8 * (i >> 2)) * st * (unsigned)sizeof(T));
    } else {
      const unsigned at = c < d ? c : 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int tok = k0 + (i & 3) + 8 * (i >> 2) + 4 * h5;
        const T v = *at32(base, at + (unsigned)(tok < n ? tok : 0) * st);
        x[i] = tok < n && c < d ? (float)v : 0.f;
      }
    }
    return x;
  }
};
template <int NP, typename V> __device__ __forceinline__ void parts(const V& x, la_bf16x8 (&p)[NP]) {
  if constexpr (NP == 1) p[0] = x;
  else split<NP>(x, p);
}
// a row of a dense fp32 matrix: columns c .. c + 7
__device__ __forceinline__ f32x8_t mat_row8(const float* m, int row, int rows, int c, int dv) {
  f32x8_t x;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const bool in = row < rows && c + i < dv;
    const float v = *at32(m, in ? row * dv + c + i : 0);
    x[i] = in ? v : 0.f;
  }
  return x;
}
// lane = column c of a dense fp32 matrix of dv columns: rows k0 .. k0 + 7 (its transpose as an operand over channels)
__device__ __forceinline__ f32x8_t mat_cols8(const float* m, int k0, int rows, int c, int dv) {
  f32x8_t x;
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const bool in = k0 + i < rows && c < dv;
    const float v = *at32(m, in ? (k0 + i) * dv + c : 0);
    x[i] = in ? v : 0.f;
  }
  return x;
}

// Keeps a loop's reads and their addresses in the loop: hoisted, what every turn needs would be spilled.
__device__ __forceinline__ void reload(int& at) { asm volatile("" : "+v"(at)); }

// The values of a masked product: what is not finite is taken out of the fragments (a masked 0 times it would be NaN) and its first (LAST: last) token kept;
// results that it reaches become NaN behind the product.
template <bool LAST> struct Poison {
  int at = LAST ? -1 : C;
  __device__ __forceinline__ void take(f32x8_t& x, int k0, int h5) {
    if (!__any(not_finite(x))) return;
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (!(fabsf(x[i]) < INFINITY)) {
        const int row = k0 + (i & 3) + 8 * (i >> 2) + 4 * h5;
        at = LAST ? max(at, row) : min(at, row);
        x[i] = 0.f;
      }
  }
  __device__ __forceinline__ void give(f32x16& o, int col, int h5) {
    if (!__any(LAST ? at >= 0 : at < C)) return;
    const int other = __shfl_xor(at, 32);
    const int all = LAST ? max(at, other) : min(at, other);
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const int a = __shfl(all, frag_row(r, h5));
      if (LAST ? col <= a : col >= a) o[r] = NAN;
    }
  }
};

// x o D as operand parts: 16 registers = tokens in fragment order
template <int PP> __device__ __forceinline__ void masked(const f32x16& st, const float* pw, int col, int h5, bool transposed, float scale, la_bf16x8 (&pp)[2][PP]) {
#pragma unroll
  for (int s = 0; s < 2; s++) {
    f32x8_t x;
#pragma unroll
    for (int r = 0; r < 8; r++) {
      const int row = frag_row(8 * s + r, h5), n = transposed ? col - row : row - col;   // (transposed: lane = later token i, registers = j)
      x[r] = n >= 0 ? st[8 * s + r] * (pw[32 + n] * scale) : 0.f;
    }
    split<PP>(x, pp[s]);
  }
}

// out[row col][c0 + 8 m + 4 h ..] = o^T, zeros behind n rows
template <typename T> __device__ __forceinline__ void store_rows(const f32x16& o, T* base, int st, int col, int h5, int n, int T_, int c0, int d, bool vec) {
  if (col >= T_) return;
  T* dst = const_cast<T*>(at32((const T*)base, (unsigned)col * (unsigned)st + c0 + 4 * h5));
#pragma unroll
  for (int m = 0; m < 4; m++) {
    f32x4 y = {o[4 * m], o[4 * m + 1], o[4 * m + 2], o[4 * m + 3]};
    if (col >= n) y = f32x4{0.f, 0.f, 0.f, 0.f};
    const int e = c0 + 4 * h5 + 8 * m;
    if (vec) { if (e < d) stv4<T>(dst + 8 * m, y); }
    else
#pragma unroll
      for (int c = 0; c < 4; c++) if (e + c < d) dst[8 * m + c] = (T)y[c];
  }
}

// acc (lane = column c0e + col, registers = rows c0d + ..) = lambda^n in + sum over tokens of a_token (x) (w b)_token
template <typename T, bool VEC, int NP>
__device__ __forceinline__ void short_state(const Rows<T, VEC>& a, const Rows<T, VEC>& b, const float* in, float* out, const float* pw, float dec, bool later, float scale,
                                            int c0d, int c0e, int col, int h5) {
  const int n = a.n, dk = a.d, dv = b.d;
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const int d = c0d + frag_row(r, h5), e = c0e + col;
    acc[r] = in && d < dk && e < dv ? in[d * dv + e] * dec : 0.f;
  }
#pragma unroll
  for (int s = 0; s < 2; s++) {
    f32x8_t x = b.col(16 * s, c0e + col, h5), y = a.col(16 * s, c0d + col, h5);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const int t = 16 * s + (i & 3) + 8 * (i >> 2) + 4 * h5;
      x[i] *= t < n ? pw[32 + (later ? t + 1 : n - 1 - t)] * scale : 0.f;
    }
    la_bf16x8 xp[3], yp[NP];
    split<3>(x, xp); split<NP>(y, yp);
    acc = mm<NP, 3>(yp, xp, acc);
  }
#pragma unroll
  for (int r = 0; r < 16; r++) {
    const int d = c0d + frag_row(r, h5), e = c0e + col;
    if (d < dk && e < dv) out[d * dv + e] = acc[r];
  }
}

template <typename T, int DK, int DV, bool VEC> __global__ void __launch_bounds__(256, VEC ? 2 : 1) la_short_fwd_kernel(Short p) {
  constexpr int NP = InParts<T>::N, PP = NP == 1 ? 2 : 3;
  typedef typename Buf<T>::vec vec;
  __shared__ float pws[4][66];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h5 = lane >> 5;
  const unsigned pair = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(wave);
  const bool live = pair < (unsigned)p.B * (unsigned)p.H;
  const int b = live ? (int)(pair / (unsigned)p.H) : 0, hd = live ? (int)(pair % (unsigned)p.H) : 0;
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const Rows<T, VEC> q(p.q, b, hd, n, p.dk), k(p.k, b, hd, n, p.dk), v(p.v, b, hd, n, p.dv);
  // all that the first value tile needs is on its way before anything is waited for
  vec kr[DK / 16], qr[DK / 16];
  f32x8_t vr[2];
#pragma unroll
  for (int s = 0; s < DK / 16; s++) { kr[s] = k.row(col, 16 * s + 8 * h5); qr[s] = q.row(col, 16 * s + 8 * h5); }
#pragma unroll
  for (int s = 0; s < 2; s++) vr[s] = v.col(16 * s, col, h5);
  const float g = p.g[hd];
  float* pw = pws[wave];
  { const Decay decay(g); if (lane < 33) pw[32 + lane] = decay(lane); }
  la_sync();
  if (!live) return;
  T* o = (T*)p.o.ptr + b * p.o.sb + hd * p.o.sh;
  const float* S = p.s_in ? p.s_in + (int64_t)pair * p.dk * p.dv : nullptr;

  f32x16 st = {};
#pragma unroll
  for (int s = 0; s < DK / 16; s++) {
    la_bf16x8 kf[NP], qf[NP];
    parts<NP>(kr[s], kf); parts<NP>(qr[s], qf);
    st = mm<NP, NP>(kf, qf, st);
  }
  la_bf16x8 pp[2][PP];
  masked<PP>(st, pw, col, h5, true, p.scale, pp);
#pragma unroll 1
  for (int e0 = 0; e0 < p.dv; e0 += 32) {
    int at = col;
    reload(at);
    f32x16 acc = {};
    if (S) {
#pragma unroll
      for (int s = 0; s < DK / 16; s++) {
        la_bf16x8 sf[PP], qf[NP];
        split<PP>(mat_cols8(S, 16 * s + 8 * h5, p.dk, e0 + at, p.dv), sf);
        parts<NP>(q.row(at, 16 * s + 8 * h5), qf);
        acc = mm<PP, NP>(sf, qf, acc);
      }
      const float a = pw[33 + col] * p.scale;
#pragma unroll
      for (int r = 0; r < 16; r++) acc[r] *= a;
    }
    Poison<false> bad;
#pragma unroll
    for (int s = 0; s < 2; s++) {
      f32x8_t x = vr[s];
      bad.take(x, 16 * s, h5);
      la_bf16x8 vf[NP];
      split<NP>(x, vf);
      acc = mm<NP, PP>(vf, pp[s], acc);
    }
    if (e0 + 32 < p.dv)
#pragma unroll
      for (int s = 0; s < 2; s++) vr[s] = v.col(16 * s, e0 + 32 + at, h5);
    bad.give(acc, col, h5);
    store_rows<T>(acc, o, (int)p.o.st, col, h5, n, p.T, e0, p.dv, VEC);
  }
  if (p.s_out) {
    const float dec = decay_pair(g, n).hi;
    for (int d0 = 0; d0 < p.dk; d0 += 32)
      for (int e0 = 0; e0 < p.dv; e0 += 32)
        short_state<T, VEC, NP>(k, v, S, p.s_out + (int64_t)pair * p.dk * p.dv, pw, dec, false, 1.f, d0, e0, col, h5);
  }
}

// dP = dO V^T:  dQ = scale ((dP o D) K + lambda^(i+1) dO S^T) ,  dK = scale (dP o D)^T Q + lambda^(n-1-j) V R^T ,  dV = scale ((Q K^T) o D)^T dO + lambda^(n-1-j) K R
// with R the gradient of the state that left, and the gradient of the one that came in lambda^n R + scale sum_i lambda^(i+1) q_i do_i^T.
template <typename T, int DK, int DV, bool VEC> __global__ void __launch_bounds__(256, VEC && DK + DV < 256 ? 2 : 1) la_short_bwd_kernel(Short p) {
  constexpr int NP = InParts<T>::N, PP = NP == 1 ? 2 : 3;
  typedef typename Buf<T>::vec vec;
  __shared__ float pws[4][66];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 31, h5 = lane >> 5;
  const unsigned pair = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(wave);
  const bool live = pair < (unsigned)p.B * (unsigned)p.H;
  const int b = live ? (int)(pair / (unsigned)p.H) : 0, hd = live ? (int)(pair % (unsigned)p.H) : 0;
  const int n = p.lengths ? min(max(p.lengths[b], 0), p.T) : p.T;
  const Rows<T, VEC> q(p.q, b, hd, n, p.dk), k(p.k, b, hd, n, p.dk), v(p.v, b, hd, n, p.dv), go(p.dout, b, hd, n, p.dv);
  la_bf16x8 dpt[2][PP], dp[2][PP], pp[2][PP];
  f32x8_t kr[2], qr[2], gr[2];   // columns of the first tiles
  float* pw = pws[wave];
  const float g = p.g[hd];
  {
    vec vr[DV / 16], gw[DV / 16], kw[DK / 16], qw[DK / 16];
#pragma unroll
    for (int s = 0; s < DV / 16; s++) { vr[s] = v.row(col, 16 * s + 8 * h5); gw[s] = go.row(col, 16 * s + 8 * h5); }
#pragma unroll
    for (int s = 0; s < DK / 16; s++) { kw[s] = k.row(col, 16 * s + 8 * h5); qw[s] = q.row(col, 16 * s + 8 * h5); }
    { const Decay decay(g); if (lane < 33) pw[32 + lane] = decay(lane); }
    la_sync();
    if (!live) return;
    f32x16 a = {}, c = {};
#pragma unroll
    for (int s = 0; s < DV / 16; s++) {
      la_bf16x8 vf[NP], gf[NP];
      parts<NP>(vr[s], vf); parts<NP>(gw[s], gf);
      a = mm<NP, NP>(vf, gf, a);
      c = mm<NP, NP>(gf, vf, c);
    }
#pragma unroll
    for (int s = 0; s < 2; s++) { kr[s] = k.col(16 * s, col, h5); qr[s] = q.col(16 * s, col, h5); }
    masked<PP>(a, pw, col, h5, true, p.scale, dpt);
    masked<PP>(c, pw, col, h5, false, p.scale, dp);
    a = {};
#pragma unroll
    for (int s = 0; s < DK / 16; s++) {
      la_bf16x8 kf[NP], qf[NP];
      parts<NP>(kw[s], kf); parts<NP>(qw[s], qf);
      a = mm<NP, NP>(qf, kf, a);
    }
    masked<PP>(a, pw, col, h5, false, p.scale, pp);
  }
#pragma unroll
  for (int s = 0; s < 2; s++) gr[s] = go.col(16 * s, col, h5);
  const float* S = p.s_in ? p.s_in + (int64_t)pair * p.dk * p.dv : nullptr;
  const float* R = p.ds_out ? p.ds_out + (int64_t)pair * p.dk * p.dv : nullptr;
  const float later = col < n ? pw[32 + n - 1 - col] : 0.f;   // lambda^(n - 1 - j) of this lane's token
#pragma unroll 1
  for (int d0 = 0; d0 < p.dk; d0 += 32) {
    int at = col;
    reload(at);
    f32x16 aq = {}, ak = {};
    if (S) {
#pragma unroll
      for (int s = 0; s < DV / 16; s++) {
        la_bf16x8 sf[PP], gf[NP];
        split<PP>(mat_row8(S, d0 + at, p.dk, 16 * s + 8 * h5, p.dv), sf);
        parts<NP>(go.row(at, 16 * s + 8 * h5), gf);
        aq = mm<PP, NP>(sf, gf, aq);
      }
      const float w = pw[33 + col] * p.scale;
#pragma unroll
      for (int r = 0; r < 16; r++) aq[r] *= w;
    }
    if (R) {
#pragma unroll
      for (int s = 0; s < DV / 16; s++) {
        la_bf16x8 rf[PP], vf[NP];
        split<PP>(mat_row8(R, d0 + at, p.dk, 16 * s + 8 * h5, p.dv), rf);
        parts<NP>(v.row(at, 16 * s + 8 * h5), vf);
        ak = mm<PP, NP>(rf, vf, ak);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) ak[r] *= later;
    }
    Poison<false> badk;
    Poison<true> badq;
#pragma unroll
    for (int s = 0; s < 2; s++) {
      f32x8_t x = kr[s], y = qr[s];
      badk.take(x, 16 * s, h5); badq.take(y, 16 * s, h5);
      la_bf16x8 f[NP];
      split<NP>(x, f);
      aq = mm<NP, PP>(f, dpt[s], aq);
      split<NP>(y, f);
      ak = mm<NP, PP>(f, dp[s], ak);
    }
    if (d0 + 32 < p.dk)
#pragma unroll
      for (int s = 0; s < 2; s++) { kr[s] = k.col(16 * s, d0 + 32 + at, h5); qr[s] = q.col(16 * s, d0 + 32 + at, h5); }
    badk.give(aq, col, h5); badq.give(ak, col, h5);
    store_rows<T>(aq, (T*)p.dq.ptr + b * p.dq.sb + hd * p.dq.sh, (int)p.dq.st, col, h5, n, p.T, d0, p.dk, VEC);
    store_rows<T>(ak, (T*)p.dk_.ptr + b * p.dk_.sb + hd * p.dk_.sh, (int)p.dk_.st, col, h5, n, p.T, d0, p.dk, VEC);
  }
#pragma unroll 1
  for (int e0 = 0; e0 < p.dv; e0 += 32) {
    int at = col;
    reload(at);
    f32x16 av = {};
    if (R) {
#pragma unroll
      for (int s = 0; s < DK / 16; s++) {
        la_bf16x8 rf[PP], kf[NP];
        split<PP>(mat_cols8(R, 16 * s + 8 * h5, p.dk, e0 + at, p.dv), rf);
        parts<NP>(k.row(at, 16 * s + 8 * h5), kf);
        av = mm<PP, NP>(rf, kf, av);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) av[r] *= later;
    }
    Poison<true> bad;
#pragma unroll
    for (int s = 0; s < 2; s++) {
      f32x8_t x = gr[s];
      bad.take(x, 16 * s, h5);
      la_bf16x8 f[NP];
      split<NP>(x, f);
      av = mm<NP, PP>(f, pp[s], av);
    }
    if (e0 + 32 < p.dv)
#pragma unroll
      for (int s = 0; s < 2; s++) gr[s] = go.col(16 * s, e0 + 32 + at, h5);
    bad.give(av, col, h5);
    store_rows<T>(av, (T*)p.dv_.ptr + b * p.dv_.sb + hd * p.dv_.sh, (int)p.dv_.st, col, h5, n, p.T, e0, p.dv, VEC);
  }
  if (p.ds_in) {
    const float dec = decay_pair(g, n).hi;
    for (int d0 = 0; d0 < p.dk; d0 += 32)
      for (int e0 = 0; e0 < p.dv; e0 += 32)
        short_state<T, VEC, NP>(q, go, R, p.ds_in + (int64_t)pair * p.dk * p.dv, pw, dec, true, p.scale, d0, e0, col, h5);
  }
}

// One token: the state is read and written once, which is all the time there is (256 sequences of 16 heads, 128 / 128: 104 us for 541 MB, 5.2 TB/s, the rate of a
// copy; one sequence of 8 heads, 64 / 64: 4.6 us, a launch).  A workgroup owns `tile` columns of one sequence and head; thread (r, c) the rows r, r + rows, ... of
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

// Segments of a sequence: enough workgroups (of one wave per 32 value columns) for two waves on each of the chip's 1024 SIMDs, segments of at least 128
// tokens.  Kernels of a forward pass with as many, twice as many, half as many, bf16: B 1, T 65536, H 8, 128 / 128: 258, 279, 284 us; B 8, T 4096, H 16, 64 / 64:
// 91, 116, 120 us; forward and backward of B 2, T 8192, H 16, 128 / 128: 454, 519, 457 us.  (More of them: more states written and read; fewer: one wave a SIMD.)
struct Split { int nseg, tokens; };
Split make_split(int B, int T, int H, int dv) {
  const int chunks = (T + CW - 1) / CW, waves = dv <= 32 ? 1 : dv <= 64 ? 2 : 4;
  const int64_t pairs = (int64_t)B * H, want = (2048 / waves + pairs - 1) / pairs;
  int n = (int)(want < chunks / 2 ? want : chunks / 2);
  if (n <= 1) return {1, T};
  const int per = (chunks + n - 1) / n;
  return {(chunks + per - 1) / per, per * CW};
}
size_t seg_floats(int B, int T, int H, int dk, int dv) {
  if (B <= 0 || T <= C) return 0;
  const int n = make_split(B, T, H, dk > dv ? dk : dv).nseg;
  return n > 1 ? (size_t)B * H * n * dk * dv : 0;
}
// Few small states in front of a segment are joined by every workgroup for itself (one launch less), more of them once for all: at most this many floats are read
// by the last one.  The main sweep alone or with the joining kernel: B 6, T 1531, H 6, 48 / 80 fp32, 12 segments, 46000 floats: 34.9 us or 30.1 + 6.7; B 8, T 4096,
// H 16, 64 / 64, 32768 floats: 63.1 or 57.2 + 8.8; training at B 2, T 8192, H 16, 128 / 128, 262000 floats: 660 or 335 + 34.
constexpr int JOIN_BY_KERNEL = 65536;

// Rows that can be moved 16 bytes at a time, of tokens that do not overlap, and whose chunk spans less than 2^29 bytes.  (Other tensors take the one kernel
// that is built for them: 128 / 128, channel by channel.  Its price, forward and backward, fp32: B 2, T 4096, H 8, 12 / 12: 125 and 329 us, where 16 / 16 take 36 and 80; 100 /
// 100: 145 and 331, 104 / 104: 105 and 243; B 2048, T 24, H 4, 12 / 12: 165 and 339, 16 / 16: 19 and 71; 100 / 100: 383 and 865, 104 / 104: 87 and 267.)
bool vec_ok(const sfSeq& t, int d, int bytes) {
  const int per = 16 / bytes;
  return ((uintptr_t)t.ptr & 15) == 0 && d % 8 == 0 && t.sb % per == 0 && t.st % per == 0 && t.sh % per == 0 && t.st >= d && t.st < (1 << 29) / bytes / CW - 128;
}

template <typename T, int DK, int DV, bool VEC, bool STATES> int launch_chunks(const Sweeps& w, hipStream_t st) {
  const Sweep& p = w.s[0];
  const int pieces = p.B * p.H * (STATES && !p.s_out ? p.nseg - 1 : p.nseg);
  hipLaunchKernelGGL((la_chunk_kernel<T, DK, DV, VEC, STATES>), dim3((unsigned)((pieces + 7) / 8 * 8 * w.n)), dim3(DV * 2), (chunk_lds<T, DK, DV, STATES>()), st, w);
  SF_CHECK_LAUNCH("sf_linear_attention");
  return 0;
}
template <int DK, int DV, bool STATES> int launch_wide(const Sweeps& w, hipStream_t st) {
  const Sweep& p = w.s[0];
  const int pieces = p.B * p.H * (STATES && !p.s_out ? p.nseg - 1 : p.nseg);
  const dim3 grid((unsigned)((pieces + 7) / 8 * 8 * w.n)), block(DV * 2);
  bool state = false;
  for (int i = 0; i < w.n; i++) state |= w.s[i].s_out && p.nseg == 1;
  if (STATES) hipLaunchKernelGGL((la_wide_kernel<DK, DV, WIDE_STATES>), grid, block, (wide_lds<DK, DV, true>()), st, w);
  else if (state) hipLaunchKernelGGL((la_wide_kernel<DK, DV, WIDE_SWEEP_STATE>), grid, block, (wide_lds<DK, DV, false>()), st, w);
  else hipLaunchKernelGGL((la_wide_kernel<DK, DV, WIDE_SWEEP>), grid, block, (wide_lds<DK, DV, false>()), st, w);
  SF_CHECK_LAUNCH("sf_linear_attention");
  return 0;
}
int width_of(int d) { return d <= 32 ? 0 : d <= 64 ? 1 : 2; }

// The wide kernel wins wherever it applies, bf16 tensors with both widths above 32.  The main sweep there and with chunks of 32 tokens instead: B 1, T 65536, H 8,
// 128 / 128: 161 and 183 us (with its gradients at B 2, T 8192, H 16: 334 and 383); B 8, T 4096, H 16, 64 / 64: 63.1 and 65.5; B 3, T 777, H 5, 40 / 72: 14.5 and
// 19.2, its dv (72 / 40): 27.7 and 30.4.
template <typename T, bool STATES> int chunks_of(const Sweeps& w, bool vec, hipStream_t st) {
  if (w.n == 0) return 0;
  const Sweep& p = w.s[0];
  const int a = width_of(p.dk), b = width_of(p.dv);
  if (!vec) return launch_chunks<T, 128, 128, false, STATES>(w, st);
  switch (a * 3 + b) {
    case 0: return launch_chunks<T, 32, 32, true, STATES>(w, st);
    case 1: return launch_chunks<T, 32, 64, true, STATES>(w, st);
    case 2: return launch_chunks<T, 32, 128, true, STATES>(w, st);
    case 3: return launch_chunks<T, 64, 32, true, STATES>(w, st);
    case 6: return launch_chunks<T, 128, 32, true, STATES>(w, st);
    default: break;
  }
  if constexpr (sizeof(T) == 2) {
    if (b == 1) return a == 1 ? launch_wide<64, 64, STATES>(w, st) : launch_wide<128, 64, STATES>(w, st);
    return a == 1 ? launch_wide<64, 128, STATES>(w, st) : launch_wide<128, 128, STATES>(w, st);
  } else {
    if (b == 1) return a == 1 ? launch_chunks<T, 64, 64, true, STATES>(w, st) : launch_chunks<T, 128, 64, true, STATES>(w, st);
    return a == 1 ? launch_chunks<T, 64, 128, true, STATES>(w, st) : launch_chunks<T, 128, 128, true, STATES>(w, st);
  }
}

// The states between the segments of a sweep, in its own orientation.
template <typename T> int states_of(const Sweep& p, bool vec, hipStream_t st) {
  if (p.nseg < 2) return 0;
  Sweeps w = {{p}, 1};
  if (int rc = chunks_of<T, true>(w, vec, st)) return rc;
  if (!p.joined) return 0;
  hipLaunchKernelGGL(la_join_kernel, dim3((unsigned)(p.B * p.H), (p.dk * p.dv + 255) / 256), dim3(256), 0, st, p);
  SF_CHECK_LAUNCH("sf_linear_attention");
  return 0;
}

template <typename T> int forward_of(const Sweep& p, hipStream_t st) {
  const int by = sizeof(T);
  const bool vec = vec_ok(p.q, p.dk, by) && vec_ok(p.k, p.dk, by) && vec_ok(p.v, p.dv, by) && vec_ok(p.o, p.dv, by);
  if (int rc = states_of<T>(p, vec, st)) return rc;
  Sweeps w = {{p}, 1};
  return chunks_of<T, false>(w, vec, st);
}

// fwd: the sweep of the forward pass; seg its states (computed here unless `have`), rseg the gradients' ones.
template <typename T>
int backward_of(const Sweep& fwd, const sfSeq& go, const sfSeq& dq, const sfSeq& dk, const sfSeq& dv, const float* ds_out, float* ds_in, float* rseg, bool have, hipStream_t st) {
  const int by = sizeof(T);
  const bool vec = vec_ok(fwd.q, fwd.dk, by) && vec_ok(fwd.k, fwd.dk, by) && vec_ok(fwd.v, fwd.dv, by) && vec_ok(go, fwd.dv, by) && vec_ok(dq, fwd.dk, by) &&
                   vec_ok(dk, fwd.dk, by) && vec_ok(dv, fwd.dv, by);
  if (!have)
    if (int rc = states_of<T>(fwd, vec, st)) return rc;
  // dv: state R, read by k, written q (x) do; lambda times its last state is the gradient of s_in
  Sweep pv = fwd;
  pv.q = fwd.k; pv.k = fwd.q; pv.v = go; pv.o = dv; pv.s_in = ds_out; pv.s_out = ds_in; pv.seg = rseg;
  pv.kscale = fwd.oscale; pv.oscale = 1.f; pv.reverse = pv.plain_init = pv.decay_out = 1;
  if (int rc = states_of<T>(pv, vec, st)) return rc;
  // dk: state R^T, read by v, written do (x) q
  Sweep pk = pv;
  pk.q = fwd.v; pk.k = go; pk.v = fwd.q; pk.o = dk; pk.dk = fwd.dv; pk.dv = fwd.dk; pk.in_d = 1; pk.in_e = fwd.dv; pk.s_out = nullptr; pk.decay_out = 0;
  // dq: state S^T, read by do, written v (x) k
  Sweep pq = fwd;
  pq.q = go; pq.k = fwd.v; pq.v = fwd.k; pq.o = dq; pq.dk = fwd.dv; pq.dv = fwd.dk; pq.in_d = 1; pq.in_e = fwd.dv; pq.s_out = nullptr;
  if (!vec || width_of(fwd.dk) == width_of(fwd.dv)) {
    Sweeps w = {{pq, pk, pv}, 3};
    return chunks_of<T, false>(w, vec, st);
  }
  Sweeps w = {{pq, pk}, 2}, x = {{pv}, 1};
  if (int rc = chunks_of<T, false>(w, vec, st)) return rc;
  return chunks_of<T, false>(x, vec, st);
}

// (32-bit byte offsets over C tokens)
bool short_ok(const sfSeq& t) { return t.st >= 0 && t.st < (1 << 25) - 4; }

template <typename T, bool BWD> int short_of(Short& p, hipStream_t st) {
  const int by = sizeof(T), a = width_of(p.dk), b = width_of(p.dv);
  const bool vec = vec_ok(p.q, p.dk, by) && vec_ok(p.k, p.dk, by) && vec_ok(p.v, p.dv, by) &&
                   (BWD ? vec_ok(p.dout, p.dv, by) && vec_ok(p.dq, p.dk, by) && vec_ok(p.dk_, p.dk, by) && vec_ok(p.dv_, p.dv, by) : vec_ok(p.o, p.dv, by));
  const dim3 grid((unsigned)(((int64_t)p.B * p.H + 3) / 4));
#define SF_LA_SHORT(DK, DV, VEC)                                                                             \
  do {                                                                                                       \
    if (BWD) hipLaunchKernelGGL((la_short_bwd_kernel<T, DK, DV, VEC>), grid, dim3(256), 0, st, p);           \
    else hipLaunchKernelGGL((la_short_fwd_kernel<T, DK, DV, VEC>), grid, dim3(256), 0, st, p);               \
  } while (0)
  if (!vec) SF_LA_SHORT(128, 128, false);
  else switch (a * 3 + b) {
    case 0: SF_LA_SHORT(32, 32, true); break;
    case 1: SF_LA_SHORT(32, 64, true); break;
    case 2: SF_LA_SHORT(32, 128, true); break;
    case 3: SF_LA_SHORT(64, 32, true); break;
    case 4: SF_LA_SHORT(64, 64, true); break;
    case 5: SF_LA_SHORT(64, 128, true); break;
    case 6: SF_LA_SHORT(128, 32, true); break;
    case 7: SF_LA_SHORT(128, 64, true); break;
    default: SF_LA_SHORT(128, 128, true); break;
  }
#undef SF_LA_SHORT
  SF_CHECK_LAUNCH("sf_linear_attention");
  return 0;
}
template <bool BWD> int run_short(Short& p, int dtype, hipStream_t st) { return dtype == SF_BF16 ? short_of<__bf16, BWD>(p, st) : short_of<float, BWD>(p, st); }

Sweep make_sweep(const sfSeq& q, const sfSeq& k, const sfSeq& v, const float* g, const float* s_in, const int32_t* lengths, int B, int T, int H, int dk, int dv,
                 float scale, void* seg) {
  Sweep p = {};
  p.q = q; p.k = k; p.v = v; p.g = g; p.s_in = s_in; p.in_d = dv; p.in_e = 1; p.lengths = lengths; p.B = B; p.T = T; p.H = H; p.dk = dk; p.dv = dv;
  p.kscale = 1.f; p.oscale = scale; p.seg = (float*)seg;
  const Split sp = make_split(B, T, H, dk > dv ? dk : dv);
  p.nseg = sp.nseg; p.seg_tokens = sp.tokens; p.joined = sp.nseg * dk * dv > JOIN_BY_KERNEL;
  return p;
}

int check_dims(const char* name, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, int32_t dtype) {
  SF_REQUIRE(B >= 0 && T >= 0 && H > 0, "%s: B %d, T %d, H %d", name, B, T, H);
  SF_REQUIRE(dk >= 1 && dk <= 128 && dv >= 1 && dv <= 128, "%s: head widths %d / %d (1 .. 128)", name, dk, dv);
  SF_REQUIRE(dtype == SF_F32 || dtype == SF_BF16, "%s: unsupported storage type %d", name, dtype);
  SF_REQUIRE((int64_t)T + 64 < 0x7fffffff, "%s: T %d", name, T);
  SF_REQUIRE((int64_t)B * H <= 1 << 22, "%s: %d sequences of %d heads (at most 2^22 together)", name, B, H);
  return 0;
}

}  // namespace

extern "C" {

size_t sf_linear_attention_workspace_bytes(int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, int32_t pass) {
  if (B <= 0 || T <= 0 || H <= 0 || dk <= 0 || dv <= 0) return 0;
  return seg_floats(B, T, H, dk, dv) * sizeof(float) * (pass == 2 ? 2 : 1);
}

int sf_linear_attention_fwd(sfSeq q, sfSeq k, sfSeq v, sfSeq o, const float* log_decay, const float* s_in, float* s_out, const int32_t* lengths, int32_t B,
                            int32_t T, int32_t H, int32_t dk, int32_t dv, float scale, int32_t dtype, void* workspace, size_t workspace_bytes,
                            sfStream stream) {
  const char* name = "sf_linear_attention_fwd";
  if (int rc = check_dims(name, B, T, H, dk, dv, dtype)) return rc;
  SF_REQUIRE(log_decay != nullptr && (T == 0 || B == 0 || (q.ptr && k.ptr && v.ptr && o.ptr)), "%s: missing tensor", name);
  SF_REQUIRE(workspace_bytes >= sf_linear_attention_workspace_bytes(B, T, H, dk, dv, 0), "%s: workspace too small", name);
  SF_REQUIRE(workspace_bytes == 0 || workspace != nullptr, "%s: no workspace", name);
  if (B == 0) return 0;
  if (T > 0 && T <= C && short_ok(q) && short_ok(k) && short_ok(v) && short_ok(o)) {
    Short p = {};
    p.q = q; p.k = k; p.v = v; p.o = o; p.g = log_decay; p.s_in = s_in; p.s_out = s_out; p.lengths = lengths;
    p.B = B; p.T = T; p.H = H; p.dk = dk; p.dv = dv; p.scale = scale;
    return run_short<false>(p, dtype, (hipStream_t)stream);
  }
  Sweep p = make_sweep(q, k, v, log_decay, s_in, lengths, B, T, H, dk, dv, scale, workspace);
  p.o = o; p.s_out = s_out;
  return dtype == SF_BF16 ? forward_of<__bf16>(p, (hipStream_t)stream) : forward_of<float>(p, (hipStream_t)stream);
}

int sf_linear_attention_bwd(sfSeq q, sfSeq k, sfSeq v, sfSeq dout, const float* log_decay, const float* s_in, const float* ds_out, const int32_t* lengths,
                            const void* states, sfSeq dq, sfSeq dk_out, sfSeq dv_out, float* ds_in, int32_t B, int32_t T, int32_t H, int32_t dk, int32_t dv, float scale,
                            int32_t dtype, void* workspace, size_t workspace_bytes, sfStream stream) {
  const char* name = "sf_linear_attention_bwd";
  if (int rc = check_dims(name, B, T, H, dk, dv, dtype)) return rc;
  SF_REQUIRE(log_decay != nullptr && (T == 0 || B == 0 || (q.ptr && k.ptr && v.ptr && dout.ptr && dq.ptr && dk_out.ptr && dv_out.ptr)), "%s: missing tensor", name);
  SF_REQUIRE(workspace_bytes >= sf_linear_attention_workspace_bytes(B, T, H, dk, dv, states ? 1 : 2), "%s: workspace too small", name);
  SF_REQUIRE(workspace_bytes == 0 || workspace != nullptr, "%s: no workspace", name);
  if (B == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  if (T > 0 && T <= C && short_ok(q) && short_ok(k) && short_ok(v) && short_ok(dout) && short_ok(dq) && short_ok(dk_out) && short_ok(dv_out)) {
    Short p = {};
    p.q = q; p.k = k; p.v = v; p.dout = dout; p.dq = dq; p.dk_ = dk_out; p.dv_ = dv_out; p.g = log_decay; p.s_in = s_in; p.ds_out = ds_out; p.ds_in = ds_in;
    p.lengths = lengths; p.B = B; p.T = T; p.H = H; p.dk = dk; p.dv = dv; p.scale = scale;
    return run_short<true>(p, dtype, st);
  }
  float* mine = (float*)workspace;
  const Sweep p = make_sweep(q, k, v, log_decay, s_in, lengths, B, T, H, dk, dv, scale, states ? const_cast<void*>(states) : mine + seg_floats(B, T, H, dk, dv));
  return dtype == SF_BF16 ? backward_of<__bf16>(p, dout, dq, dk_out, dv_out, ds_out, ds_in, mine, states != nullptr, st)
                          : backward_of<float>(p, dout, dq, dk_out, dv_out, ds_out, ds_in, mine, states != nullptr, st);
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
