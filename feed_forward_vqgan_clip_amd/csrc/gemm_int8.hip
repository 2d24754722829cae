// gemm_int8.hip — Linear in 8-bit integers with one scale per token (row of x) and one per channel (row of w):
//
//     xs[m] = max_k |x[m, k]| / 127 (fp32)        xq[m, k] = round-half-even(x[m, k] / xs[m])        (the weight's rows likewise, once)
//     y[m, n] = act(xs[m] * ws[n] * sum_k xq[m, k] wq[n, k] + bias[n]) + residual[m, n]
//
// The integer sum is exact (32-bit accumulators, |sum| <= 127^2 K < 2^31 for K <= 131072), so the quantisation is the only approximation
// and the result does not depend on how K is cut.  Rounding to 8 bits follows the definition exactly: the quotient is formed with a
// reciprocal, then corrected with one fused residual (x - q xs is exact in fp32 once q is within one step of x / xs).
// A row of zeros has scale 0 and stays 0; a row that holds an inf or a NaN gets scale NaN, so its outputs are NaN and nothing is hidden.
#include <type_traits>

#include "common.h"

#pragma clang fp contract(off)      // a product and a sum fuse only where fmaf says so: the kernels below agree bit for bit on a row's outputs

namespace {

typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef __attribute__((address_space(3))) void* lds_vp;
typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(16))) int i32x16_t;
constexpr uint32_t OOB = 0xFFFFFFF0u;

// 64 lanes x 16 bytes from a bounded buffer into consecutive LDS; `soff` is wave-uniform and not part of the range check
__device__ __forceinline__ void dma16(rsrc_t r, uint32_t off, int soff, unsigned char* lds) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_vp)lds, 16, off, soff, 0, 0);
}

__device__ __forceinline__ float row_scale(float amax) {           // amax >= 0, or NaN
  return amax <= 3.4028235e38f ? amax / 127.0f : __uint_as_float(0x7fc00000u);
}
__device__ __forceinline__ float amax_with_nan(float m, float v) {  // fmaxf drops a NaN: keep it
  const float a = fabsf(v);
  return a > m || a != a ? a : m;
}
// One row's scale, ready to divide by: rows whose 1 / s would overflow are lifted by a power of two first (exact).  Such a scale may itself be
// subnormal, and so a coarse amax / 127: only there can a quotient pass 127.
struct RowQuant {
  float s, inv, up;
  __device__ __forceinline__ RowQuant(float scale) {
    up = scale < 0x1p-100f ? 0x1p100f : 1.0f;
    s = scale * up;
    inv = s > 0.0f ? 1.0f / s : 0.0f;                               // 0: a row of zeros or one with a NaN / inf, stored as zeros
  }
};
__device__ __forceinline__ uint32_t pack_i8(int a, int b, int c, int d) {
  const uint32_t lo = __builtin_amdgcn_perm((uint32_t)b, (uint32_t)a, 0x0c0c0400u), hi = __builtin_amdgcn_perm((uint32_t)d, (uint32_t)c, 0x04000c0cu);
  return lo | hi;
}
// round-half-even(x / s) of eight values.  x * inv is within 127 * 2^-23 of the quotient (two roundings of at most half a unit each), so its
// rounding is right unless it lies within 2^-15 of a border; then (3 % of the waves) the remainder x - q s, which one fma gives exactly,
// decides, a remainder of exactly half a step going to the even neighbour.
__device__ __forceinline__ u32x2_t quant8(const f32x8& v, const RowQuant& r) {
  float x[8], q[8];
  float far = 0.0f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    x[j] = r.inv > 0.0f ? v.v[j] * r.up : 0.0f;
    const float f = x[j] * r.inv;
    q[j] = rintf(f);
    far = fmaxf(far, fabsf(f - q[j]));
  }
  if (__any(far > 0.5f - 0x1p-15f)) {
    const float half = 0.5f * r.s;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float d = fmaf(-q[j], r.s, x[j]);
      const bool odd = ((int)q[j] & 1) != 0;
      if (fabsf(d) > half || (odd && fabsf(d) == half)) q[j] += d > 0.0f ? 1.0f : -1.0f;
    }
  }
  int i[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) i[j] = (int)q[j];
  if (r.up != 1.0f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) i[j] = min(max(i[j], -127), 127);
  }
  u32x2_t o;
  o[0] = pack_i8(i[0], i[1], i[2], i[3]);
  o[1] = pack_i8(i[4], i[5], i[6], i[7]);
  return o;
}

// wave maximum that keeps a NaN
__device__ __forceinline__ float wave_amax(float m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = amax_with_nan(m, __shfl_xor(m, o, 64));
  return m;
}

// Where the quantised value (row, k) goes: rows of ldq bytes, or (ldq 0) panels of 64 consecutive k, [ceil(K / 64)][rows][64], the last one
// filled up with zeros.  In panels the 64-byte pieces of neighbouring rows share a cache line, so a K step of the product reads whole lines.
__device__ __forceinline__ int8_t* q_at(int8_t* q, int64_t ldq, int64_t rows, int64_t row, int k) {
  return ldq ? q + row * ldq + k : q + ((int64_t)(k >> 6) * rows + row) * 64 + (k & 63);
}

// One wave per row; a row of up to 64 * 8 * CH values stays in registers between the two passes, longer ones are read again (from L2).
// Bound by bytes: 16448 rows of 4096 bf16 in 45 us (202 MB, 4.5 TB/s; 56 us with a branch around each load), of 1024 in 13.
template <typename T, int CH>
__global__ __launch_bounds__(256) void int8_quant_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                         float* __restrict__ scale, int64_t rows, int K) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const T* xr = x + row * ldx;
  const int Kq = ldq ? K : (K + 63) & ~63;
  f32x8 v[CH];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int k = (i * 64 + lane) * 8;
    v[i] = load8(xr + (k < K ? k : 0));                       // (no branch: all loads under way at once)
  }
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const bool in = (i * 64 + lane) * 8 < K;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[i].v[j] = in ? v[i].v[j] : 0.0f;
      m = amax_with_nan(m, v[i].v[j]);
    }
  }
  for (int k = (CH * 64 + lane) * 8; k < K; k += 512) {
    const f32x8 t = load8(xr + k);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = amax_with_nan(m, t.v[j]);
  }
  const float s = row_scale(wave_amax(m));
  const RowQuant rq(s);
  if (lane == 0) scale[row] = s;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int k = (i * 64 + lane) * 8;
    if (k < Kq) *(u32x2_t*)q_at(q, ldq, rows, row, k) = quant8(v[i], rq);
  }
  for (int k = (CH * 64 + lane) * 8; k < Kq; k += 512) {
    u32x2_t o = {0u, 0u};
    if (k < K) o = quant8(load8(xr + k), rq);
    *(u32x2_t*)q_at(q, ldq, rows, row, k) = o;
  }
}

// ---- epilogue ----------------------------------------------------------------------------------------------------------------------
// The activation (and its derivative); 16-bit outputs take the hardware exp / rcp forms (errors ~2^-22; erf after Abramowitz & Stegun 7.1.26,
// 1.5e-7), fp32 outputs the accurate ones.
template <bool FAST, int ACT, bool GRAD>
__device__ __forceinline__ void activate(float z, float& y, float& g) {
  if constexpr (ACT == FFVC_ACT_GELU) {
    if constexpr (FAST) {
      const float u = fabsf(z) * 0.70710678118654752440f;
      const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, u, 1.0f));
      const float e = __builtin_amdgcn_exp2f(-1.44269504088896341f * (u * u));
      const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
      const float cdf = fmaf(copysignf(0.5f, z), fmaf(-q, e, 1.0f), 0.5f);
      y = z * cdf;
      if constexpr (GRAD) g = fmaf(z * 0.39894228040143267794f, e, cdf);
    } else {
      y = act_gelu(z);
      if constexpr (GRAD) g = act_gelu_grad(z);
    }
  } else if constexpr (ACT == FFVC_ACT_QUICKGELU) {
    const float s = FAST ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.45546696f * z)) : 1.0f / (1.0f + expf(-1.702f * z));
    y = z * s;
    if constexpr (GRAD) g = s * (1.0f + 1.702f * z * (1.0f - s));
  } else {
    y = z;
    g = 1.0f;
  }
}
template <bool FAST, bool GRAD>
__device__ __forceinline__ void activate_by(int act, float z, float& y, float& g) {
  if (act == FFVC_ACT_GELU)
    activate<FAST, FFVC_ACT_GELU, GRAD>(z, y, g);
  else if (act == FFVC_ACT_QUICKGELU)
    activate<FAST, FFVC_ACT_QUICKGELU, GRAD>(z, y, g);
  else
    activate<FAST, FFVC_ACT_NONE, GRAD>(z, y, g);
}

struct I8Args {
  const int8_t* x;
  const int8_t* w;
  const float* xs;
  const float* ws;
  const float* bias;
  const void* res;
  void* y;
  void* aux;              // act'(pre-activation), may be null
  int64_t xrows;          // rows of a panel of x (quantised), or the row stride of 16-bit x (linear_int8_few)
  int64_t ldw, ldy, ldr;
  int M, N, K;
  int act;
  int res_f32;
  int vec;                // rows of y / res / aux take 16-byte accesses and N % 8 == 0
};

// one output from its row-scaled sum (v = sum * xs[m]); every kernel of this file takes the same steps, so they agree bit for bit
template <typename L, typename YT>
__device__ __forceinline__ void store_one(const I8Args& p, float v, int64_t m, int n) {
  const float z = fmaf(v, p.ws[n], p.bias ? p.bias[n] : 0.0f);
  float y, g;
  activate_by<sizeof(YT) == 2, true>(p.act, z, y, g);
  if (p.res) y += p.res_f32 ? ((const float*)p.res)[m * p.ldr + n] : ElemTraits<L>::load((const L*)p.res + m * p.ldr + n);
  ElemTraits<YT>::store((YT*)p.y + m * p.ldy + n, y);
  if (p.aux) ElemTraits<L>::store((L*)p.aux + m * p.N + n, g);
}

// ---- the tiled product -----------------------------------------------------------------------------------------------------------------
// BM x 128 outputs per workgroup of four waves ((BM / 2) x 64 each), K steps of 64 bytes.  x comes in panels (see q_at), a step of a tile is one
// contiguous block, three LDS slots; w keeps its rows, two steps (128 bytes, a whole cache line of each row) at a time, two slots.  LDS-DMA
// runs two steps ahead with one barrier per step, the youngest pieces may still be under way.  Two workgroups share a CU (BM = 256: 80 KiB
// each), so the epilogue of one, as long as its K loop where K is 1024 and an activation is due, runs under the products of the other.
// (With 64-byte steps of plain rows every step fetched each line twice: 104 us at 16384 x 4096 x 1024, 96 as it is; 86 at 16384 x 1024 x 4096.)
// What bounds it is the stream from L2 into LDS, about 9.5 TB/s over the chip (137 GOP at 86 us are 0.8 GB): the matrix units are busy half the
// time.  Tiles of 256 x 256, one per CU and two K steps of 128 bytes under way, move two thirds of the bytes at the same rate and cannot run an
// epilogue beside a K loop: 73 us for 16384 x 1024 x 4096, but 119 for 16384 x 4096 x 1024; not kept.
// 16-byte chunks are XOR-swizzled inside 256-byte lines (4 rows of x, 2 of w): the fragment reads hit every bank evenly.
constexpr int BN = 128, BK = 64;

__device__ __forceinline__ u32x4_t frag_x(const unsigned char* tile, int row, int chunk) {        // chunk 0..3
  return *(const u32x4_t*)(tile + row * 64 + ((chunk ^ ((row >> 2) & 3)) << 4));
}
__device__ __forceinline__ u32x4_t frag_w(const unsigned char* tile, int row, int chunk) {        // chunk 0..7
  const int line = row >> 1;
  return *(const u32x4_t*)(tile + line * 256 + (((((row & 1) << 3) | chunk) ^ (line & 15)) << 4));
}

// staging of BM panel rows by four waves: a piece is 16 rows of 64 bytes
template <int ROWS>
struct PanelDma {
  static constexpr int NP = ROWS / 64;
  const int8_t* base;
  int64_t panel;
  uint32_t off[NP];
  int bytes;
  __device__ __forceinline__ void init(const int8_t* x, int64_t xrows, int row0, int rows, int wave, int lane) {
    const int live = rows - row0 < ROWS ? rows - row0 : ROWS;
    base = x + (int64_t)row0 * 64;
    panel = xrows * 64;
    bytes = live * 64;                                       // rows past the end read as zeros
    const int chunk = (lane & 3) ^ ((lane >> 4) & 3);
#pragma unroll
    for (int i = 0; i < NP; ++i) off[i] = ((wave * NP + i) * 16 + (lane >> 2)) * 64 + chunk * 16;
  }
  __device__ __forceinline__ void issue(unsigned char* tile, int kt, int nk, int wave) {      // steps past the last one fetch zeros
    const rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(base + (kt < nk ? kt : 0) * panel), 0, kt < nk ? bytes : 0, 0x00020000);
#pragma unroll
    for (int i = 0; i < NP; ++i) dma16(rs, off[i], 0, tile + (wave * NP + i) * 1024);
  }
};
// staging of 128 rows of w, 128 bytes wide, by four waves: a piece is 8 rows
struct WideDma {
  static constexpr int NP = 4;
  rsrc_t rs;
  uint32_t off[NP];
  int chunk[NP];
  __device__ __forceinline__ void init(const int8_t* w, int64_t ld, int row0, int rows, int K, int wave, int lane) {
    const int live = rows - row0 < BN ? rows - row0 : BN;
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)(w + row0 * ld), 0, (int)((live - 1) * ld + K), 0x00020000);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int line = (wave * NP + i) * 4 + (lane >> 4), cp = (lane & 15) ^ (line & 15);
      const int row = 2 * line + (cp >> 3);
      chunk[i] = (cp & 7) * 16;
      off[i] = row < live ? (uint32_t)(row * ld + chunk[i]) : OOB;
    }
  }
  __device__ __forceinline__ void issue(unsigned char* tile, int k0, int K, int wave) {       // (chunks past K read as zeros)
#pragma unroll
    for (int i = 0; i < NP; ++i) dma16(rs, k0 + chunk[i] < K ? off[i] : OOB, k0 < K ? k0 : 0, tile + (wave * NP + i) * 1024);
  }
};

template <typename L, typename YT, int ACT, int BM>
__global__ __launch_bounds__(256, 2) void gemm_int8_kernel(const I8Args p, int tiles_n) {
  constexpr int MT = BM / 64, XS = BM * BK, WS = BN * 128;
  constexpr int XP = PanelDma<BM>::NP, WP = WideDma::NP;  // LDS-DMA instructions per wave and slot
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  unsigned char* wmem = smem + 3 * XS;
  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  // Consecutive workgroups go to the 8 XCDs in turn: give each XCD a contiguous run of the whole tiles.  The tiles of a last, partly filled row
  // block come after all others, spread over the XCDs: their dead 32-row blocks are skipped, so they are short.
  int tile = blockIdx.x;
  const int whole = (p.M / BM) * tiles_n;
  if (tile < whole) {
    const int q = whole >> 3, r = whole & 7, xcd = tile & 7;
    tile = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (tile >> 3);
  }
  const int tm = tile / tiles_n, tn = tile - tm * tiles_n;
  const int m0 = tm * BM, n0 = tn * BN;
  PanelDma<BM> dx;
  WideDma dw;
  dx.init(p.x, p.xrows, m0, p.M, wave, lane);
  dw.init(p.w, p.ldw, n0, p.N, p.K, wave, lane);
  i32x16_t acc[2][MT];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0;
  const int nk = (p.K + BK - 1) / BK;
  const int live = min(MT, (p.M - m0 - wm * (32 * MT) + 31) / 32);   // 32-row blocks of this wave that hold a row (may be < 1)
  dx.issue(smem, 0, nk, wave);
  dw.issue(wmem, 0, p.K, wave);
  dx.issue(smem + XS, 1, nk, wave);
  auto steps = [&](auto partial) {
    constexpr bool PARTIAL = decltype(partial)::value;
    int cur = 0, nxt = 2;
    auto step = [&](int kt, const unsigned char* sw, int half) {
      const unsigned char* sx = smem + cur * XS;
      u32x4_t fa[2][2], fb[2][MT];                          // the whole step's fragments are requested before its first product
#pragma unroll
      for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int t = 0; t < 2; ++t) fa[s][t] = frag_w(sw, wn * 64 + t * 32 + l31, 4 * half + 2 * s + h);
#pragma unroll
        for (int t = 0; t < MT; ++t) fb[s][t] = frag_x(sx, wm * (32 * MT) + t * 32 + l31, 2 * s + h);
      }
      if constexpr (!PARTIAL) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int b = 0; b < MT; ++b)
          if (!PARTIAL || b < live) {
#pragma unroll
            for (int a = 0; a < 2; ++a)
              acc[a][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4_t, fa[s][a]), __builtin_bit_cast(i32x4_t, fb[s][b]), acc[a][b], 0, 0, 0);
          }
      cur = cur == 2 ? 0 : cur + 1;
      nxt = nxt == 2 ? 0 : nxt + 1;
    };
#pragma unroll 1
    for (int kt = 0; kt < nk; kt += 2) {
      const unsigned char* sw = wmem + ((kt >> 1) & 1) * WS;
      // my pieces of this step have landed (x of the next may be under way), then everyone's; and nobody reads the slots filled next
      // (the bare barrier: __syncthreads would wait for the pieces under way as well)
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(XP) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      dx.issue(smem + nxt * XS, kt + 2, nk, wave);
      dw.issue(wmem + (((kt >> 1) & 1) ^ 1) * WS, (kt + 2) * BK, p.K, wave);
      step(kt, sw, 0);
      asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(XP + WP) : "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      dx.issue(smem + nxt * XS, kt + 3, nk, wave);
      step(kt + 1, sw, 1);                                  // (an odd last step multiplies zeros)
    }
  };
  if (live == MT)
    steps(std::false_type{});
  else
    steps(std::true_type{});
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // the zero pieces of the steps past the end
  __syncthreads();
  // A lane holds 4 neighbouring n of one m: it scales them by its row's xs.  Through an 8 KiB pad of its wave (in the stage memory nobody reads
  // any more) 32 rows x 64 columns at a time leave as 8 outputs per lane, 8 lanes to a row; the lane's columns, and so their scales and
  // biases, stay the same throughout.  Row scales and residuals are requested before they are needed.
  unsigned char* pad = smem + wave * 8192;
  const int c8 = lane & 7, r8 = lane >> 3;
  const int n = n0 + wn * 64 + 8 * c8;
  const int mw = m0 + wm * (32 * MT);
  float xs[MT], ws[8], bias[8];
#pragma unroll
  for (int b = 0; b < MT; ++b) {
    const int m = mw + 32 * b + l31;
    xs[b] = p.xs[m < p.M ? m : p.M - 1];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int nn = n + j < p.N ? n + j : p.N - 1;
    ws[j] = p.ws[nn];
    bias[j] = p.bias ? p.bias[nn] : 0.0f;
  }
#pragma unroll
  for (int b = 0; b < MT; ++b) {
    if (b >= live) break;
    const int mb = mw + 32 * b;
    f32x8 res[4];
    if (p.vec && p.res) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = mb + r8 + 8 * i;
        if (m < p.M && n < p.N) res[i] = p.res_f32 ? load8((const float*)p.res + m * p.ldr + n) : load8((const L*)p.res + m * p.ldr + n);
      }
    }
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)acc[a][b][4 * q + j] * xs[b];
        *(f32x4_t*)(pad + l31 * 256 + (((8 * a + 2 * q + h) ^ (l31 & 15)) << 4)) = v;
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (p.vec) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = r8 + 8 * i, m = mb + row;
        const f32x4_t lo = *(const f32x4_t*)(pad + row * 256 + (((2 * c8) ^ (row & 15)) << 4));
        const f32x4_t hi = *(const f32x4_t*)(pad + row * 256 + (((2 * c8 + 1) ^ (row & 15)) << 4));
        if (m < p.M && n < p.N) {
          constexpr bool FAST = sizeof(YT) == 2;
          f32x8 o, g;
          if (p.aux) {
#pragma unroll
            for (int j = 0; j < 8; ++j) activate<FAST, ACT, true>(fmaf(j < 4 ? lo[j & 3] : hi[j & 3], ws[j], bias[j]), o.v[j], g.v[j]);
            store8((L*)p.aux + (int64_t)m * p.N + n, g);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) activate<FAST, ACT, false>(fmaf(j < 4 ? lo[j & 3] : hi[j & 3], ws[j], bias[j]), o.v[j], g.v[j]);
          }
          if (p.res) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o.v[j] += res[i].v[j];
          }
          store8((YT*)p.y + m * p.ldy + n, o);
        }
      }
    } else {
#pragma unroll 1
      for (int x = lane; x < 32 * 64; x += 64) {             // odd widths or unaligned rows: one output at a time
        const int row = x >> 6, col = x & 63;
        const int m = mb + row, nn = n0 + wn * 64 + col;
        const float v = *(const float*)(pad + row * 256 + (((col >> 2) ^ (row & 15)) << 4) + (col & 3) * 4);
        if (m < p.M && nn < p.N) store_one<L, YT>(p, v, m, nn);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// ---- few outputs ------------------------------------------------------------------------------------------------------------------------------
// A workgroup owns 16 rows x 16 columns, its eight waves take pairs of K panels (a 128-byte line of every weight row) in turn, operands straight
// from global memory (a lane reads the 16 bytes of its row that its MFMA needs); the partial sums meet in LDS, exactly.  Where tiles would be few
// they walk K alone, one after the other's latency: 64 x 1024 x 4096 takes 19.3 us in tiles, 4.9 here (22 with 64 x 32 outputs per workgroup: it is
// bound by the loads a CU can have under way, so by the CUs that it reaches).
// Measured, us in tiles / here: 256 x 2048 x 512 6.6 / 5.9, 384 x 2048 x 512 6.6 / 7.5, 128 x 4096 x 1024 8.7 / 8.5, 192 x 4096 x 1024 8.8 / 11.1,
// 384 x 1024 x 4096 20.1 / 18.4: up to eight workgroups per CU.
inline bool few_outputs(int64_t M, int64_t N) { return (M + 15) / 16 * ((N + 15) / 16) <= 2048; }

template <typename L, typename YT>
__global__ __launch_bounds__(512) void gemm_int8_skinny_kernel(const I8Args p) {
  __shared__ int part[8][4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16;
  const int8_t* wr = p.w + (int64_t)(n0 + l15 < p.N ? n0 + l15 : p.N - 1) * p.ldw;
  const int8_t* xr = p.x + (m0 + l15 < p.M ? m0 + l15 : p.M - 1) * 64;      // (rows past the last give outputs that nobody stores)
  const int64_t panel = p.xrows * 64;
  i32x4_t acc = {0, 0, 0, 0};
  const u32x4_t z = {0u, 0u, 0u, 0u};
#pragma unroll 4
  for (int k0 = wave * 128; k0 < p.K; k0 += 1024) {
    u32x4_t a[2], b[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int kk = k0 + 64 * s + 16 * q, kc = kk < p.K ? kk : k0;         // K % 16 == 0: a 16-byte chunk is inside or outside (then zeros of w)
      a[s] = *(const u32x4_t*)(wr + kc);
      b[s] = *(const u32x4_t*)(xr + (kc >> 6) * panel + (kc & 63));
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, k0 + 64 * s + 16 * q < p.K ? a[s] : z), __builtin_bit_cast(i32x4_t, b[s]), acc, 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[wave][i][lane] = acc[i];
  __syncthreads();
  if (tid < 256) {
    const int col = tid & 15, row = tid >> 4;                 // consecutive lanes -> consecutive columns
    const int reg = col & 3, ln = 16 * (col >> 2) + row;      // where the product's (column, row) sits
    int sum = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) sum += part[w][reg][ln];
    const int m = m0 + row;
    if (m < p.M && n0 + col < p.N) store_one<L, YT>(p, (float)sum * p.xs[m], m, n0 + col);
  }
}

template <typename L, typename YT>
int launch_skinny(const I8Args& p, hipStream_t st) {
  hipLaunchKernelGGL((gemm_int8_skinny_kernel<L, YT>), dim3(ceil_div(p.N, 16), ceil_div(p.M, 16)), dim3(512), 0, st, p);
  FFVC_LAUNCH_CHECK();
  return 0;
}

template <typename L, typename YT, int ACT, int BM>
int launch_tile(const I8Args& p, hipStream_t st) {
  constexpr int lds = 3 * BM * BK + 2 * BN * 128;
  const int tiles_n = ceil_div(p.N, BN);
  const int64_t n_tiles = (int64_t)ceil_div(p.M, BM) * tiles_n;
  FFVC_CHECK_ARG(ffvc_launch_fits(n_tiles, 256), "ffvc_gemm_int8: too many tiles for one launch");
  static ffvc_lds_once once;
  const int rc = once.set((const void*)gemm_int8_kernel<L, YT, ACT, BM>, lds);
  if (rc) return rc;
  hipLaunchKernelGGL((gemm_int8_kernel<L, YT, ACT, BM>), dim3((unsigned)n_tiles), dim3(256), lds, st, p, tiles_n);
  FFVC_LAUNCH_CHECK();
  return 0;
}

template <typename L, typename YT, int ACT>
int launch_gemm(const I8Args& p, hipStream_t st) {
  if (few_outputs(p.M, p.N)) return launch_skinny<L, YT>(p, st);
  // 256-row tiles from one per CU on (2056 x 4096 x 1024, 256 whole tiles: 19.3 against 22.8 us with 128 rows; 4617 x 512 x 2048, 72 tiles: 20.6
  // against 13.5).  Just above the border a short K gains nothing: 4617 x 2048 x 512, 288 whole tiles, 15.6 against 15.1; 8192 x 2048 x 512, 512 tiles, 19.3
  // against 19.8.  Up to 64 rows past the last whole tile go to the kernel above where the whole tiles fill the chip's two places per CU (16448 x
  // 4096 x 1024: 100 against 108 us; but 224 rows of 12000 x 2048 x 1024 45 against 38); with fewer they run beside the others anyway.
  const int64_t whole = (int64_t)(p.M / 256) * ceil_div(p.N, BN);
  if (whole < 256) return launch_tile<L, YT, ACT, 128>(p, st);
  const int rest = p.M % 256;
  if (rest == 0 || rest > 64 || !few_outputs(rest, p.N) || whole < 512) return launch_tile<L, YT, ACT, 256>(p, st);
  I8Args head = p, tail = p;
  head.M = p.M - rest;
  const int64_t m = head.M;
  tail.M = rest;
  tail.x += m * 64;
  tail.xs += m;
  tail.y = (YT*)p.y + m * p.ldy;
  if (p.res) tail.res = p.res_f32 ? (const void*)((const float*)p.res + m * p.ldr) : (const void*)((const L*)p.res + m * p.ldr);
  if (p.aux) tail.aux = (L*)p.aux + m * p.N;
  const int rc = launch_skinny<L, YT>(tail, st);             // (first: it runs beside the first tiles)
  return rc ? rc : launch_tile<L, YT, ACT, 256>(head, st);
}

// ---- a handful of rows ---------------------------------------------------------------------------------------------------------------------
// M <= 16 rows in ONE launch: every workgroup quantises the rows itself (a few KiB out of L2) and owns 16 output columns; its four waves
// split K.  v_mfma_i32_16x16x64_i8: A = 16 weight rows straight from global memory, B = the quantised rows from LDS.
// Against quantisation and the kernel above, us on the device: 1 x 2048 x 512 4.3 / 5.1, 16 x 2048 x 512 7.9 / 5.4, 16 x 4096 x 1024 10.8 / 6.6, 4 x 1024 x 4080
// 11.6 / 10.4, 16 x 1024 x 4080 31 / 11.5.  A launch less is worth 4 us to a caller: up to 16384 elements of x.
constexpr int FEW_M = 16, FEW_MK = 16384;

template <typename L, typename YT>
__global__ __launch_bounds__(256) void linear_int8_few_kernel(const L* __restrict__ x, const I8Args p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ldk = p.K + 16;                                 // LDS row stride in bytes
  float* xs = (float*)(smem + p.M * ldk);                   // [16]
  int* part = (int*)(xs + FEW_M);                           // [4 waves][4][64]
  for (int r = wave; r < p.M; r += 4) {
    const L* xr = x + r * p.xrows;
    float m = 0.0f;
    for (int k = lane * 8; k < p.K; k += 512) {
      const f32x8 v = load8(xr + k);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = amax_with_nan(m, v.v[j]);
    }
    const float s = row_scale(wave_amax(m));
    const RowQuant rq(s);
    if (lane == 0) xs[r] = s;
    for (int k = lane * 8; k < p.K; k += 512) *(u32x2_t*)(smem + r * ldk + k) = quant8(load8(xr + k), rq);
  }
  __syncthreads();
  const int l15 = lane & 15, g4 = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int8_t* wr = p.w + (int64_t)(n0 + l15 < p.N ? n0 + l15 : p.N - 1) * p.ldw;
  i32x4_t acc = {0, 0, 0, 0};
  const u32x4_t z = {0u, 0u, 0u, 0u};
#pragma unroll 4
  for (int k = wave * 64; k < p.K; k += 256) {
    const int kk = k + 16 * g4;                             // K % 16 == 0: a 16-byte chunk is inside or outside
    const u32x4_t a = kk < p.K ? *(const u32x4_t*)(wr + kk) : z;
    const u32x4_t b = kk < p.K && l15 < p.M ? *(const u32x4_t*)(smem + l15 * ldk + kk) : z;
    acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b), acc, 0, 0, 0);
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) part[(wave * 4 + r) * 64 + lane] = acc[r];
  __syncthreads();
  if (wave || l15 >= p.M) return;                           // column l15 of the product = row m, rows 4 g4 + r = output n0 + ...
#pragma unroll 1
  for (int r = 0; r < 4; ++r) {
    const int n = n0 + 4 * g4 + r;
    if (n >= p.N) break;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += part[(w * 4 + r) * 64 + lane];
    store_one<L, YT>(p, (float)sum * xs[l15], l15, n);
  }
}

template <typename L, typename YT>
int launch_few(const void* x, const I8Args& p, hipStream_t st) {
  const int lds = p.M * (p.K + 16) + FEW_M * 4 + 4 * 4 * 64 * 4;
  hipLaunchKernelGGL((linear_int8_few_kernel<L, YT>), dim3(ceil_div(p.N, 16)), dim3(256), lds, st, (const L*)x, p);
  FFVC_LAUNCH_CHECK();
  return 0;
}

// the storage types of one call: 16-bit lo (x of the one-launch form, aux, a 16-bit residual), y fp32 or lo
template <typename F>
int by_types(int lo, int y_dtype, F&& f) {
  if (lo == FFVC_F16) return y_dtype == FFVC_F32 ? f(f16_t{}, float{}) : f(f16_t{}, f16_t{});
  return y_dtype == FFVC_F32 ? f(uint16_t{}, float{}) : f(uint16_t{}, uint16_t{});
}

int check_out(const char* who, int lo, int M, int N, int K, const int8_t* w, int64_t ldw, const float* ws, const float* bias, int act, const void* res,
              int res_dtype, int64_t ldr, const void* y, int y_dtype, int64_t ldy) {
  FFVC_CHECK_ARG(lo == FFVC_BF16 || lo == FFVC_F16, "%s: the 16-bit type must be bf16 or f16", who);
  FFVC_CHECK_ARG(M > 0 && N > 0 && K > 0 && K % 16 == 0 && K <= 131072, "%s: bad problem (M=%d N=%d K=%d; K a multiple of 16, at most 131072)", who, M, N, K);
  FFVC_CHECK_ARG(w && ws && y, "%s: null pointer", who);
  FFVC_CHECK_ARG((uintptr_t)w % 16 == 0 && ldw % 16 == 0 && ldw >= K && ldw < (1 << 22), "%s: weight rows must be 16-byte aligned", who);
  FFVC_CHECK_ARG(y_dtype == FFVC_F32 || y_dtype == lo, "%s: y must be fp32 or the 16-bit type", who);
  FFVC_CHECK_ARG(!res || res_dtype == FFVC_F32 || res_dtype == lo, "%s: residual must be fp32 or the 16-bit type", who);
  FFVC_CHECK_ARG(act == FFVC_ACT_NONE || act == FFVC_ACT_GELU || act == FFVC_ACT_QUICKGELU, "%s: activation %d unsupported", who, act);
  FFVC_CHECK_ARG(ldy >= N && (!res || ldr >= N), "%s: output / residual rows shorter than N", who);
  return 0;
}
bool rows_vec(const void* p, int dtype, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % (dtype == FFVC_F32 ? 4 : 8) == 0; }

}  // namespace

extern "C" int ffvc_int8_quant(const void* x, int x_dtype, int64_t ldx, int8_t* q, int64_t ldq, float* scale, int64_t rows, int K, void* stream) {
  FFVC_CHECK_ARG(x && q && scale && rows > 0 && K > 0 && K % 16 == 0, "ffvc_int8_quant: bad args (K must be a multiple of 16)");
  FFVC_CHECK_ARG(ffvc_dtype_ok(x_dtype), "ffvc_int8_quant: bad dtype %d", x_dtype);
  FFVC_CHECK_ARG((uintptr_t)x % 16 == 0 && ldx % (16 / ffvc_dtype_size(x_dtype)) == 0 && ldx >= K && (uintptr_t)q % 16 == 0 && ldq % 16 == 0 && (ldq == 0 || ldq >= K),
                 "ffvc_int8_quant: rows must be 16-byte aligned");
  FFVC_CHECK_ARG(ffvc_launch_fits((rows + 3) / 4, 256), "ffvc_int8_quant: too many rows for one launch (%lld, at most %lld)", (long long)rows, 4 * ((1ll << 24) - 1));
  const dim3 grid((unsigned)((rows + 3) / 4)), block(256);
  hipStream_t st = (hipStream_t)stream;
  DISPATCH_DT(x_dtype, T, {
    if (K <= 512)
      hipLaunchKernelGGL((int8_quant_kernel<T, 1>), grid, block, 0, st, (const T*)x, ldx, q, ldq, scale, rows, K);
    else if (K <= 1024)
      hipLaunchKernelGGL((int8_quant_kernel<T, 2>), grid, block, 0, st, (const T*)x, ldx, q, ldq, scale, rows, K);
    else
      hipLaunchKernelGGL((int8_quant_kernel<T, 8>), grid, block, 0, st, (const T*)x, ldx, q, ldq, scale, rows, K);
  });
  FFVC_LAUNCH_CHECK();
  return 0;
}

extern "C" int ffvc_gemm_int8(const int8_t* x, const float* xs, const int8_t* w, int64_t ldw, const float* ws, const float* bias, int act,
                              const void* residual, int res_dtype, int64_t ldr, void* y, int y_dtype, int64_t ldy, void* actgrad, int lo_dtype, int M,
                              int N, int K, void* stream) {
  const int rc = check_out("ffvc_gemm_int8", lo_dtype, M, N, K, w, ldw, ws, bias, act, residual, res_dtype, ldr, y, y_dtype, ldy);
  if (rc) return rc;
  FFVC_CHECK_ARG(x && xs && (uintptr_t)x % 16 == 0, "ffvc_gemm_int8: x must be non-null and 16-byte aligned");
  I8Args p{x, w, xs, ws, bias, residual, y, actgrad, M, ldw, ldy, ldr, M, N, K, act, res_dtype == FFVC_F32, 0};
  p.vec = N % 8 == 0 && rows_vec(y, y_dtype, ldy) && (!residual || rows_vec(residual, res_dtype, ldr)) && (!actgrad || rows_vec(actgrad, lo_dtype, N));
  hipStream_t st = (hipStream_t)stream;
  return by_types(lo_dtype, y_dtype, [&](auto l, auto yt) {
    using L = decltype(l);
    using YT = decltype(yt);
    if (act == FFVC_ACT_GELU) return launch_gemm<L, YT, FFVC_ACT_GELU>(p, st);
    if (act == FFVC_ACT_QUICKGELU) return launch_gemm<L, YT, FFVC_ACT_QUICKGELU>(p, st);
    return launch_gemm<L, YT, FFVC_ACT_NONE>(p, st);
  });
}

extern "C" int ffvc_linear_int8_few_ok(int M, int K) {
  return M >= 1 && M <= FEW_M && K >= 16 && K % 16 == 0 && (int64_t)M * K <= FEW_MK;
}

extern "C" int ffvc_linear_int8_few(const void* x, int lo_dtype, int64_t ldx, const int8_t* w, int64_t ldw, const float* ws, const float* bias, int act,
                                    const void* residual, int res_dtype, int64_t ldr, void* y, int y_dtype, int64_t ldy, void* actgrad, int M, int N,
                                    int K, void* stream) {
  const int rc = check_out("ffvc_linear_int8_few", lo_dtype, M, N, K, w, ldw, ws, bias, act, residual, res_dtype, ldr, y, y_dtype, ldy);
  if (rc) return rc;
  FFVC_CHECK_ARG(ffvc_linear_int8_few_ok(M, K), "ffvc_linear_int8_few: M=%d K=%d unsupported", M, K);
  FFVC_CHECK_ARG(x && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 && ldx >= K, "ffvc_linear_int8_few: x rows must be 16-byte aligned");
  const I8Args p{nullptr, w, nullptr, ws, bias, residual, y, actgrad, ldx, ldw, ldy, ldr, M, N, K, act, res_dtype == FFVC_F32, 0};
  return by_types(lo_dtype, y_dtype, [&](auto l, auto yt) { return launch_few<decltype(l), decltype(yt)>(x, p, (hipStream_t)stream); });
}
