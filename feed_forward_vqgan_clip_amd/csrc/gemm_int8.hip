// gemm_int8.hip — Linear in 8-bit integers with one scale per token (row of x) and one per channel (row of w):
//
//     xs[m] = max_k |x[m, k]| / 127 (fp32)        xq[m, k] = round-half-even(x[m, k] / xs[m])        (the weight's rows likewise, once)
//     y[m, n] = act(xs[m] * ws[n] * sum_k xq[m, k] wq[n, k] + bias[n]) + residual[m, n]
//
// The integer sum is exact (32-bit accumulators, |sum| <= 127^2 K < 2^31 for K <= 131072), so the quantisation is the only approximation
// and the result does not depend on how K is cut.  Rounding to 8 bits follows the definition exactly: the quotient is formed with a
// reciprocal, then corrected with one fused residual (x - q xs is exact in fp32 once q is within one step of x / xs).
// A row of zeros has scale 0 and stays 0; a row that holds an inf or a NaN gets scale NaN, so its outputs are NaN and nothing is hidden.
#include "common.h"

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
// round-half-even(x / s); inv = 1 / s.  (Only where s itself is subnormal, and so a coarse amax / 127, can the quotient pass 127.)
__device__ __forceinline__ int quant1(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x);                                   // exact: what is left after q steps
  const float half = 0.5f * s;
  const bool odd = ((int)q & 1) != 0;
  if (fabsf(r) > half || (odd && fabsf(r) == half)) q += r > 0.0f ? 1.0f : -1.0f;
  return (int)fminf(fmaxf(q, -127.0f), 127.0f);
}
__device__ __forceinline__ uint32_t pack_i8(int a, int b, int c, int d) {
  return (uint32_t)(a & 255) | ((uint32_t)(b & 255) << 8) | ((uint32_t)(c & 255) << 16) | ((uint32_t)d << 24);
}
// One row's scale, ready to divide by: rows whose 1 / s would overflow are lifted by a power of two first (exact)
struct RowQuant {
  float s, inv, up;
  __device__ __forceinline__ RowQuant(float scale) {
    up = scale < 0x1p-100f ? 0x1p100f : 1.0f;
    s = scale * up;
    inv = s > 0.0f ? 1.0f / s : 0.0f;                               // 0: a row of zeros or one with a NaN / inf, stored as zeros
  }
};
__device__ __forceinline__ u32x2_t quant8(const f32x8& v, const RowQuant& r) {
  int q[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) q[j] = r.inv > 0.0f ? quant1(v.v[j] * r.up, r.s, r.inv) : 0;
  u32x2_t o;
  o[0] = pack_i8(q[0], q[1], q[2], q[3]);
  o[1] = pack_i8(q[4], q[5], q[6], q[7]);
  return o;
}

// wave maximum that keeps a NaN
__device__ __forceinline__ float wave_amax(float m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = amax_with_nan(m, __shfl_xor(m, o, 64));
  return m;
}

// One wave per row; a row of up to 64 * 8 * CH values stays in registers between the two passes, longer ones are read again (from L2).
template <typename T, int CH>
__global__ __launch_bounds__(256) void int8_quant_kernel(const T* __restrict__ x, int64_t ldx, int8_t* __restrict__ q, int64_t ldq,
                                                         float* __restrict__ scale, int64_t rows, int K) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const T* xr = x + row * ldx;
  int8_t* qr = q + row * ldq;
  f32x8 v[CH];
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int k = (i * 64 + lane) * 8;
    if (k < K) {
      v[i] = load8(xr + k);
#pragma unroll
      for (int j = 0; j < 8; ++j) m = amax_with_nan(m, v[i].v[j]);
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
    if (k < K) *(u32x2_t*)(qr + k) = quant8(v[i], rq);
  }
  for (int k = (CH * 64 + lane) * 8; k < K; k += 512) *(u32x2_t*)(qr + k) = quant8(load8(xr + k), rq);
}

// ---- epilogue ----------------------------------------------------------------------------------------------------------------------
// The activation and its derivative; 16-bit outputs take the hardware exp / rcp forms (errors ~2^-22), fp32 outputs the accurate ones.
template <bool FAST>
__device__ __forceinline__ void act_and_grad(int act, float z, float& y, float& g) {
  if (act == FFVC_ACT_GELU) {
    if constexpr (FAST) {
      float cdf, e;
      gelu_parts_fast(z, cdf, e);
      y = z * cdf;
      g = cdf + z * 0.39894228040143267794f * e;
    } else {
      y = act_gelu(z);
      g = act_gelu_grad(z);
    }
  } else if (act == FFVC_ACT_QUICKGELU) {
    const float s = FAST ? sigmoid_fast_(1.702f * z) : 1.0f / (1.0f + expf(-1.702f * z));
    y = z * s;
    g = s * (1.0f + 1.702f * z * (1.0f - s));
  } else {
    y = z;
    g = 1.0f;
  }
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
  int64_t ldx, ldw, ldy, ldr;
  int M, N, K;
  int act;
  int vec;                // rows of y / res / aux take 16-byte accesses and N % 8 == 0
};

// eight neighbouring outputs of row m.  YT: float or the 16-bit storage type; RT: the residual's type
template <typename L, typename YT, typename RT>
__device__ __forceinline__ void store_oct(const I8Args& p, const float (&acc)[8], int m, int n) {
  constexpr bool FAST = sizeof(YT) == 2;
  const float xs = p.xs[m];
  float v[8], g[8];
  YT* yr = (YT*)p.y + m * p.ldy + n;
  const RT* rr = (const RT*)p.res + m * p.ldr + n;
  L* ar = (L*)p.aux + (int64_t)m * p.N + n;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int nn = n + j < p.N ? n + j : p.N - 1;
    const float z = fmaf(acc[j], xs * p.ws[nn], p.bias ? p.bias[nn] : 0.0f);
    act_and_grad<FAST>(p.act, z, v[j], g[j]);
  }
  if (p.vec) {
    f32x8 o;
    if (p.res) {
      const f32x8 r = load8(rr);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += r.v[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) o.v[j] = v[j];
    store8(yr, o);
    if (p.aux) {
#pragma unroll
      for (int j = 0; j < 8; ++j) o.v[j] = g[j];
      store8(ar, o);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n + j < p.N) {
        ElemTraits<YT>::store(yr + j, v[j] + (p.res ? ElemTraits<RT>::load(rr + j) : 0.0f));
        if (p.aux) ElemTraits<L>::store(ar + j, g[j]);
      }
  }
}

// ---- the tiled product -----------------------------------------------------------------------------------------------------------------
// BM x BN outputs per workgroup, waves of (32 MT) x 64; K steps of 128 bytes, two LDS stages filled by LDS-DMA.  A staged row is 128 bytes,
// two rows to a 256-byte line, 16-byte chunks XOR-swizzled by the line: the 16-byte fragment reads of 32 rows hit every bank evenly.
__device__ __forceinline__ u32x4_t frag_i8(const unsigned char* tile, int row, int sub, int h) {
  const int line = row >> 1;
  return *(const u32x4_t*)(tile + line * 256 + (((((row & 1) << 3) | (2 * sub + h)) ^ (line & 15)) << 4));
}

template <int ROWS, int NW>
struct RowsDma {
  static constexpr int NP = ROWS / (8 * NW);
  rsrc_t rs;
  uint32_t off[NP];
  // rows row0 .. of a matrix with `rows` rows of K bytes; the descriptor ends with the last staged row, rows past it read as zeros
  __device__ __forceinline__ void init(const int8_t* base, int64_t ld, int row0, int rows, int K, int wave, int lane) {
    const int live = rows - row0 < ROWS ? rows - row0 : ROWS;
    rs = __builtin_amdgcn_make_buffer_rsrc((void*)(base + row0 * ld), 0, (int)((live - 1) * ld + K), 0x00020000);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int pos = (wave * NP + i) * 64 + lane, line = pos >> 4;
      const int cp = (pos & 15) ^ (line & 15);
      const int row = 2 * line + (cp >> 3);
      off[i] = row < live ? (uint32_t)(row * ld + (cp & 7) * 16) : OOB;
    }
  }
  __device__ __forceinline__ void issue(unsigned char* tile, int k0, int K, int wave) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      uint32_t o = off[i];
      if (k0 + 128 > K) {                    // K tail: chunks past K read as zeros
        const int pos = (wave * NP + i) * 64 + (threadIdx.x & 63), line = pos >> 4;
        if (k0 + ((((pos & 15) ^ (line & 15)) & 7) * 16) >= K) o = OOB;
      }
      dma16(rs, o, k0, tile + (wave * NP + i) * 1024);
    }
  }
};

template <typename L, typename YT, typename RT, int BM, int BN>
__global__ __launch_bounds__(2 * BN, (BM == 256 ? 2 : 1)) void gemm_int8_kernel(const I8Args p, int tiles_n, int n_tiles) {
  constexpr int MT = BM / 64, NW = 2 * (BN / 64);
  constexpr int XT = BM * 128, WT = BN * 128, STAGE = XT + WT;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  int tile;
  {   // consecutive workgroups go to the 8 XCDs in turn: give each XCD a contiguous run of tiles
    const int bid = blockIdx.x, q = n_tiles >> 3, r = n_tiles & 7, xcd = bid & 7;
    tile = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
  }
  const int tm = tile / tiles_n, tn = tile - tm * tiles_n;
  const int m0 = tm * BM, n0 = tn * BN;
  RowsDma<BM, NW> dx;
  RowsDma<BN, NW> dw;
  dx.init(p.x, p.ldx, m0, p.M, p.K, wave, lane);
  dw.init(p.w, p.ldw, n0, p.N, p.K, wave, lane);
  i32x16_t acc[2][MT];
#pragma unroll
  for (int a = 0; a < 2; ++a)
#pragma unroll
    for (int b = 0; b < MT; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0;
  const int nk = (p.K + 127) / 128;
  dx.issue(smem, 0, p.K, wave);
  dw.issue(smem + XT, 0, p.K, wave);
#pragma unroll 1
  for (int kt = 0; kt < nk; ++kt) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const unsigned char* sx = smem + (kt & 1) * STAGE;
    const unsigned char* sw = sx + XT;
    if (kt + 1 < nk) {
      unsigned char* nx = smem + ((kt + 1) & 1) * STAGE;
      dx.issue(nx, (kt + 1) * 128, p.K, wave);
      dw.issue(nx + XT, (kt + 1) * 128, p.K, wave);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u32x4_t fa[2], fb[MT];
#pragma unroll
      for (int t = 0; t < 2; ++t) fa[t] = frag_i8(sw, wn * 64 + t * 32 + l31, s, h);
#pragma unroll
      for (int t = 0; t < MT; ++t) fb[t] = frag_i8(sx, wm * (32 * MT) + t * 32 + l31, s, h);
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < MT; ++b)
          acc[a][b] = __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4_t, fa[a]), __builtin_bit_cast(i32x4_t, fb[b]), acc[a][b], 0, 0, 0);
    }
  }
  // A lane holds 4 neighbouring n of one m; through a 4 KiB pad of its wave (in the stage memory nobody reads any more) a block of
  // 32 x 32 leaves as rows of 8 outputs per lane.
  __syncthreads();
  unsigned char* pad = smem + wave * 4096;
#pragma unroll
  for (int b = 0; b < MT; ++b)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4_t v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)acc[a][b][4 * q + j];
        *(f32x4_t*)(pad + l31 * 128 + (((2 * q + h) ^ (l31 & 7)) << 4)) = v;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      const int cc = lane & 3;
      const int n = n0 + wn * 64 + a * 32 + 8 * cc;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = (lane >> 2) + 16 * i;
        const int m = m0 + wm * (32 * MT) + b * 32 + row;
        const f32x4_t lo = *(const f32x4_t*)(pad + row * 128 + (((2 * cc) ^ (row & 7)) << 4));
        const f32x4_t hi = *(const f32x4_t*)(pad + row * 128 + (((2 * cc + 1) ^ (row & 7)) << 4));
        const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        if (m < p.M && n < p.N) store_oct<L, YT, RT>(p, v, m, n);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
}

template <typename L, typename YT, typename RT, int BM, int BN>
int launch_tile(const I8Args& p, hipStream_t st) {
  constexpr int lds = 2 * (BM * 128 + BN * 128);
  const int tiles_n = ceil_div(p.N, BN);
  const int64_t n_tiles = (int64_t)ceil_div(p.M, BM) * tiles_n;
  FFVC_CHECK_ARG(n_tiles < (1ll << 31), "ffvc_gemm_int8: too many tiles for one launch");
  static ffvc_lds_once once;
  const int rc = once.set((const void*)gemm_int8_kernel<L, YT, RT, BM, BN>, lds);
  if (rc) return rc;
  hipLaunchKernelGGL((gemm_int8_kernel<L, YT, RT, BM, BN>), dim3((unsigned)n_tiles), dim3(2 * BN), lds, st, p, tiles_n, (int)n_tiles);
  FFVC_LAUNCH_CHECK();
  return 0;
}

template <typename L, typename YT, typename RT>
int launch_gemm(const I8Args& p, hipStream_t st) {
  const int64_t big = (int64_t)ceil_div(p.M, 256) * ceil_div(p.N, 256);
  if (big >= 192) return launch_tile<L, YT, RT, 256, 256>(p, st);
  return launch_tile<L, YT, RT, 128, 128>(p, st);
}

// ---- a handful of rows ---------------------------------------------------------------------------------------------------------------------
// M <= 16 rows in ONE launch: every workgroup quantises the rows itself (a few KiB out of L2) and owns 16 output columns; its four waves
// split K.  v_mfma_i32_16x16x64_i8: A = 16 weight rows straight from global memory, B = the quantised rows from LDS.
constexpr int FEW_M = 16;

template <typename L, typename YT, typename RT>
__global__ __launch_bounds__(256) void linear_int8_few_kernel(const L* __restrict__ x, const I8Args p) {
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ldk = p.K + 16;                                 // LDS row stride in bytes
  float* xs = (float*)(smem + p.M * ldk);                   // [16]
  int* part = (int*)(xs + FEW_M);                           // [4 waves][4][64]
  for (int r = wave; r < p.M; r += 4) {
    const L* xr = x + r * p.ldx;
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
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int n = n0 + 4 * g4 + r;
    if (n >= p.N) break;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) sum += part[(w * 4 + r) * 64 + lane];
    const float zz = fmaf((float)sum, xs[l15] * p.ws[n], p.bias ? p.bias[n] : 0.0f);
    float y, g;
    act_and_grad<sizeof(YT) == 2>(p.act, zz, y, g);
    if (p.res) y += ElemTraits<RT>::load((const RT*)p.res + l15 * p.ldr + n);
    ElemTraits<YT>::store((YT*)p.y + l15 * p.ldy + n, y);
    if (p.aux) ElemTraits<L>::store((L*)p.aux + (int64_t)l15 * p.N + n, g);
  }
}

template <typename L, typename YT, typename RT>
int launch_few(const void* x, const I8Args& p, hipStream_t st) {
  const int lds = p.M * (p.K + 16) + FEW_M * 4 + 4 * 4 * 64 * 4;
  static ffvc_lds_once once;
  const int rc = once.set((const void*)linear_int8_few_kernel<L, YT, RT>, 160 * 1024);
  if (rc) return rc;
  hipLaunchKernelGGL((linear_int8_few_kernel<L, YT, RT>), dim3(ceil_div(p.N, 16)), dim3(256), lds, st, (const L*)x, p);
  FFVC_LAUNCH_CHECK();
  return 0;
}

// the storage types of one call: 16-bit lo (x of the one-launch form, aux), y fp32 or lo, residual fp32 or lo
template <typename F>
int by_types(int lo, int y_dtype, int r_dtype, F&& f) {
  auto with = [&](auto l) {
    using L = decltype(l);
    if (y_dtype == FFVC_F32) return r_dtype == FFVC_F32 ? f(L{}, float{}, float{}) : f(L{}, float{}, L{});
    return r_dtype == FFVC_F32 ? f(L{}, L{}, float{}) : f(L{}, L{}, L{});
  };
  return lo == FFVC_F16 ? with(f16_t{}) : with(uint16_t{});
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
  FFVC_CHECK_ARG((uintptr_t)x % 16 == 0 && ldx % (16 / ffvc_dtype_size(x_dtype)) == 0 && ldx >= K && (uintptr_t)q % 16 == 0 && ldq % 16 == 0 && ldq >= K,
                 "ffvc_int8_quant: rows must be 16-byte aligned");
  FFVC_CHECK_ARG((rows + 3) / 4 < (1ll << 31), "ffvc_int8_quant: too many rows");
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

extern "C" int ffvc_gemm_int8(const int8_t* x, int64_t ldx, const float* xs, const int8_t* w, int64_t ldw, const float* ws, const float* bias, int act,
                              const void* residual, int res_dtype, int64_t ldr, void* y, int y_dtype, int64_t ldy, void* actgrad, int lo_dtype, int M,
                              int N, int K, void* stream) {
  const int rc = check_out("ffvc_gemm_int8", lo_dtype, M, N, K, w, ldw, ws, bias, act, residual, res_dtype, ldr, y, y_dtype, ldy);
  if (rc) return rc;
  FFVC_CHECK_ARG(x && xs && (uintptr_t)x % 16 == 0 && ldx % 16 == 0 && ldx >= K && ldx < (1 << 22), "ffvc_gemm_int8: x rows must be 16-byte aligned");
  I8Args p{x, w, xs, ws, bias, residual, y, actgrad, ldx, ldw, ldy, ldr, M, N, K, act, 0};
  p.vec = N % 8 == 0 && rows_vec(y, y_dtype, ldy) && (!residual || rows_vec(residual, res_dtype, ldr)) && (!actgrad || rows_vec(actgrad, lo_dtype, N));
  return by_types(lo_dtype, y_dtype, residual ? res_dtype : y_dtype, [&](auto l, auto yt, auto rt) {
    return launch_gemm<decltype(l), decltype(yt), decltype(rt)>(p, (hipStream_t)stream);
  });
}

extern "C" int ffvc_linear_int8_few_ok(int M, int K) {
  return M >= 1 && M <= FEW_M && K >= 16 && K % 16 == 0 && (int64_t)M * (K + 16) <= 64 * 1024;
}

extern "C" int ffvc_linear_int8_few(const void* x, int lo_dtype, int64_t ldx, const int8_t* w, int64_t ldw, const float* ws, const float* bias, int act,
                                    const void* residual, int res_dtype, int64_t ldr, void* y, int y_dtype, int64_t ldy, void* actgrad, int M, int N,
                                    int K, void* stream) {
  const int rc = check_out("ffvc_linear_int8_few", lo_dtype, M, N, K, w, ldw, ws, bias, act, residual, res_dtype, ldr, y, y_dtype, ldy);
  if (rc) return rc;
  FFVC_CHECK_ARG(ffvc_linear_int8_few_ok(M, K), "ffvc_linear_int8_few: M=%d K=%d unsupported", M, K);
  FFVC_CHECK_ARG(x && (uintptr_t)x % 16 == 0 && ldx % 8 == 0 && ldx >= K, "ffvc_linear_int8_few: x rows must be 16-byte aligned");
  const I8Args p{nullptr, w, nullptr, ws, bias, residual, y, actgrad, ldx, ldw, ldy, ldr, M, N, K, act, 0};
  return by_types(lo_dtype, y_dtype, residual ? res_dtype : y_dtype, [&](auto l, auto yt, auto rt) {
    return launch_few<decltype(l), decltype(yt), decltype(rt)>(x, p, (hipStream_t)stream);
  });
}
