// embed.hip — embedding lookup with scaling, and its gradient by sorted tokens.
//
//     out[t]    = scale * table[ids[t]] + pos[place[t]]          (rows of `dim`; an index outside its table reads a zero row)
//     dtable[v] = scale * sum over {t : ids[t] = v} of dout[t]   (every row is written once, rows nobody asked for as zeros)
//
// Gradient.  fp32 atomics would need a zero pass over the table and would sum in an order that changes from run to run (and one opening
// token per prompt makes thousands of adds collide on one row).  Here the token positions are sorted by id first — stable, so the sum of a
// row runs over its tokens in their order — and then every table row is produced by one owner: no zero pass, no atomics, the same bits
// every time.  Runs of equal ids are cut into chunks of CHUNK sorted positions whose sums a first kernel leaves in a workspace, so a row
// with thousands of tokens costs its owner a few dozen reads.
// Sorting: up to RANK_MAX tokens one launch ranks every key against all others out of LDS (n^2 compares spread over the chip); above, a
// least-significant-digit radix sort, 8 bits per pass, three launches each.
#include "common.h"

namespace {

constexpr int RANK_MAX = 8192;      // tokens
constexpr int CHUNK = 32;
constexpr int RT = 4096;            // keys per workgroup of a radix pass

template <typename T, int VEC>
struct Vec {
  float v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Vec<T, VEC> load_vec(const T* p) {
  Vec<T, VEC> r;
  if constexpr (VEC == 8) {
    const f32x8 a = load8(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) r.v[j] = a.v[j];
  } else {
    r.v[0] = ElemTraits<T>::load(p);
  }
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
  if constexpr (VEC == 8) {
    f32x8 a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a.v[j] = v[j];
    store8(p, a);
  } else {
    ElemTraits<T>::store(p, v[0]);
  }
}

// one wave per token
template <typename TT, typename OT, int VEC>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const TT* __restrict__ table, int64_t ld, int64_t vocab, const int64_t* __restrict__ ids,
                                                        float scale, const TT* __restrict__ pos, int64_t pos_ld, int64_t npos,
                                                        const int64_t* __restrict__ place, OT* __restrict__ out, int64_t ldo, int64_t n, int dim) {
  const int lane = threadIdx.x & 63;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= n) return;
  const int64_t id = ids[t];
  const bool ok = id >= 0 && id < vocab;
  const int64_t pl = pos ? (place ? place[t] : t) : -1;
  const bool okp = pl >= 0 && pl < npos;
  const TT* src = table + (ok ? id : 0) * ld;
  const TT* ps = pos + (okp ? pl : 0) * pos_ld;
  OT* dst = out + t * ldo;
  for (int c = lane * VEC; c < dim; c += 64 * VEC) {
    float v[VEC];
    Vec<TT, VEC> a, b;
    if (ok) a = load_vec<TT, VEC>(src + c);
    if (okp) b = load_vec<TT, VEC>(ps + c);
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = (ok ? scale * a.v[j] : 0.0f) + (okp ? b.v[j] : 0.0f);
    store_vec<OT, VEC>(dst + c, v);
  }
}

// ids outside the table sort behind every row
__device__ __forceinline__ uint32_t key_of(int64_t id, int64_t vocab) { return id >= 0 && id < vocab ? (uint32_t)id : (uint32_t)vocab; }

// ---- sort, small: position of token t = #{keys below its own} + #{equal keys before it}.  A workgroup ranks 32 tokens; its 32 half-waves
// split the keys (all of a half-wave's lanes read the same key: an LDS broadcast).
__global__ __launch_bounds__(1024) void embed_rank_kernel(const int64_t* __restrict__ ids, int64_t vocab, int n, uint32_t* __restrict__ keys,
                                                          uint32_t* __restrict__ vals) {
  __shared__ __attribute__((aligned(16))) uint32_t k[RANK_MAX];
  __shared__ int cnt[32];
  const int tid = threadIdx.x;
  const int np = (n + 127) / 128 * 128;                       // whole groups of 4 keys per part
  for (int i = tid; i < np; i += 1024) k[i] = i < n ? key_of(ids[i], vocab) : 0xFFFFFFFFu;
  if (tid < 32) cnt[tid] = 0;
  __syncthreads();
  const int t = blockIdx.x * 32 + (tid & 31), part = tid >> 5;
  const int per = np / 32, lo = part * per, hi = lo + per;
  const uint32_t me = t < n ? k[t] : 0u;
  int c = 0;
  const int mid = min(max(t, lo), hi) & ~3;                  // keys lo .. mid are all before t, from mid + 4 on none is
  for (int i = lo; i < mid; i += 4) {
    const u32x4_t q = *(const u32x4_t*)(k + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) c += q[j] <= me;
  }
  for (int i = mid; i < hi; i += 4) {
    const u32x4_t q = *(const u32x4_t*)(k + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) c += q[j] < me || (q[j] == me && i + j < t);
  }
  atomicAdd(&cnt[tid & 31], c);                               // integers: any order gives the same count
  __syncthreads();
  if (tid < 32 && t < n) {
    keys[cnt[tid]] = me;
    vals[cnt[tid]] = (uint32_t)t;
  }
}

// ---- sort, large ----------------------------------------------------------------------------------------------------------------------
// hist[digit][tile] of the 8 bits at `shift`
__global__ __launch_bounds__(256) void embed_hist_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ keys, int64_t vocab, int64_t n,
                                                         int shift, uint32_t* __restrict__ hist, int tiles) {
  __shared__ uint32_t h[256];
  const int tid = threadIdx.x;
  h[tid] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * RT;
  for (int i = tid; i < RT; i += 256) {
    const int64_t t = base + i;
    if (t < n) atomicAdd(&h[((ids ? key_of(ids[t], vocab) : keys[t]) >> shift) & 255u], 1u);
  }
  __syncthreads();
  hist[(int64_t)tid * tiles + blockIdx.x] = h[tid];
}

// exclusive scan of one digit's row of `hist`; the digit's total
__global__ __launch_bounds__(256) void embed_scan_kernel(uint32_t* __restrict__ hist, uint32_t* __restrict__ total, int tiles) {
  __shared__ uint32_t part[4];
  uint32_t* row = hist + (int64_t)blockIdx.x * tiles;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t run = 0;
  for (int b = 0; b < tiles; b += 256) {
    const uint32_t v = b + tid < tiles ? row[b + tid] : 0u;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(s, o, 64);
      if (lane >= o) s += u;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    uint32_t before = run;
    for (int w = 0; w < wave; ++w) before += part[w];
    if (b + tid < tiles) row[b + tid] = before + s - v;
    run += part[0] + part[1] + part[2] + part[3];
    __syncthreads();
  }
  if (tid == 0) total[blockIdx.x] = run;
}

// Stable scatter: wave w of a tile owns its keys 1024 w .. + 1023 and walks them 64 at a time; lanes of one digit find each other by ballots.
__global__ __launch_bounds__(256) void embed_scatter_kernel(const int64_t* __restrict__ ids, const uint32_t* __restrict__ keys,
                                                            const uint32_t* __restrict__ vals, int64_t vocab, int64_t n, int shift,
                                                            const uint32_t* __restrict__ hist, const uint32_t* __restrict__ total, int tiles,
                                                            uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out) {
  __shared__ uint32_t at[4][256];                            // next position of each digit, per wave
  __shared__ uint32_t part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int PW = RT / 4;
#pragma unroll
  for (int w = 0; w < 4; ++w) at[w][tid] = 0;
  uint32_t base;                                              // keys of smaller digits, and of this digit in earlier tiles
  {
    const uint32_t v = total[tid];
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(s, o, 64);
      if (lane >= o) s += u;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    base = s - v + hist[(int64_t)tid * tiles + blockIdx.x];
    for (int w = 0; w < wave; ++w) base += part[w];
  }
  const int64_t first = (int64_t)blockIdx.x * RT + wave * PW;
  for (int i = 0; i < PW; i += 64) {
    const int64_t t = first + i + lane;
    if (t < n) atomicAdd(&at[wave][((ids ? key_of(ids[t], vocab) : keys[t]) >> shift) & 255u], 1u);
  }
  __syncthreads();
  {   // counts -> starts
    uint32_t run = base;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t c = at[w][tid];
      at[w][tid] = run;
      run += c;
    }
  }
  __syncthreads();
  for (int i = 0; i < PW; i += 64) {
    const int64_t t = first + i + lane;
    const bool in = t < n;
    const uint32_t key = in ? (ids ? key_of(ids[t], vocab) : keys[t]) : 0u;
    const uint32_t val = in ? (vals ? vals[t] : (uint32_t)t) : 0u;
    const uint32_t d = (key >> shift) & 255u;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const uint64_t m = __ballot((d >> b) & 1u);
      same &= (d >> b) & 1u ? m : ~m;
    }
    const int before = __popcll(same & ((1ull << lane) - 1ull));
    uint32_t p = 0;
    if (in) p = at[wave][d] + before;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");    // everyone has read before the first lane of a digit moves it on
    if (in && before == 0) at[wave][d] = p + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (in) {
      keys_out[p] = key;
      vals_out[p] = val;
    }
  }
}

// ---- sums ------------------------------------------------------------------------------------------------------------------------------
// part[c] = sum of dout over sorted positions CHUNK c .. + CHUNK - 1, where they all hold one id (others are not needed).  One wave each.
template <typename DT, int VEC>
__global__ __launch_bounds__(256) void embed_part_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, int64_t n,
                                                         uint32_t vocab, const DT* __restrict__ dout, int64_t ld, int dim, float* __restrict__ part) {
  const int lane = threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t p0 = c * CHUNK;
  if (p0 + CHUNK > n) return;
  const uint32_t key = keys[p0];
  if (key >= vocab || keys[p0 + CHUNK - 1] != key) return;
  for (int d = lane * VEC; d < dim; d += 64 * VEC) {
    float acc[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
#pragma unroll 8
    for (int i = 0; i < CHUNK; ++i) {
      const Vec<DT, VEC> a = load_vec<DT, VEC>(dout + (int64_t)vals[p0 + i] * ld + d);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += a.v[j];
    }
    store_vec<float, VEC>(part + c * dim + d, acc);
  }
}

// first sorted position whose key is >= v, 64 probes at a time (one wave)
__device__ __forceinline__ int64_t lower_bound64(const uint32_t* __restrict__ keys, int64_t n, uint32_t v, int lane) {
  int64_t lo = 0, hi = n;                                     // the answer is in lo .. hi
  while (hi > lo) {
    const int64_t step = (hi - lo + 63) / 64;
    const int64_t p = lo + lane * step;
    const uint64_t below = __ballot(p < hi && keys[p] < v);
    const int k = __popcll(below);                            // probes 0 .. k - 1 are below v
    if (k == 0) return lo;
    hi = min(hi, lo + k * step);
    lo += (k - 1) * step + 1;
  }
  return lo;
}

// R table rows per workgroup.  A row's tokens: single ones up to a chunk border, whole chunks, single ones behind; the four waves take
// them in four consecutive shares whose sums meet in LDS in order (short rows: one wave takes the row alone).
template <typename DT, typename TT, int VEC>
__global__ __launch_bounds__(256) void embed_reduce_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, int64_t n, int64_t vocab,
                                                           const DT* __restrict__ dout, int64_t ld, int dim, float scale,
                                                           const float* __restrict__ part, TT* __restrict__ dtable, int R) {
  constexpr int SHORT = 16;
  __shared__ int64_t edge[17];                                // R <= 16
  __shared__ float sums[4][64 * VEC];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t v0 = (int64_t)blockIdx.x * R;
  const int nr = (int)(vocab - v0 < R ? vocab - v0 : R);
  for (int r = wave; r <= nr; r += 4) {
    const int64_t e = lower_bound64(keys, n, (uint32_t)(v0 + r), lane);
    if (lane == 0) edge[r] = e;
  }
  __syncthreads();
  // items of a row: head tokens a .. h, chunks h / CHUNK .. t / CHUNK, tail tokens t .. b
  auto add_items = [&](float (&acc)[VEC], int64_t a, int64_t h, int64_t t, int64_t i0, int64_t i1, int d) {
    const int64_t nh = h - a, nc = (t - h) / CHUNK;
    int64_t i = i0;
#pragma unroll 4
    for (; i < i1 && i < nh; ++i) {
      const Vec<DT, VEC> x = load_vec<DT, VEC>(dout + (int64_t)vals[a + i] * ld + d);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += x.v[j];
    }
#pragma unroll 4
    for (; i < i1 && i < nh + nc; ++i) {
      const Vec<float, VEC> x = load_vec<float, VEC>(part + (h / CHUNK + i - nh) * dim + d);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += x.v[j];
    }
#pragma unroll 4
    for (; i < i1; ++i) {
      const Vec<DT, VEC> x = load_vec<DT, VEC>(dout + (int64_t)vals[t + i - nh - nc] * ld + d);
#pragma unroll
      for (int j = 0; j < VEC; ++j) acc[j] += x.v[j];
    }
  };
  for (int r = 0; r < nr; ++r) {
    const int64_t a = edge[r], b = edge[r + 1];
    const int64_t up = (a + CHUNK - 1) / CHUNK * CHUNK, dn = b / CHUNK * CHUNK;
    const int64_t h = up < dn ? up : b, t = up < dn ? dn : b;    // no whole chunk: every token is a head token
    const int64_t items = (h - a) + (t - h) / CHUNK + (b - t);
    TT* row = dtable + (v0 + r) * dim;
    if (items <= SHORT) {
      if ((r & 3) == wave)
        for (int d = lane * VEC; d < dim; d += 64 * VEC) {
          float acc[VEC];
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
          add_items(acc, a, h, t, 0, items, d);
#pragma unroll
          for (int j = 0; j < VEC; ++j) acc[j] *= scale;
          store_vec<TT, VEC>(row + d, acc);
        }
    } else {
      for (int d0 = 0; d0 < dim; d0 += 64 * VEC) {
        const int d = d0 + lane * VEC;
        float acc[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
        if (d < dim) add_items(acc, a, h, t, items * wave / 4, items * (wave + 1) / 4, d);
#pragma unroll
        for (int j = 0; j < VEC; ++j) sums[wave][lane * VEC + j] = acc[j];
        __syncthreads();
        if (wave == 0 && d < dim) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const int x = lane * VEC + j;
            acc[j] = (((sums[0][x] + sums[1][x]) + sums[2][x]) + sums[3][x]) * scale;
          }
          store_vec<TT, VEC>(row + d, acc);
        }
        __syncthreads();
      }
    }
  }
}

struct Layout {      // the workspace: two (keys, vals) pairs, the radix counters, the chunk sums
  int64_t pair, tiles, hist, part, bytes;
  Layout(int64_t n, int dim) {
    pair = (n * 4 + 15) / 16 * 16;
    tiles = (n + RT - 1) / RT;
    hist = 4 * pair;
    part = hist + (n > RANK_MAX ? (256 * tiles + 256) * 4 : 0);
    bytes = part + n / CHUNK * dim * 4;
  }
};

template <typename DT, typename TT, int VEC>
int run_sums(const uint32_t* keys, const uint32_t* vals, int64_t n, int64_t vocab, const void* dout, int64_t ld, int dim, float scale, float* part,
             void* dtable, hipStream_t st) {
  const int64_t chunks = n / CHUNK;
  if (chunks)
    hipLaunchKernelGGL((embed_part_kernel<DT, VEC>), dim3((unsigned)((chunks + 3) / 4)), dim3(256), 0, st, keys, vals, n, (uint32_t)vocab, (const DT*)dout,
                       ld, dim, part);
  // rows per workgroup: enough workgroups to fill the chip first, then fewer searches per row
  const int R = (int)(vocab / 1024 < 1 ? 1 : (vocab / 1024 > 16 ? 16 : vocab / 1024));
  hipLaunchKernelGGL((embed_reduce_kernel<DT, TT, VEC>), dim3((unsigned)((vocab + R - 1) / R)), dim3(256), 0, st, keys, vals, n, vocab, (const DT*)dout, ld,
                     dim, scale, part, (TT*)dtable, R);
  FFVC_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" int ffvc_embed_fwd(const void* table, int table_dtype, int64_t ld, int64_t vocab, const int64_t* ids, float scale, const void* pos,
                              int64_t pos_ld, int64_t npos, const int64_t* place, void* out, int out_dtype, int64_t ldo, int64_t n, int dim, void* stream) {
  FFVC_CHECK_ARG(table && ids && out && n > 0 && dim > 0 && vocab > 0, "ffvc_embed_fwd: bad args");
  FFVC_CHECK_ARG(ffvc_dtype_ok(table_dtype) && ffvc_dtype_ok(out_dtype), "ffvc_embed_fwd: bad dtype");
  FFVC_CHECK_ARG(ld >= dim && ldo >= dim && (!pos || (pos_ld >= dim && npos > 0)), "ffvc_embed_fwd: rows shorter than dim");
  FFVC_CHECK_ARG((n + 3) / 4 < (1ll << 31), "ffvc_embed_fwd: too many tokens for one launch");
  auto al = [](const void* p, int dt, int64_t l) { return (uintptr_t)p % 16 == 0 && l % (16 / ffvc_dtype_size(dt)) == 0; };
  const bool vec = dim % 8 == 0 && al(table, table_dtype, ld) && al(out, out_dtype, ldo) && (!pos || al(pos, table_dtype, pos_ld));
  const dim3 grid((unsigned)((n + 3) / 4)), block(256);
  hipStream_t st = (hipStream_t)stream;
  DISPATCH_DT(table_dtype, TT, DISPATCH_DT(out_dtype, OT, {
    if (vec)
      hipLaunchKernelGGL((embed_fwd_kernel<TT, OT, 8>), grid, block, 0, st, (const TT*)table, ld, vocab, ids, scale, (const TT*)pos, pos_ld, npos, place,
                         (OT*)out, ldo, n, dim);
    else
      hipLaunchKernelGGL((embed_fwd_kernel<TT, OT, 1>), grid, block, 0, st, (const TT*)table, ld, vocab, ids, scale, (const TT*)pos, pos_ld, npos, place,
                         (OT*)out, ldo, n, dim);
  }));
  FFVC_LAUNCH_CHECK();
  return 0;
}

extern "C" int64_t ffvc_embed_bwd_ws_bytes(int64_t n, int dim) { return n > 0 && dim > 0 ? Layout(n, dim).bytes : 0; }

extern "C" int ffvc_embed_bwd(const void* dout, int dout_dtype, int64_t ld, const int64_t* ids, int64_t n, int64_t vocab, int dim, float scale,
                              void* dtable, int table_dtype, void* ws, int64_t ws_bytes, void* stream) {
  FFVC_CHECK_ARG(dout && ids && dtable && ws && n > 0 && dim > 0 && vocab > 0, "ffvc_embed_bwd: bad args");
  FFVC_CHECK_ARG(ffvc_dtype_ok(dout_dtype) && ffvc_dtype_ok(table_dtype), "ffvc_embed_bwd: bad dtype");
  FFVC_CHECK_ARG(ld >= dim, "ffvc_embed_bwd: rows shorter than dim");
  FFVC_CHECK_ARG(n < (1ll << 31) && vocab < (1ll << 31), "ffvc_embed_bwd: token count and vocabulary must stay below 2^31");
  const Layout lay(n, dim);
  FFVC_CHECK_ARG((uintptr_t)ws % 16 == 0 && ws_bytes >= lay.bytes, "ffvc_embed_bwd: workspace of %lld bytes needed, got %lld", (long long)lay.bytes,
                 (long long)ws_bytes);
  hipStream_t st = (hipStream_t)stream;
  char* w = (char*)ws;
  uint32_t* keys[2] = {(uint32_t*)w, (uint32_t*)(w + 2 * lay.pair)};
  uint32_t* vals[2] = {(uint32_t*)(w + lay.pair), (uint32_t*)(w + 3 * lay.pair)};
  int cur = 0;
  if (n <= RANK_MAX) {
    hipLaunchKernelGGL(embed_rank_kernel, dim3((unsigned)((n + 31) / 32)), dim3(1024), 0, st, ids, vocab, (int)n, keys[0], vals[0]);
  } else {
    uint32_t* hist = (uint32_t*)(w + lay.hist);
    uint32_t* total = hist + 256 * lay.tiles;
    const int tiles = (int)lay.tiles;
    bool first = true;
    for (int shift = 0; shift == 0 || (shift < 32 && (vocab >> shift) != 0); shift += 8) {
      const int64_t* src = first ? ids : nullptr;
      const int nx = first ? 0 : cur ^ 1;
      hipLaunchKernelGGL(embed_hist_kernel, dim3(tiles), dim3(256), 0, st, src, keys[cur], vocab, n, shift, hist, tiles);
      hipLaunchKernelGGL(embed_scan_kernel, dim3(256), dim3(256), 0, st, hist, total, tiles);
      hipLaunchKernelGGL(embed_scatter_kernel, dim3(tiles), dim3(256), 0, st, src, keys[cur], first ? nullptr : vals[cur], vocab, n, shift, hist, total,
                         tiles, keys[nx], vals[nx]);
      cur = nx;
      first = false;
    }
  }
  auto al = [](const void* p, int dt, int64_t l) { return (uintptr_t)p % 16 == 0 && l % (16 / ffvc_dtype_size(dt)) == 0; };
  const bool vec = dim % 8 == 0 && al(dout, dout_dtype, ld) && al(dtable, table_dtype, dim);
  float* part = (float*)(w + lay.part);
  DISPATCH_DT(dout_dtype, DT, DISPATCH_DT(table_dtype, TT, {
    return vec ? run_sums<DT, TT, 8>(keys[cur], vals[cur], n, vocab, dout, ld, dim, scale, part, dtable, st)
               : run_sums<DT, TT, 1>(keys[cur], vals[cur], n, vocab, dout, ld, dim, scale, part, dtable, st);
  }));
  return 0;
}
