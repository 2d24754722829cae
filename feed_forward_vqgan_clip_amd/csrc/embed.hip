// embed.hip — embedding lookup with scaling, and its gradient by sorted tokens.
//
//     out[t]    = scale * table[ids[t]] + pos[place[t]]          (rows of `dim`; an index outside its table reads a zero row)
//     dtable[v] = scale * sum over {t : ids[t] = v} of dout[t]   (every row is written once, rows nobody asked for as zeros)
//
// Gradient.  fp32 atomics would need a zero pass over the table and would sum in an order that changes from run to run (and one opening
// token per prompt makes thousands of adds collide on one row).  Here the token positions are sorted by id first — stable, so the sum of a
// row runs over its tokens in their order — and then every table row is produced by one owner: no zero pass, no atomics, the same bits
// every time.  The work is cut by sorted positions, not by rows (ids come ordered by frequency, so a few neighbouring rows hold most tokens): a
// wave sums a chunk of them and writes the rows whose tokens it has all seen, a second kernel joins the parts of longer runs and writes the zeros.
// Bound by bytes: 113000 tokens of 1024 bf16 read for both tables in 99 us (4.7 TB/s); the rows kernel (41 us there) by its workgroups' launches and
// the longest runs' joins.  The lookup is one wave per token and bound by its writes (82 us there: 232 MB out, about 100 in).
// Sorting: up to RANK_MAX tokens one launch ranks every key against all others out of LDS (n^2 compares spread over the chip); above, a
// least-significant-digit radix sort, 8 bits per pass, two or three launches each.
#include <type_traits>

#include "common.h"

namespace {

constexpr int RANK_MAX = 8192;      // tokens
constexpr int RT = 1024;            // keys per workgroup of a radix pass

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

// One table's gradient.  The token table's and the position table's are two chains of small launches over the same dout: they go through every
// launch together, blockIdx.z (or the block's place) picks the table (509 prompts, 21000 tokens of 512, 77 positions: 52 us for both, 50 for the
// token table alone, 32 more for the positions in launches of their own).
struct Job {
  const int64_t* ids;          // null: row t for token t
  int64_t vocab;
  float scale;
  void* dtable;
  uint32_t *keys[2], *vals[2];
  uint32_t *hist, *total;      // radix counters
  int* span;                   // [vocab][2]: each row's first sorted token and the place after its last
  float* part;
  int sorted;                  // which pair holds the sorted tokens
};
struct Jobs {
  Job j[2];
};

// span[v][0] = -1 (no token) for every row, by the first kernel of the chain
__device__ __forceinline__ void clear_span(const Job& job) {
  for (int64_t v = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; v < job.vocab; v += (int64_t)gridDim.x * blockDim.x) job.span[2 * v] = -1;
}

// ids outside the table sort behind every row
__device__ __forceinline__ uint32_t key_of(const Job& job, int64_t t) {
  const int64_t id = job.ids ? job.ids[t] : t;
  return (uint32_t)(id >= 0 && id < job.vocab ? id : job.vocab);
}

// ---- sort, small: position of token t = #{keys below its own} + #{equal keys before it}.  A workgroup ranks 32 tokens; its 32 half-waves
// split the keys (all of a half-wave's lanes read the same key: an LDS broadcast).
__global__ __launch_bounds__(1024) void embed_rank_kernel(const Jobs jobs, int n) {
  const Job& job = jobs.j[blockIdx.z];
  uint32_t *keys = job.keys[0], *vals = job.vals[0];
  clear_span(job);
  extern __shared__ __attribute__((aligned(16))) uint32_t k[];
  const int tid = threadIdx.x;
  const int np = (n + 127) / 128 * 128;                       // whole groups of 4 keys per part
  int* cnt = (int*)(k + np);                                  // [32]
  for (int i = tid; i < np; i += 1024) k[i] = i < n ? key_of(job, i) : 0xFFFFFFFFu;
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
// A table's passes are those of its own bits: the other one's further launches find nothing to do.
__device__ __forceinline__ bool pass_done(const Job& job, int shift) { return shift > 0 && (job.vocab >> shift) == 0; }

// hist[digit][tile] of the 8 bits at `shift`
__global__ __launch_bounds__(256) void embed_hist_kernel(const Jobs jobs, int64_t n, int shift, int tiles) {
  const Job& job = jobs.j[blockIdx.z];
  if (pass_done(job, shift)) return;
  const uint32_t* keys = job.keys[(shift / 8 + 1) & 1];
  if (shift == 0) clear_span(job);
  __shared__ uint32_t h[256];
  const int tid = threadIdx.x;
  h[tid] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * RT;
  for (int i = tid; i < RT; i += 256) {
    const int64_t t = base + i;
    if (t < n) atomicAdd(&h[((shift == 0 ? key_of(job, t) : keys[t]) >> shift) & 255u], 1u);
  }
  __syncthreads();
  job.hist[(int64_t)tid * tiles + blockIdx.x] = h[tid];
}

// exclusive scan of one digit's row of `hist`; the digit's total
__global__ __launch_bounds__(256) void embed_scan_kernel(const Jobs jobs, int shift, int tiles) {
  __shared__ uint32_t part[4];
  const Job& job = jobs.j[blockIdx.z];
  if (pass_done(job, shift)) return;
  uint32_t* row = job.hist + (int64_t)blockIdx.x * tiles;
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
  if (tid == 0) job.total[blockIdx.x] = run;
}

// Stable scatter: wave w of a tile owns a quarter of its keys and walks them 64 at a time; lanes of one digit find each other by ballots.
__global__ __launch_bounds__(256) void embed_scatter_kernel(const Jobs jobs, int64_t n, int shift, int tiles, int scanned) {
  const Job& job = jobs.j[blockIdx.z];
  if (pass_done(job, shift)) return;
  const int to = (shift / 8) & 1;
  const uint32_t *keys = job.keys[to ^ 1], *vals = job.vals[to ^ 1], *hist = job.hist;
  uint32_t *keys_out = job.keys[to], *vals_out = job.vals[to];
  __shared__ uint32_t at[4][256];                            // next position of each digit, per wave
  __shared__ uint32_t part[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int PW = RT / 4;                                  // keys of a wave
#pragma unroll
  for (int w = 0; w < 4; ++w) at[w][tid] = 0;
  uint32_t base;                                              // keys of smaller digits, and of this digit in earlier tiles
  {
    uint32_t v = 0, mine = 0;                                 // this digit's keys in all tiles, in earlier tiles
    if (scanned) {
      v = job.total[tid];
      mine = hist[(int64_t)tid * tiles + blockIdx.x];
    } else {
#pragma unroll 8
      for (int t = 0; t < tiles; ++t) {
        const uint32_t c = hist[(int64_t)tid * tiles + t];
        mine += t < (int)blockIdx.x ? c : 0u;
        v += c;
      }
    }
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t u = __shfl_up(s, o, 64);
      if (lane >= o) s += u;
    }
    if (lane == 63) part[wave] = s;
    __syncthreads();
    base = s - v + mine;
    for (int w = 0; w < wave; ++w) base += part[w];
  }
  const int64_t first = (int64_t)blockIdx.x * RT + wave * PW;
  for (int i = 0; i < PW; i += 64) {
    const int64_t t = first + i + lane;
    if (t < n) atomicAdd(&at[wave][((shift == 0 ? key_of(job, t) : keys[t]) >> shift) & 255u], 1u);
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
    const uint32_t key = in ? (shift == 0 ? key_of(job, t) : keys[t]) : 0u;
    const uint32_t val = in ? (shift == 0 ? (uint32_t)t : vals[t]) : 0u;
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
// One wave per chunk of `chunk` <= 64 sorted positions and block of 64 * VEC columns.  Runs of one id that begin and end inside the chunk go straight
// to their table row; one that came in from the chunk before leaves its sum in part[2 c], one that goes on into the next in part[2 c + 1].
// span: the rows kernel's map.
template <typename DT, typename TT, int VEC>
__global__ __launch_bounds__(256) void embed_runs_kernel(const Jobs jobs, int n, const DT* __restrict__ dout, int64_t ld, int dim, int chunk) {
  const Job& job = jobs.j[blockIdx.z];
  const uint32_t* __restrict__ keys = job.keys[job.sorted];
  const uint32_t* __restrict__ vals = job.vals[job.sorted];
  const uint32_t vocab = (uint32_t)job.vocab;
  const float scale = job.scale;
  float* __restrict__ part = job.part;
  TT* __restrict__ dtable = (TT*)job.dtable;
  const int lane = threadIdx.x & 63;
  const int64_t c = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t p0 = c * chunk;
  if (p0 >= n) return;
  const int m = __builtin_amdgcn_readfirstlane((int)(n - p0 < chunk ? n - p0 : chunk));
  const uint32_t key = lane < m ? keys[p0 + lane] : 0xFFFFFFFFu;
  const uint32_t val = lane < m ? vals[p0 + lane] : 0u;
  const uint32_t left = p0 + lane > 0 && lane <= m ? keys[p0 + lane - 1] : 0xFFFFFFFFu;      // (lane m: the chunk's last key)
  const uint32_t next = p0 + m < n ? keys[p0 + m] : 0xFFFFFFFFu;                              // first key of the next chunk
  const uint64_t starts = __ballot(lane < m && key != left);
  if (blockIdx.y == 0 && lane < m && key < vocab) {
    if (key != left) job.span[2 * (int64_t)key] = (int)(p0 + lane);
    const uint32_t right = lane + 1 < m ? keys[p0 + lane + 1] : next;
    if (key != right) job.span[2 * (int64_t)key + 1] = (int)(p0 + lane + 1);
  }
  const bool in = !(starts & 1ull);                            // the chunk's first run came in from the chunk before
  const bool out = p0 + m < n && __builtin_amdgcn_readlane(key, m - 1) == __builtin_amdgcn_readfirstlane(next);
  const int d = (blockIdx.y * 64 + lane) * VEC;
  const bool live = d < dim;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
  auto flush = [&](int j) {                                    // the run that ends before token j
    const uint32_t k = __builtin_amdgcn_readlane(key, j - 1);
    const bool came = in && (starts & ((2ull << (j - 1)) - 1ull)) == 0;
    if (k < vocab && live) {
      if (came) {
        store_vec<float, VEC>(part + 2 * c * dim + d, acc);
      } else if (j == m && out) {
        store_vec<float, VEC>(part + (2 * c + 1) * dim + d, acc);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= scale;
        store_vec<TT, VEC>(dtable + (int64_t)k * dim + d, acc);
      }
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
  };
  constexpr int U = 8;                                         // rows under way
  for (int j0 = 0; j0 < m; j0 += U) {
    Vec<DT, VEC> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      x[u] = load_vec<DT, VEC>(dout + (int64_t)__builtin_amdgcn_readlane(val, j0 + u < m ? j0 + u : m - 1) * ld + (live ? d : 0));
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (j0 + u < m) {
        if (j0 + u > 0 && ((starts >> (j0 + u)) & 1)) flush(j0 + u);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += x[u].v[e];
      }
  }
  flush(m);
}

// The rows the runs kernel has not written: zeros where no token asked for the row, the sum of the parts where its run crosses chunks.  ROWS rows
// per workgroup (the long case 2 / 4 / 8 / 16 of them: 42 / 39 / 43 / 52 us: launches against the few longest runs, which are neighbours); up to SHORT
// parts one wave sums them, more are taken by the four waves in consecutive shares that meet in LDS in order.
constexpr int ROWS = 4, SHORT = 8;
template <typename TT, int VEC>
__global__ __launch_bounds__(256) void embed_rows_kernel(const Jobs jobs, int dim, int chunk, int blocks1) {
  __shared__ float sums[4][64 * VEC];
  const int which = (int)blockIdx.x < blocks1;                 // the second table's (fewer and longer) rows first
  const Job& job = jobs.j[which];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t v0 = (int64_t)(blockIdx.x - (which ? 0 : blocks1)) * ROWS, vocab = job.vocab;
  const float scale = job.scale;
  const float* __restrict__ part = job.part;
  TT* __restrict__ dtable = (TT*)job.dtable;
  const int nr = (int)(vocab - v0 < ROWS ? vocab - v0 : ROWS);
  const int d = (blockIdx.y * 64 + lane) * VEC;
  const bool live = d < dim;
  // parts of a row: part[2 ca + 1], then part[2 c] of the chunks ca + 1 .. cb; U loads under way (the last one again past the end, not added)
  auto add = [&](auto U, float (&acc)[VEC], int ca, int i0, int i1) {
    const float* p = part + 2 * (int64_t)ca * dim + (live ? d : 0);
    for (int i = i0; i < i1; i += U) {
      Vec<float, VEC> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = i + u < i1 ? i + u : i1 - 1;
        x[u] = load_vec<float, VEC>(p + (k ? 2 * (int64_t)k : 1) * dim);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += i + u < i1 ? x[u].v[e] : 0.0f;
    }
  };
  const int2 at = lane < nr ? ((const int2*)job.span)[v0 + lane] : make_int2(-1, 0);
  const int av = at.x;
  const int npv = av >= 0 ? (at.y - 1) / chunk - av / chunk + 1 : 0;               // 0: no token; 1: written already
  for (int r = 0; r < nr; ++r) {
    const int a = __builtin_amdgcn_readlane(av, r), np = __builtin_amdgcn_readlane(npv, r);
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
    TT* row = dtable + (v0 + r) * dim + d;
    if (np <= SHORT) {
      if (r % 4 == wave && np != 1) {
        add(std::integral_constant<int, 2>{}, acc, a / chunk, 0, np);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= scale;
        if (live) store_vec<TT, VEC>(row, acc);
      }
    } else {
      add(std::integral_constant<int, 8>{}, acc, a / chunk, (int)((int64_t)np * wave / 4), (int)((int64_t)np * (wave + 1) / 4));
#pragma unroll
      for (int e = 0; e < VEC; ++e) sums[wave][lane * VEC + e] = acc[e];
      __syncthreads();
      if (wave == 0 && live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int y = lane * VEC + e;
          acc[e] = (((sums[0][y] + sums[1][y]) + sums[2][y]) + sums[3][y]) * scale;
        }
        store_vec<TT, VEC>(row, acc);
      }
      __syncthreads();
    }
  }
}

// The workspace of `count` tables: for each two (keys, vals) pairs, the span of every row, the radix counters, the parts.
struct Layout {
  int64_t n, tiles, bytes;
  int chunk;
  bool rank;
  Jobs jobs;
  Layout(int64_t n_, int dim, int count, const int64_t (&vocab)[2], char* ws) : n(n_), bytes(0), jobs() {
    // One ranking launch against one or more radix passes of two or three: the ranking grows with n^2 (measured 17 us at 8192 tokens, 46 at 13600),
    // a pass takes 7 us up to 32768 tokens and about 15 at 100000.
    rank = n <= (vocab[0] < 256 && (count < 2 || vocab[1] < 256) ? RANK_MAX / 2 : RANK_MAX);
    tiles = (n + RT - 1) / RT;
    // Sorted positions per wave: short chunks until the waves fill the chip (21000 tokens: runs kernel 19 us with 64, 11 with 16), long ones, with
    // fewer parts to join, from there.
    chunk = n < 32768 ? 16 : 64;
    auto take = [&](int64_t b) {
      char* p = ws + bytes;
      bytes += (b + 15) / 16 * 16;
      return p;
    };
    for (int i = 0; i < count; ++i) {
      Job& j = jobs.j[i];
      j.vocab = vocab[i];
      for (int k = 0; k < 2; ++k) {
        j.keys[k] = (uint32_t*)take(n * 4);
        j.vals[k] = (uint32_t*)take(n * 4);
      }
      j.span = (int*)take(vocab[i] * 8);
      j.hist = (uint32_t*)take(rank ? 0 : 256 * tiles * 4);
      j.total = (uint32_t*)take(rank ? 0 : 256 * 4);
      j.part = (float*)take(2 * ((n + chunk - 1) / chunk) * dim * 4);
      j.sorted = rank ? 0 : (passes(vocab[i]) - 1) & 1;
    }
  }
  static int passes(int64_t vocab) {                           // keys run up to vocab itself
    int p = 1;
    while (vocab >> (8 * p)) ++p;
    return p;
  }
};

template <typename DT, typename TT, int VEC>
int run_sums(const Layout& lay, int count, const void* dout, int64_t ld, int dim, hipStream_t st) {
  const int ncb = (dim + 64 * VEC - 1) / (64 * VEC);
  const unsigned blocks0 = (unsigned)((lay.jobs.j[0].vocab + ROWS - 1) / ROWS), blocks1 = (unsigned)((lay.jobs.j[1].vocab + ROWS - 1) / ROWS);
  hipLaunchKernelGGL((embed_runs_kernel<DT, TT, VEC>), dim3((unsigned)((lay.n + 4 * lay.chunk - 1) / (4 * lay.chunk)), ncb, count), dim3(256), 0, st,
                     lay.jobs, (int)lay.n, (const DT*)dout, ld, dim, lay.chunk);
  hipLaunchKernelGGL((embed_rows_kernel<TT, VEC>), dim3(blocks0 + blocks1, ncb), dim3(256), 0, st, lay.jobs, dim, lay.chunk, (int)blocks1);
  FFVC_LAUNCH_CHECK();
  return 0;
}

int embed_bwd(const char* who, const void* dout, int dout_dtype, int64_t ld, int64_t n, int dim, int count, const int64_t* const (&ids)[2],
              const int64_t (&vocab)[2], const float (&scale)[2], void* const (&dtable)[2], int table_dtype, void* ws, int64_t ws_bytes, hipStream_t st) {
  FFVC_CHECK_ARG(dout && ws && n > 0 && dim > 0, "%s: bad args", who);
  FFVC_CHECK_ARG(ffvc_dtype_ok(dout_dtype) && ffvc_dtype_ok(table_dtype), "%s: bad dtype", who);
  FFVC_CHECK_ARG(ld >= dim, "%s: rows shorter than dim", who);
  for (int i = 0; i < count; ++i) FFVC_CHECK_ARG(dtable[i] && vocab[i] > 0, "%s: bad args", who);
  FFVC_CHECK_ARG(n < (1ll << 31) && vocab[0] < (1ll << 31) && vocab[1] < (1ll << 31), "%s: token count and vocabulary must stay below 2^31", who);
  FFVC_CHECK_ARG(ffvc_launch_fits((vocab[0] + ROWS - 1) / ROWS + (vocab[1] + ROWS - 1) / ROWS, 256), "%s: too many table rows for one launch", who);
  Layout lay(n, dim, count, vocab, (char*)ws);
  FFVC_CHECK_ARG((uintptr_t)ws % 16 == 0 && ws_bytes >= lay.bytes, "%s: workspace of %lld bytes needed, got %lld", who, (long long)lay.bytes,
                 (long long)ws_bytes);
  auto al = [](const void* p, int dt, int64_t l) { return (uintptr_t)p % 16 == 0 && l % (16 / ffvc_dtype_size(dt)) == 0; };
  bool vec = dim % 8 == 0 && al(dout, dout_dtype, ld);
  int passes = 0;
  for (int i = 0; i < count; ++i) {
    Job& j = lay.jobs.j[i];
    j.ids = ids[i];
    j.scale = scale[i];
    j.dtable = dtable[i];
    vec = vec && al(dtable[i], table_dtype, dim);
    passes = Layout::passes(vocab[i]) > passes ? Layout::passes(vocab[i]) : passes;
  }
  if (lay.rank) {
    const int lds = (int)((n + 127) / 128 * 128 * 4 + 32 * 4);
    static ffvc_lds_once once;
    const int rc = once.set((const void*)embed_rank_kernel, RANK_MAX * 4 + 32 * 4);
    if (rc) return rc;
    hipLaunchKernelGGL(embed_rank_kernel, dim3((unsigned)((n + 31) / 32), 1, count), dim3(1024), lds, st, lay.jobs, (int)n);
  } else {
    const int tiles = (int)lay.tiles, scanned = tiles > 32;    // (few tiles: every workgroup adds up the counts itself, a launch less)
    for (int shift = 0; shift < 8 * passes; shift += 8) {
      hipLaunchKernelGGL(embed_hist_kernel, dim3(tiles, 1, count), dim3(256), 0, st, lay.jobs, n, shift, tiles);
      if (scanned) hipLaunchKernelGGL(embed_scan_kernel, dim3(256, 1, count), dim3(256), 0, st, lay.jobs, shift, tiles);
      hipLaunchKernelGGL(embed_scatter_kernel, dim3(tiles, 1, count), dim3(256), 0, st, lay.jobs, n, shift, tiles, scanned);
    }
  }
  DISPATCH_DT(dout_dtype, DT, DISPATCH_DT(table_dtype, TT, {
    return vec ? run_sums<DT, TT, 8>(lay, count, dout, ld, dim, st) : run_sums<DT, TT, 1>(lay, count, dout, ld, dim, st);
  }));
  return 0;
}

}  // namespace

extern "C" int ffvc_embed_fwd(const void* table, int table_dtype, int64_t ld, int64_t vocab, const int64_t* ids, float scale, const void* pos,
                              int64_t pos_ld, int64_t npos, const int64_t* place, void* out, int out_dtype, int64_t ldo, int64_t n, int dim, void* stream) {
  FFVC_CHECK_ARG(table && ids && out && n > 0 && dim > 0 && vocab > 0, "ffvc_embed_fwd: bad args");
  FFVC_CHECK_ARG(ffvc_dtype_ok(table_dtype) && ffvc_dtype_ok(out_dtype), "ffvc_embed_fwd: bad dtype");
  FFVC_CHECK_ARG(ld >= dim && ldo >= dim && (!pos || (pos_ld >= dim && npos > 0)), "ffvc_embed_fwd: rows shorter than dim");
  FFVC_CHECK_ARG(ffvc_launch_fits((n + 3) / 4, 256), "ffvc_embed_fwd: too many tokens for one launch (%lld, at most %lld)", (long long)n, 4 * ((1ll << 24) - 1));
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

extern "C" int64_t ffvc_embed_bwd_ws_bytes(int64_t n, int64_t vocab, int dim) {
  return n > 0 && vocab > 0 && dim > 0 ? Layout(n, dim, 1, {vocab, 0}, nullptr).bytes : 0;
}

extern "C" int ffvc_embed_bwd(const void* dout, int dout_dtype, int64_t ld, const int64_t* ids, int64_t n, int64_t vocab, int dim, float scale,
                              void* dtable, int table_dtype, void* ws, int64_t ws_bytes, void* stream) {
  FFVC_CHECK_ARG(ids, "ffvc_embed_bwd: bad args");
  return embed_bwd("ffvc_embed_bwd", dout, dout_dtype, ld, n, dim, 1, {ids, nullptr}, {vocab, 0}, {scale, 0.0f}, {dtable, nullptr}, table_dtype, ws, ws_bytes,
                   (hipStream_t)stream);
}

extern "C" int64_t ffvc_embed_bwd_pair_ws_bytes(int64_t n, int64_t vocab, int64_t npos, int dim) {
  return n > 0 && vocab > 0 && npos > 0 && dim > 0 ? Layout(n, dim, 2, {vocab, npos}, nullptr).bytes : 0;
}

extern "C" int ffvc_embed_bwd_pair(const void* dout, int dout_dtype, int64_t ld, const int64_t* ids, int64_t n, int64_t vocab, int dim, float scale,
                                   void* dtable, const int64_t* place, int64_t npos, void* dpos, int table_dtype, void* ws, int64_t ws_bytes,
                                   void* stream) {
  FFVC_CHECK_ARG(ids, "ffvc_embed_bwd_pair: bad args");
  return embed_bwd("ffvc_embed_bwd_pair", dout, dout_dtype, ld, n, dim, 2, {ids, place}, {vocab, npos}, {scale, 1.0f}, {dtable, dpos}, table_dtype, ws,
                   ws_bytes, (hipStream_t)stream);
}
