// attn_packed.hip — causal attention over PACKED sequences of different lengths with grouped heads, forward and backward.
//
// The rows cu[b] .. cu[b + 1] - 1 of q / k / v are sequence b.  With c = scale * log2(e), query i of a sequence and its keys j <= i:
//     s_ij = q_i . k_j        m_i = max_j s_ij        l_i = sum_j 2^(c (s_ij - m_i))        p_ij = 2^(c (s_ij - m_i)) / l_i
//     o_i  = sum_j p_ij v_j                           lse_i = c m_i + log2 l_i   (kept for the backward: p_ij = 2^(c s_ij - lse_i),
//                                                                                 off by 2^-24 |lse_i| relatively)
//     dv_j = sum_i p_ij do_i      dp_ij = do_i . v_j      delta_i = do_i . o_i      ds_ij = scale p_ij (dp_ij - delta_i)
//     dq_i = sum_j ds_ij k_j      dk_j = sum_i ds_ij q_i  (over the heads / kv_heads query heads that share key head j's group)
//
// Work is cut without knowing the lengths on the host.  The offsets with 0 put before and `rows` behind them bound seqs + 2 pieces: the rows before the
// first sequence, the sequences, the rows behind the last one.  With tiles of BM rows the piece that starts at row c and has i pieces before it owns the
// tile slots from c / BM + i on.  Consecutive pieces never overlap (floor((c + l) / BM) + 1 - floor(c / BM) >= ceil(l / BM)), so the grid is
// rows / BM + seqs + 2 slots and a workgroup finds its piece by a search over the slot starts; a slot past its piece's last tile has
// nothing to do.  Rows of no sequence are zero-filled on request, otherwise left alone.
// Offsets into a tensor are 64 bits wide; inside a tile the buffer descriptor's 32-bit offsets are enough, its record count ends with the
// sequence, so rows past the end (and features past head_dim) read as zeros without a branch.
#include <type_traits>

#include "common.h"

namespace {

#define mma mma_lo<L>

typedef __amdgpu_buffer_rsrc_t rsrc_t;
typedef __attribute__((address_space(3))) void* lds_vp;
typedef __attribute__((address_space(3))) s16x4_t* lds_tr;
constexpr uint32_t OOB = 0xFFFFFFF0u;
constexpr float LOG2E = 1.44269504088896341f;
constexpr float NEG_BIG = -3.0e38f;
// f16 weights are held times 2^F16_UP where a product reads them: below 2^-24 f16 has no bits left, and many small weights are one output
constexpr int F16_UP = 15;
template <typename L>
constexpr bool IS_F16 = std::is_same<L, f16_t>::value;
// Exponents from here on are rounded so coarsely that a weight of 1 may come out as another power of two
constexpr float LONG_EXP = 0x1p20f;
// 64 lanes x 16 (4) bytes from a bounded buffer into consecutive LDS
__device__ __forceinline__ void dma16(rsrc_t r, uint32_t off, unsigned char* lds) { __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_vp)lds, 16, off, 0, 0, 0); }
__device__ __forceinline__ void dma4(rsrc_t r, uint32_t off, float* lds) { __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_vp)lds, 4, off, 0, 0, 0); }
// everything but the N youngest loads of this wave has landed and its LDS reads are done, then everyone's; nothing moves across
template <int N>
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- a tile of rows x DP features in LDS: rows of DP * 2 bytes in lines of 256, 16-byte chunks XOR-swizzled so that both the 16-byte
// row reads (16 rows of one chunk column) and the transposing 8-byte reads (4 rows x 32 bytes) spread over all banks
template <int DP>
__device__ __forceinline__ int tile_off(int row, int chunk) {       // byte offset of 16-byte chunk `chunk` of row `row`
  if constexpr (DP == 128) {
    return row * 256 + ((chunk ^ (((row & 3) << 2) | ((row >> 2) & 3))) << 4);
  } else {
    const int line = row >> 1;
    return line * 256 + (((((row & 1) << 3) | chunk) ^ (((line & 1) << 2) | ((line >> 1) & 3))) << 4);
  }
}
template <int DP>
__device__ __forceinline__ void tile_src(int pos, int& row, int& chunk) {   // the inverse: what 16-byte position `pos` of the tile holds
  const int line = pos >> 4, slot = pos & 15;
  if constexpr (DP == 128) {
    row = line;
    chunk = slot ^ (((row & 3) << 2) | ((row >> 2) & 3));
  } else {
    const int cp = slot ^ (((line & 1) << 2) | ((line >> 1) & 3));
    row = 2 * line + (cp >> 3);
    chunk = cp & 7;
  }
}

// LDS-DMA of one tile by NW waves: piece i of a wave fills 64 consecutive chunk positions; the lane's source offset inside the tile is fixed
template <int DP, int NW, int ROWS>
struct TileDma {
  static constexpr int NP = ROWS * DP / 8 / 64 / NW;
  uint32_t off[NP];
  __device__ __forceinline__ void init(int64_t rs, int D, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      int row, chunk;
      tile_src<DP>((wave * NP + i) * 64 + lane, row, chunk);
      off[i] = chunk * 8 < D ? (uint32_t)((row * rs + chunk * 8) * 2) : OOB;
    }
  }
  // base: element (row0, feature 0) of the tile; live: rows of the sequence from row0 on (none: zeros)
  __device__ __forceinline__ void issue(const uint16_t* base, int64_t rs, int D, int64_t live, unsigned char* tile, int wave) {
    const int64_t bytes = live > 0 ? ((live < ROWS ? live : ROWS) - 1) * rs * 2 + D * 2 : 0;
    const rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (int)bytes, 0x00020000);
#pragma unroll
    for (int i = 0; i < NP; ++i)
      dma16(r, off[i], tile + (wave * NP + i) * 1024);
  }
};

// A fragment (rows of the tile): features 16 s + 8 h .. + 7 of row `row`
template <int DP>
__device__ __forceinline__ u32x4_t frag_rows(const unsigned char* tile, int row, int s, int h) {
  return *(const u32x4_t*)(tile + tile_off<DP>(row, 2 * s + h));
}
// A fragment of the transposed tile: lane -> feature 32 dt + lane % 32, elements = rows r0 + 4 h + {0..3} and r0 + 8 + 4 h + {0..3}: the
// order in which eight consecutive accumulator registers of a 32 x 32 product run over its rows, so those are the B fragment as they are
template <int DP>
__device__ __forceinline__ u32x4_t frag_cols(const unsigned char* tile, int dt, int r0, int lane) {
  const int c = lane & 15, h = lane >> 5;
  const int d = 32 * dt + 16 * ((lane >> 4) & 1) + 4 * (c & 3);
  const int row = r0 + 4 * h + (c >> 2);
  union {
    s16x4_t x[2];
    u32x4_t v;
  } u;
  u.x[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr)(tile + tile_off<DP>(row, d >> 3) + (d & 7) * 2));
  u.x[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr)(tile + tile_off<DP>(row + 8, d >> 3) + (d & 7) * 2));
  return u.v;
}

template <typename L>
__device__ __forceinline__ u32x4_t pack8(const f32x16_t& t, int first) {
  u32x4_t r;
#pragma unroll
  for (int e = 0; e < 4; ++e) r[e] = lo_pack2<L>(t[first + 2 * e], t[first + 2 * e + 1]);
  return r;
}

__device__ __forceinline__ void zero16(f32x16_t& t) {
#pragma unroll
  for (int r = 0; r < 16; ++r) t[r] = 0.0f;
}
__device__ __forceinline__ int acc_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// the other half-wave's value of the same column
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }

struct Place {
  int64_t row0;      // first row of the sequence
  int64_t len;       // its rows
  int64_t tile;      // tile inside the sequence
  bool outside;      // rows of no sequence: before the first or behind the last one
};

__device__ __forceinline__ int64_t cu_at(const int32_t* cu, int b, int64_t rows) {
  const int64_t c = cu[b];
  return c < 0 ? 0 : (c > rows ? rows : c);
}

// slot -> (piece, tile).  64 probes at a time; a cu that is not ascending gives some sequence's clamped rows, never one outside [0, rows).
template <int BM>
__device__ __forceinline__ Place find_slot(const int32_t* __restrict__ cu, int seqs, int64_t rows, int64_t slot) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = seqs + 2;                       // candidates lo .. lo + n - 1; piece i is sequence i - 1
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int b = lo + lane * step;
    const bool le = lane * step < n && (b ? cu_at(cu, b - 1, rows) : 0) / BM + b <= slot;
    const uint64_t m = __ballot(le) | 1ull;       // (candidate lo always holds)
    const int k = 63 - __builtin_clzll(m);
    lo += k * step;
    n = min(step, n - k * step);
  }
  lo = __builtin_amdgcn_readfirstlane(lo);
  Place p;
  p.row0 = lo ? cu_at(cu, lo - 1, rows) : 0;
  const int64_t end = lo <= seqs ? cu_at(cu, lo, rows) : rows;
  p.len = end > p.row0 ? end - p.row0 : 0;
  p.tile = slot - (p.row0 / BM + lo);
  p.outside = lo == 0 || lo > seqs;
  return p;
}

// The r-th longest piece of work: tiles in the order of their walks' lengths, so that the last ones to start are short (KEYS: a key tile's walk is
// over the rows from it on, otherwise over the rows up to it).  Among 2 .. 63 sequences, level j holds the tiles with j others of their sequence on
// their walk; cum(j) = sum_b max(tiles_b - j, 0) counts the levels from j on, 64 probes at a time.  A single sequence is in order as it is.
template <int BM, bool KEYS>
__device__ __forceinline__ Place find_tile(const int32_t* __restrict__ cu, int seqs, int64_t rows, int64_t slots, int64_t r) {
  if (seqs == 1 || seqs > 63) return find_slot<BM>(cu, seqs, rows, KEYS ? r : slots - 1 - r);
  const int lane = threadIdx.x & 63;
  const int c0 = (int)(lane <= seqs ? cu_at(cu, lane, rows) : rows);
  const int c1 = (int)(lane < seqs ? cu_at(cu, lane + 1, rows) : rows);
  const int tiles = lane < seqs && c1 > c0 ? (int)(((int64_t)c1 - c0 + BM - 1) / BM) : 0;
  Place p;
  int lo = 0, n = (int)(rows / BM) + 1, at = 0;        // levels lo .. lo + n - 1; cum(lo)
  do {
    const int step = (n + 63) / 64, j = lo + lane * step;
    int cum = 0;
    for (int b = 0; b < seqs; ++b) cum += max(__builtin_amdgcn_readlane(tiles, b) - j, 0);
    const uint64_t m = __ballot(lane * step < n && cum > r);
    if (m == 0) {                                       // behind all tiles: the rows behind the last sequence, then those before the first one
      const int last = __builtin_amdgcn_readlane(c0, seqs);
      const int64_t behind = (rows - last + BM - 1) / BM;
      p.tile = r - __builtin_amdgcn_readlane(cum, 0);
      const bool head = p.tile >= behind;
      p.row0 = head ? 0 : last;
      p.len = head ? __builtin_amdgcn_readlane(c0, 0) : rows - last;
      p.tile -= head ? behind : 0;
      p.outside = true;
      return p;
    }
    const int k = 63 - __builtin_clzll(m);
    at = __builtin_amdgcn_readlane(cum, k);
    lo += k * step;
    n = min(step, n - k * step);
  } while (n > 1);
  const uint64_t level = __ballot(tiles > lo);
  const int rank = (int)(r - (at - __popcll(level)));
  const bool mine = ((level >> lane) & 1) && __popcll(level & ((1ull << lane) - 1)) == rank;
  const int b = __builtin_ctzll(__ballot(mine) | 1ull << 63);
  p.row0 = __builtin_amdgcn_readlane(c0, b);
  p.len = __builtin_amdgcn_readlane(c1, b) - p.row0;
  p.tile = KEYS ? __builtin_amdgcn_readlane(tiles, b) - 1 - lo : lo;
  p.outside = false;
  return p;
}

// block -> (rank of the tile, head).  Consecutive workgroups go to the 8 XCDs in turn: with a multiple of 8 heads each XCD keeps heads / 8
// neighbouring heads, so the heads of one key / value group read it through one L2.
__device__ __forceinline__ void block_place(int heads, int64_t& rank, int& head) {
  const int64_t i = blockIdx.x;
  const int j = (int)(i % heads);
  head = heads % 8 == 0 ? (j & 7) * (heads >> 3) + (j >> 3) : j;
  rank = i / heads;
}

// o[row0 + lane % 32][32 dt + ...] = acc, rows < n; the wave's tile is transposed (lane = row, registers = features)
template <typename L, int DP>
__device__ __forceinline__ void store_rows(uint16_t* base, int64_t rs, int D, const f32x16_t (&acc)[DP / 32], int row, bool ok, int h) {
  if (!ok) return;
  uint16_t* p = base + row * rs;
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + 8 * g + 4 * h;
      if (d < D) {
        u32x2_t v;
        v[0] = lo_pack2<L>(acc[dt][4 * g], acc[dt][4 * g + 1]);
        v[1] = lo_pack2<L>(acc[dt][4 * g + 2], acc[dt][4 * g + 3]);
        *(u32x2_t*)(p + d) = v;
      }
    }
}

__device__ __forceinline__ void zero_rows(uint16_t* base, int64_t rs, int D, int64_t nrows, int tid, int threads) {
  const int ch = D / 8;
  const u32x4_t z = {0u, 0u, 0u, 0u};
  for (int64_t i = tid; i < nrows * ch; i += threads) {
    const int64_t r = i / ch;
    *(u32x4_t*)(base + r * rs + (i - r * ch) * 8) = z;
  }
}

// eight features of row `row` (16 s + 8 h ..) of one head; zeros past the sequence or past head_dim
__device__ __forceinline__ u32x4_t row_frag(const uint16_t* base, int64_t rs, int64_t row, bool ok, int s, int h, int D) {
  const u32x4_t z = {0u, 0u, 0u, 0u};
  const int d = 16 * s + 8 * h;
  return ok && d < D ? *(const u32x4_t*)(base + row * rs + d) : z;
}

// whether the lane's accumulators hold an inf or a NaN
template <int ND>
__device__ __forceinline__ bool nonfinite(const f32x16_t (&acc)[ND]) {
  float z = 0.0f;
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) z = fmaf(acc[t][r], 0.0f, z);        // 0 * inf = NaN
  return !(z == 0.0f);
}

// ---- rows next to a non-finite value ---------------------------------------------------------------------------------------------------
// On the diagonal a tile multiplies masked weights of 0 with rows that their queries (keys) must not see; where such a row holds an inf or a NaN
// the product is NaN.  A wave whose result is not finite therefore looks at those rows, and only if one of them is not finite either does it
// sum its rows again without them: a lane per partner for the weights, a lane per feature for the sums.  (Values the row does see, the
// common way to a NaN, leave the check after at most 95 rows read.)

// any non-finite value in rows r0 .. r1 - 1 (at most 95) of one head
template <typename L>
__device__ __forceinline__ bool any_nonfinite(const uint16_t* base, int64_t rs, int D, int64_t r0, int64_t r1, int lane) {
  bool bad = false;
  for (int64_t r = r0; r < r1; ++r)
    for (int d = lane; d < D; d += 64) {
      const float v = lo_unpack<L>(base[r * rs + d]);
      bad |= !(fabsf(v) <= 3.4028235e38f);
    }
  return __any(bad);
}
template <typename L>
__device__ __forceinline__ float dot_rows(const uint16_t* a, const uint16_t* b, int D) {
  float s = 0.0f;
  for (int d = 0; d < D; d += 8) {
    const f32x8 x = unpack8<L>(*(const u32x4_t*)(a + d)), y = unpack8<L>(*(const u32x4_t*)(b + d));
#pragma unroll
    for (int e = 0; e < 8; ++e) s = fmaf(x.v[e], y.v[e], s);
  }
  return s;
}
// o[e] += sum over the 64 lanes' weights of w * row[lane + 64 e]; lane j's row is base + (j0 + j) * rs, n of them
template <typename L>
__device__ __forceinline__ void add_weighted(float (&o)[2], float w, const uint16_t* base, int64_t rs, int D, int n, int lane) {
  for (int j = 0; j < n; ++j) {
    const float wj = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), j));
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < D) o[e] = fmaf(wj, lo_unpack<L>(base[j * rs + lane + 64 * e]), o[e]);
  }
}
// nothing left to learn about a row: a NaN stays one (a tensor full of them costs a wave one chunk per row)
__device__ __forceinline__ bool all_nan(const float (&o)[2], int D, int lane) {
  return __all((lane >= D || o[0] != o[0]) && (lane + 64 >= D || o[1] != o[1]));
}
template <typename L>
__device__ __forceinline__ void put_row(uint16_t* row, const float (&o)[2], float mul, int D, int lane) {
#pragma unroll
  for (int e = 0; e < 2; ++e)
    if (lane + 64 * e < D) row[lane + 64 * e] = (uint16_t)(lo_pack2<L>(o[e] * mul, 0.0f) & 0xffffu);
}

// outputs of queries i0 .. i1 - 1 from their own keys alone
template <typename L>
__device__ __forceinline__ void redo_out(const uint16_t* Q, int64_t q_rs, const uint16_t* K, int64_t k_rs, const uint16_t* V, int64_t v_rs, uint16_t* O,
                                         int64_t o_rs, int D, float c, int64_t i0, int64_t i1, int lane) {
  for (int64_t i = i0; i < i1; ++i) {
    float m = NEG_BIG, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (int64_t j0 = 0; j0 <= i; j0 += 64) {
      const int n = (int)(i - j0 < 63 ? i - j0 + 1 : 64);
      const float s = lane < n ? dot_rows<L>(Q + i * q_rs, K + (j0 + lane) * k_rs, D) : -INFINITY;
      const float mx = fmaxf(m, wave_max(s)), a = __builtin_amdgcn_exp2f((m - mx) * c);
      const float w = lane < n ? __builtin_amdgcn_exp2f((s - mx) * c) : 0.0f;
      m = mx;
      l = l * a + wave_sum(w);
      o[0] *= a;
      o[1] *= a;
      add_weighted<L>(o, w, V + j0 * v_rs, v_rs, D, n, lane);
      if (all_nan(o, D, lane)) break;
    }
    put_row<L>(O + i * o_rs, o, 1.0f / l, D, lane);
  }
}

// ---- forward -------------------------------------------------------------------------------------------------------------------
// The weights are rounded to the 16-bit type, as the matrix instructions take them; their sum l is not.
// NW waves x 32 queries; key / value tiles of KB = 64 rows in a ring of NST LDS slots, filled by LDS-DMA NST - 1 tiles ahead.  Every variant takes a
// row's keys 64 at a time in the same steps, so a sequence's output does not depend on what it is packed with.
// Bound by the softmax arithmetic beside the matrix instructions at two (128 features) or three waves per SIMD: 8192 rows, 16 heads of 128, 337 us
// (816 TFLOP/s of visible pairs; medians of a kernel trace); two sequences of 16000, 32 heads, 4.26 ms (970); of 64 features 199 us (690).
template <typename L, int DP, int NW, int NST, int KB>
__global__ __launch_bounds__(64 * NW, 2) void attn_packed_fwd_kernel(const ffvc_attn_packed_desc p, int64_t slots) {
  constexpr int BM = 32 * NW, NS = DP / 16, ND = DP / 32, TB = KB * DP * 2;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t rank;
  int head;
  block_place(p.heads, rank, head);
  const Place pl = find_slot<BM>(p.cu, p.seqs, p.rows, slots - 1 - rank);      // (a sequence's last tiles, with the longest walks, first)
  const int64_t q0 = pl.tile * BM;
  if (q0 < 0 || q0 >= pl.len) return;
  const int D = p.head_dim;
  uint16_t* O = (uint16_t*)p.out + pl.row0 * p.o_rs + head * p.o_hs;
  if (pl.outside) {
    if (p.zero_tail) zero_rows(O + q0 * p.o_rs, p.o_rs, D, pl.len - q0 < BM ? pl.len - q0 : BM, tid, 64 * NW);
    return;
  }
  const int kvh = head / (p.heads / p.kv_heads);
  const uint16_t* Q = (const uint16_t*)p.q + pl.row0 * p.q_rs + head * p.q_hs;
  const uint16_t* Kp = (const uint16_t*)p.k + pl.row0 * p.k_rs + kvh * p.k_hs;
  const uint16_t* V = (const uint16_t*)p.v + pl.row0 * p.v_rs + kvh * p.v_hs;
  const float c = p.scale * LOG2E;
  TileDma<DP, NW, KB> dk, dv;
  dk.init(p.k_rs, D, wave, lane);
  dv.init(p.v_rs, D, wave, lane);
  const int64_t qend = q0 + BM < pl.len ? q0 + BM : pl.len;
  const int nkb = (int)((qend + KB - 1) / KB);
  constexpr int PIECES = 2 * TileDma<DP, NW, KB>::NP;
  int slot_in = 0, slot_out = 0;                           // LDS slots filled / read next
  auto issue = [&](int kb) {                               // (tiles past the last one fetch zeros: the counts stay the same)
    const int64_t k0 = kb < nkb ? (int64_t)kb * KB : 0, live = kb < nkb ? pl.len - k0 : 0;
    unsigned char* st = smem + slot_in * 2 * TB;
    dk.issue(Kp + k0 * p.k_rs, p.k_rs, D, live, st, wave);
    dv.issue(V + k0 * p.v_rs, p.v_rs, D, live, st + TB, wave);
    slot_in = slot_in + 1 == NST ? 0 : slot_in + 1;
  };
#pragma unroll
  for (int i = 0; i < (NST > 1 ? NST - 1 : 1); ++i) issue(i);
  const int64_t qw = q0 + 32 * wave;                       // this wave's first query
  const int64_t qi = qw + l31;
  const bool ok = qi < pl.len;
  u32x4_t fq[NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) fq[s] = row_frag(Q, p.q_rs, qi, ok, s, h, D);
  f32x16_t acc[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) zero16(acc[t]);
  float m = NEG_BIG, l = 0.0f;
  // NH: 32-key halves of the tile that any query of the wave sees (the second one is all later keys where the wave starts on the tile's first row:
  // leaving it out gives the same bits)
  auto tile = [&](auto halves, const unsigned char* sk, const unsigned char* sv, int64_t k0) {
    constexpr int NH = decltype(halves)::value;
    f32x16_t S[NH];
#pragma unroll
    for (int kt = 0; kt < NH; ++kt) {
      zero16(S[kt]);
#pragma unroll
      for (int s = 0; s < NS; ++s) mma(S[kt], frag_rows<DP>(sk, 32 * kt + l31, s, h), fq[s]);
    }
    if (k0 + 32 * NH - 1 > qw) {                           // the diagonal crosses this tile
      const int lim = (int)(qi - k0);                      // last visible key of this lane's query
#pragma unroll
      for (int kt = 0; kt < NH; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[kt][r] = 32 * kt + acc_row(r, h) <= lim ? S[kt][r] : -INFINITY;
    }
    float mx = m;
#pragma unroll
    for (int kt = 0; kt < NH; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, S[kt][r]);
    mx = fmaxf(mx, other_half(mx));
    if (__any(mx > m)) {                                   // most tiles of a long row leave the maximum alone
      const float a = __builtin_amdgcn_exp2f((m - mx) * c);
      l *= a;
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] *= a;
      m = mx;
    }
    constexpr float UP = IS_F16<L> ? F16_UP : 0.0f;
    float mc = IS_F16<L> ? fmaf(m, c, -UP) : m * c;
    if (__builtin_expect(__any(fabsf(mc) > LONG_EXP), 0)) { // the difference first, then: the row's largest weight is 1 (2^UP) whatever the scores are
      const float sub = fabsf(mc) > LONG_EXP ? m : 0.0f;
      mc = fabsf(mc) > LONG_EXP ? -UP : mc;
#pragma unroll
      for (int kt = 0; kt < NH; ++kt)
#pragma unroll
        for (int r = 0; r < 16; ++r) S[kt][r] -= sub;
    }
    float sum = 0.0f;
#pragma unroll
    for (int kt = 0; kt < NH; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        S[kt][r] = __builtin_amdgcn_exp2f(fmaf(S[kt][r], c, -mc));
        sum += S[kt][r];
      }
    l += sum;
#pragma unroll
    for (int kt = 0; kt < NH; ++kt)
#pragma unroll
      for (int sg = 0; sg < 2; ++sg) {
        const u32x4_t fp = pack8<L>(S[kt], 8 * sg);
#pragma unroll
        for (int t = 0; t < ND; ++t) mma(acc[t], frag_cols<DP>(sv, t, 32 * kt + 16 * sg, lane), fp);
      }
  };
#pragma unroll 1
  for (int kb = 0; kb < nkb; ++kb) {
    arrive<(NST > 2 ? NST - 2 : 0) * PIECES>();
    if constexpr (NST > 1) issue(kb + NST - 1);
    const unsigned char* sk = smem + slot_out * 2 * TB;
    const unsigned char* sv = sk + TB;
    slot_out = slot_out + 1 == NST ? 0 : slot_out + 1;
    const int64_t k0 = (int64_t)kb * KB;
    if (k0 <= qw + 31 && qw < pl.len) {                    // (otherwise every key of the tile is later than this wave's queries)
      // (one wave at 64 features: elsewhere the second body costs the long rows more, 4.6 against 4.1 ms, than it saves)
      if (NW > 1 || DP > 64 || k0 + 32 <= qw + 31)
        tile(std::integral_constant<int, 2>{}, sk, sv, k0);
      else
        tile(std::integral_constant<int, 1>{}, sk, sv, k0);
    }
    if constexpr (NST == 1) {
      arrive<0>();
      if (kb + 1 < nkb) issue(kb + 1);
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // no load may outlive the workgroup's LDS
  l += other_half(l);
  const float inv = 1.0f / l;
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] *= inv;
  if (p.lse && ok && h == 0) p.lse[(int64_t)head * p.rows + pl.row0 + qi] = m * c + (__builtin_amdgcn_logf(l) - (IS_F16<L> ? (float)F16_UP : 0.0f));
  store_rows<L, DP>(O + qw * p.o_rs, p.o_rs, D, acc, l31, ok, h);
  if (__any(ok && nonfinite<ND>(acc))) {
    const int64_t far = (qw / KB + 1) * KB, last = far < pl.len ? far : pl.len;       // keys past qw that its last tile holds
    if (any_nonfinite<L>(V, p.v_rs, D, qw + 1, last, lane))
      redo_out<L>(Q, p.q_rs, Kp, p.k_rs, V, p.v_rs, O, p.o_rs, D, c, qw, qw + 32 < pl.len ? qw + 32 : pl.len, lane);
  }
}

// ---- the range of f16 in the backward -----------------------------------------------------------------------------------------------------
// P and dS are rounded to the 16-bit type, for the matrix instructions that multiply them with 16-bit rows: one rounding per weight.  bf16 has the range
// of fp32; in f16 a dS of 65520 is infinite and one below 2^-24 has no bits left, though the sums that it belongs to fit.  So f16 weights carry a
// power of two, 2^BWD_UP at first, per query (dq) or key (dk, dv): it enters through the exponent, or through the accumulator that the scores start
// from, and is taken out of the sums.  A tile whose largest |f dS| passes 2^15 (|dS| > 1: loss-scaled gradients) lowers the factor and what has
// been summed so far.  Cost, dq + dk / dv of 8192 rows with 16 heads: 516 -> 556 us with 64 features, 967 -> 993 with 128 (the maximum; the branch is
// taken a few times per walk at most); bf16 compiles without it.
// (Less than the forward's: a weight of the backward passes 1 by the rounding of its exponent, a power of two from exponents of 2^24 on.)
constexpr int BWD_UP = 12;
// 0, or the (negative) power by which the lane's factor has to change; the half-waves share their column
__device__ __forceinline__ int lower_by(const f32x16_t& t) {
  float mx = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(t[r]));
  if (__builtin_expect(!__any(mx > 32768.0f), 1)) return 0;
  mx = fmaxf(mx, other_half(mx));
  return mx > 32768.0f && mx < INFINITY ? 15 - __builtin_amdgcn_frexp_expf(mx) : 0;         // (an inf stays one)
}
template <int N>
__device__ __forceinline__ void scale_all(f32x16_t (&t)[N], float by) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) t[i][r] *= by;
}

// ---- backward: dq (and delta) ----------------------------------------------------------------------------------------------------
// acc of part 0 += the other parts', in order, through [part - 1][wave][register][lane] over the stages nobody reads any more
template <int ND, int NW, int SPLIT>
__device__ __forceinline__ void join_parts(f32x16_t (&acc)[ND], float* mem, int wave, int part, int lane) {
  constexpr int W = ND * 16 * 64;
  float* join = mem + wave * W + lane;
  __syncthreads();
  if (part)
#pragma unroll
    for (int t = 0; t < ND; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) join[(part - 1) * NW * W + (t * 16 + r) * 64] = acc[t][r];
  __syncthreads();
  if (!part)
#pragma unroll
    for (int o = 0; o < SPLIT - 1; ++o)
#pragma unroll
      for (int t = 0; t < ND; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[t][r] += join[o * NW * W + (t * 16 + r) * 64];
}

// delta is taken from the output as it is stored, in 16 bits: the exact one would need the output in 32 bits or another walk.  In bf16 gradients are then
// off by 0.0025 (relative norm), by 0.0023 with the exact delta, by 0.0017 with nothing rounded but themselves; the rest is P's and dS's rounding.
// The forward's walk once more with three products per tile (s, dp, dq): 8192 rows, 16 heads of 128, 412 us (1000 TFLOP/s); of 64 features 200 us.
// SPLIT = 2: twice NW waves, each NW of them take every other key tile of the same queries; the sums join in LDS at the end (run_bwd has the rule).
template <typename L, int DP, int NW, int NST, int KB, int SPLIT>
__global__ __launch_bounds__(64 * NW * SPLIT, DP == 64 && SPLIT == 1 ? 3 : 2) void attn_packed_dq_kernel(const ffvc_attn_packed_desc p, int64_t slots) {
  constexpr int BM = 32 * NW, NS = DP / 16, ND = DP / 32, TB = KB * DP * 2;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem_all[];
  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
  const int wave_all = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wave_all % NW, part = wave_all / NW;
  unsigned char* smem = smem_all + part * (NST * 2 * TB);
  int64_t rank;
  int head;
  block_place(p.heads, rank, head);
  const Place pl = find_tile<BM, false>(p.cu, p.seqs, p.rows, slots, rank);
  const int64_t q0 = pl.tile * BM;
  if (q0 < 0 || q0 >= pl.len) return;
  const int D = p.head_dim;
  uint16_t* dQ = (uint16_t*)p.dq + pl.row0 * p.dq_rs + head * p.dq_hs;
  if (pl.outside) {
    if (p.zero_tail) zero_rows(dQ + q0 * p.dq_rs, p.dq_rs, D, pl.len - q0 < BM ? pl.len - q0 : BM, tid, 64 * NW * SPLIT);
    return;
  }
  const int kvh = head / (p.heads / p.kv_heads);
  const uint16_t* Q = (const uint16_t*)p.q + pl.row0 * p.q_rs + head * p.q_hs;
  const uint16_t* Kp = (const uint16_t*)p.k + pl.row0 * p.k_rs + kvh * p.k_hs;
  const uint16_t* V = (const uint16_t*)p.v + pl.row0 * p.v_rs + kvh * p.v_hs;
  const uint16_t* Oh = (const uint16_t*)p.out + pl.row0 * p.o_rs + head * p.o_hs;
  const uint16_t* dO = (const uint16_t*)p.dout + pl.row0 * p.do_rs + head * p.do_hs;
  const float c = p.scale * LOG2E;
  TileDma<DP, NW, KB> dk, dv;
  dk.init(p.k_rs, D, wave, lane);
  dv.init(p.v_rs, D, wave, lane);
  const int64_t qend = q0 + BM < pl.len ? q0 + BM : pl.len;
  const int nkb = (int)((qend + KB - 1) / KB), steps = (nkb + SPLIT - 1) / SPLIT;
  constexpr int PIECES = 2 * TileDma<DP, NW, KB>::NP;
  int slot_in = 0, slot_out = 0;                           // LDS slots filled / read next
  auto issue = [&](int it) {                               // (tiles past the last one fetch zeros: the counts stay the same)
    const int kb = it * SPLIT + part;
    const int64_t k0 = kb < nkb ? (int64_t)kb * KB : 0, live = kb < nkb ? pl.len - k0 : 0;
    unsigned char* st = smem + slot_in * 2 * TB;
    dk.issue(Kp + k0 * p.k_rs, p.k_rs, D, live, st, wave);
    dv.issue(V + k0 * p.v_rs, p.v_rs, D, live, st + TB, wave);
    slot_in = slot_in + 1 == NST ? 0 : slot_in + 1;
  };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) issue(i);
  const int64_t qw = q0 + 32 * wave;
  const int64_t qi = qw + l31;
  const bool ok = qi < pl.len;
  const int64_t stat = (int64_t)head * p.rows + pl.row0 + qi;
  u32x4_t fq[NS], fo[NS];
  float dl = 0.0f;
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    fq[s] = row_frag(Q, p.q_rs, qi, ok, s, h, D);
    fo[s] = row_frag(dO, p.do_rs, qi, ok, s, h, D);
    const f32x8 a = unpack8<L>(row_frag(Oh, p.o_rs, qi, ok, s, h, D)), b = unpack8<L>(fo[s]);
#pragma unroll
    for (int e = 0; e < 8; ++e) dl = fmaf(a.v[e], b.v[e], dl);
  }
  dl += other_half(dl);
  float ls = ok ? p.lse[stat] : 0.0f;
  if constexpr (IS_F16<L>) ls -= (float)BWD_UP;
  if (ok && h == 0 && part == 0) p.delta[stat] = -dl;                   // (negative: the accumulator of dp starts from it)
  f32x16_t acc[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) zero16(acc[t]);
#pragma unroll 1
  for (int it = 0; it < steps; ++it) {
    arrive<(NST - 2) * PIECES>();
    issue(it + NST - 1);
    const unsigned char* sk = smem + slot_out * 2 * TB;
    const unsigned char* sv = sk + TB;
    slot_out = slot_out + 1 == NST ? 0 : slot_out + 1;
    const int64_t k0 = (int64_t)(it * SPLIT + part) * KB;
    if (k0 > qw + 31 || qw >= pl.len) continue;
    const bool diag = k0 + KB - 1 > qw;
    const int lim = (int)(qi - k0);
#pragma unroll
    for (int kt = 0; kt < KB / 32; ++kt) {
      if (kt && k0 + 32 * kt > qw + 31) break;              // a half of later keys only
      f32x16_t S, dP;
      zero16(S);
#pragma unroll
      for (int r = 0; r < 16; ++r) dP[r] = -dl;
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        mma(S, frag_rows<DP>(sk, 32 * kt + l31, s, h), fq[s]);
        mma(dP, frag_rows<DP>(sv, 32 * kt + l31, s, h), fo[s]);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) dP[r] *= __builtin_amdgcn_exp2f(fmaf(S[r], c, -ls));      // ds / scale
      if (diag) {
#pragma unroll
        for (int r = 0; r < 16; ++r) dP[r] = 32 * kt + acc_row(r, h) > lim ? 0.0f : dP[r];
      }
      if constexpr (IS_F16<L>) {
        const int e = lower_by(dP);
        if (__builtin_expect(__any(e != 0), 0)) {
          const float by = ldexpf(1.0f, e);
#pragma unroll
          for (int r = 0; r < 16; ++r) dP[r] *= by;
          scale_all<ND>(acc, by);
          ls -= (float)e;
        }
      }
#pragma unroll
      for (int sg = 0; sg < 2; ++sg) {
        const u32x4_t fs = pack8<L>(dP, 8 * sg);
#pragma unroll
        for (int t = 0; t < ND; ++t) mma(acc[t], frag_cols<DP>(sk, t, 32 * kt + 16 * sg, lane), fs);
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if constexpr (IS_F16<L>) scale_all<ND>(acc, ldexpf(1.0f, (int)rintf(ls - (ok ? p.lse[stat] : 0.0f))));
  if constexpr (SPLIT > 1) {
    join_parts<ND, NW, SPLIT>(acc, (float*)smem_all, wave, part, lane);
    if (part) return;
  }
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[t][r] *= p.scale;
  store_rows<L, DP>(dQ + qw * p.dq_rs, p.dq_rs, D, acc, l31, ok, h);
  if (__any(ok && nonfinite<ND>(acc))) {
    const int64_t far = (qw / KB + 1) * KB, last = far < pl.len ? far : pl.len;
    if (any_nonfinite<L>(Kp, p.k_rs, D, qw + 1, last, lane))
      for (int64_t i = qw; i < qw + 32 && i < pl.len; ++i) {                           // dq of these queries from their own keys alone
        const float li = p.lse[(int64_t)head * p.rows + pl.row0 + i];
        const float di = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(dl), (int)(i - qw)));
        float o[2] = {0.0f, 0.0f};
        for (int64_t j0 = 0; j0 <= i; j0 += 64) {
          const int n = (int)(i - j0 < 63 ? i - j0 + 1 : 64);
          float w = 0.0f;
          if (lane < n) {
            const float pr = __builtin_amdgcn_exp2f(fmaf(dot_rows<L>(Q + i * p.q_rs, Kp + (j0 + lane) * p.k_rs, D), c, -li));
            w = pr * (dot_rows<L>(dO + i * p.do_rs, V + (j0 + lane) * p.v_rs, D) - di);
          }
          add_weighted<L>(o, w, Kp + j0 * p.k_rs, p.k_rs, D, n, lane);
          if (all_nan(o, D, lane)) break;
        }
        put_row<L>(dQ + i * p.dq_rs, o, p.scale, D, lane);
      }
  }
}

// ---- backward: dk, dv --------------------------------------------------------------------------------------------------------------
// NW waves x 32 keys of one key / value head; walks the query tiles (QB rows of q and dout, two LDS stages) that see them, for every query head
// of the group.  K stays in registers as the B operand of s = q k^T.  V, the B operand of dp = do v^T, stays there too at 64 features; at 128 both
// next to the two accumulators would take more than half the register file, and one wave per SIMD cannot hide its own waits: V lies in LDS
// (8192 rows, 16 heads of 128: 963 us with V in registers, 560 to 587 in LDS) and a step takes 32 queries, not 64.
//
// SPLIT > 1: SPLIT * NW waves, each NW of them take every SPLIT-th (head, query tile) of the same keys; the sums join in LDS at the end, in order.
// (run_bwd has the rule and its figures.)  Four products per tile: 8192 rows, 16 heads of 128, 587 us (936 TFLOP/s).
template <typename L, int DP, int NW, int NST, int QB, bool VLDS, int SPLIT>
__global__ __launch_bounds__(64 * NW * SPLIT, 2) void attn_packed_dkv_kernel(const ffvc_attn_packed_desc p, int64_t slots) {
  constexpr int BM = 32 * NW, NS = DP / 16, ND = DP / 32, TB = QB * DP * 2, VB = VLDS ? BM * DP * 2 : 0;
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem_all[];
  const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
  const int wave_all = __builtin_amdgcn_readfirstlane(tid >> 6), wave = wave_all % NW, part = wave_all / NW;
  unsigned char* smem = smem_all + part * (NST * 2 * TB);
  unsigned char* vmem = smem_all + SPLIT * (NST * 2 * TB);
  float* stat = (float*)(vmem + VB) + part * (NST * 2 * 64); // [slots][lse | delta][64]
  int64_t rank;
  int kvh;
  block_place(p.kv_heads, rank, kvh);
  const Place pl = find_tile<BM, true>(p.cu, p.seqs, p.rows, slots, rank);
  const int64_t k0 = pl.tile * BM;
  if (k0 < 0 || k0 >= pl.len) return;
  const int D = p.head_dim;
  uint16_t* dK = (uint16_t*)p.dk + pl.row0 * p.dk_rs + kvh * p.dk_hs;
  uint16_t* dV = (uint16_t*)p.dv + pl.row0 * p.dv_rs + kvh * p.dv_hs;
  if (pl.outside) {
    if (p.zero_tail) {
      const int64_t n = pl.len - k0 < BM ? pl.len - k0 : BM;
      zero_rows(dK + k0 * p.dk_rs, p.dk_rs, D, n, tid, 64 * NW * SPLIT);
      zero_rows(dV + k0 * p.dv_rs, p.dv_rs, D, n, tid, 64 * NW * SPLIT);
    }
    return;
  }
  const uint16_t* Kp = (const uint16_t*)p.k + pl.row0 * p.k_rs + kvh * p.k_hs;
  const uint16_t* V = (const uint16_t*)p.v + pl.row0 * p.v_rs + kvh * p.v_hs;
  const int group = p.heads / p.kv_heads;
  const float c = p.scale * LOG2E;
  TileDma<DP, NW, QB> dq, dd;
  dq.init(p.q_rs, D, wave, lane);
  dd.init(p.do_rs, D, wave, lane);
  if constexpr (VLDS) {
    TileDma<DP, NW * SPLIT, BM> dv;
    dv.init(p.v_rs, D, wave_all, lane);
    dv.issue(V + k0 * p.v_rs, p.v_rs, D, pl.len - k0, vmem, wave_all);
  }
  const int qb0 = (int)(k0 / QB);                            // first query tile that sees any of these keys
  const int nqb = (int)((pl.len + QB - 1) / QB);
  const int total = (nqb - qb0) * group;
  const int steps = (total + SPLIT - 1) / SPLIT;             // (the last step of the second half may be past the end: zeros)
  auto advance = [&](int& head, int& qb, int by) {
    qb += by;
    while (qb >= nqb) {
      qb -= nqb - qb0;
      ++head;
    }
  };
  int head_i = kvh * group, qb_i = qb0;                      // the next tile to fetch
  if (part) advance(head_i, qb_i, part);
  int head_o = head_i, qb_o = qb_i;                          // the next tile to multiply
  constexpr int PIECES = 2 * TileDma<DP, NW, QB>::NP + (NW == 1 ? 2 : 1);
  int slot_in = 0, slot_out = 0;
  auto issue = [&](int it) {                                 // (steps past the last one fetch zeros: the counts stay the same)
    const bool in = it * SPLIT + part < total;
    const int64_t r0 = in ? (int64_t)qb_i * QB : 0, live = in ? pl.len - r0 : 0;
    const int head = in ? head_i : kvh * group;
    unsigned char* st = smem + slot_in * 2 * TB;
    dq.issue((const uint16_t*)p.q + (pl.row0 + r0) * p.q_rs + head * p.q_hs, p.q_rs, D, live, st, wave);
    dd.issue((const uint16_t*)p.dout + (pl.row0 + r0) * p.do_rs + head * p.do_hs, p.do_rs, D, live, st + TB, wave);
    // even waves their lse, odd ones their delta (the same values to the same place: every wave counts the same loads); zeros past the end
    const int64_t at = (int64_t)head * p.rows + pl.row0 + r0;
    const int n = (int)(live < QB ? live : QB);
    auto fetch = [&](int which) {
      dma4(__builtin_amdgcn_make_buffer_rsrc((void*)((which ? p.delta : p.lse) + at), 0, n * 4, 0x00020000), lane * 4, stat + (slot_in * 2 + which) * 64);
    };
    if constexpr (NW == 1) {
      fetch(0);
      fetch(1);
    } else {
      fetch(wave & 1);
    }
    slot_in = slot_in + 1 == NST ? 0 : slot_in + 1;
    advance(head_i, qb_i, SPLIT);
  };
#pragma unroll
  for (int i = 0; i < NST - 1; ++i) issue(i);
  const int64_t kw = k0 + 32 * wave;
  const int64_t ki = kw + l31;
  const bool ok = ki < pl.len;
  u32x4_t fk[NS], fv[VLDS ? 1 : NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    fk[s] = row_frag(Kp, p.k_rs, ki, ok, s, h, D);
    if constexpr (!VLDS) fv[s] = row_frag(V, p.v_rs, ki, ok, s, h, D);
  }
  f32x16_t aK[ND], aV[ND];
#pragma unroll
  for (int t = 0; t < ND; ++t) {
    zero16(aK[t]);
    zero16(aV[t]);
  }
  const bool ranged = IS_F16<L> && c > 0x1p-100f;
  float up = ranged ? BWD_UP / c : 0.0f;                     // the scores start from `up`: the lane's factor is 2^(c up)
#pragma unroll 1
  for (int it = 0; it < steps; ++it) {
    arrive<(NST - 2) * PIECES>();
    issue(it + NST - 1);
    const unsigned char* sq = smem + slot_out * 2 * TB;
    const unsigned char* sd = sq + TB;
    const float* st = stat + slot_out * 2 * 64;
    slot_out = slot_out + 1 == NST ? 0 : slot_out + 1;
    const int64_t r0 = (int64_t)qb_o * QB;
    advance(head_o, qb_o, SPLIT);
    if (SPLIT > 1 && it * SPLIT + part >= total) continue;
    if (r0 + QB - 1 < kw || kw >= pl.len) continue;          // every query of the tile is earlier than this wave's keys
    const int lim = (int)(ki - r0);                           // first query of the tile that sees this lane's key
    const int end = (int)(pl.len - r0 < QB ? pl.len - r0 : QB);       // rows past the sequence are zeros: against a key with an inf they would give NaN
    const bool edge = r0 < kw + 31 || end < QB;
#pragma unroll
    for (int qt = 0; qt < QB / 32; ++qt) {
      if (r0 + 32 * qt + 31 < kw) continue;                  // a half of earlier queries only
      f32x16_t S, dP;
#pragma unroll
      for (int r = 0; r < 16; ++r) S[r] = up;
#pragma unroll
      for (int g = 0; g < 4; ++g) {                          // dp starts from -delta
        const f32x4_t d4 = *(const f32x4_t*)(st + 64 + 32 * qt + 8 * g + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) dP[4 * g + j] = d4[j];
      }
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        mma(S, frag_rows<DP>(sq, 32 * qt + l31, s, h), fk[s]);
        if constexpr (VLDS)
          mma(dP, frag_rows<DP>(sd, 32 * qt + l31, s, h), frag_rows<DP>(vmem, 32 * wave + l31, s, h));
        else
          mma(dP, frag_rows<DP>(sd, 32 * qt + l31, s, h), fv[s]);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4_t l4 = *(const f32x4_t*)(st + 32 * qt + 8 * g + 4 * h);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int r = 4 * g + j;
          S[r] = __builtin_amdgcn_exp2f(fmaf(S[r], c, -l4[j]));
          dP[r] *= S[r];                                      // ds / scale
        }
      }
      if (edge) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int i = 32 * qt + acc_row(r, h);
          const bool see = i >= lim && i < end;
          S[r] = see ? S[r] : 0.0f;
          dP[r] = see ? dP[r] : 0.0f;
        }
      }
      if constexpr (IS_F16<L>) {
        const int e = ranged ? lower_by(dP) : 0;
        if (__builtin_expect(__any(e != 0), 0)) {
          const float by = ldexpf(1.0f, e);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            S[r] *= by;
            dP[r] *= by;
          }
          scale_all<ND>(aK, by);
          scale_all<ND>(aV, by);
          up = (rintf(up * c) + (float)e) / c;
        }
      }
#pragma unroll
      for (int sg = 0; sg < 2; ++sg) {
        const u32x4_t fp = pack8<L>(S, 8 * sg), fs = pack8<L>(dP, 8 * sg);
#pragma unroll
        for (int t = 0; t < ND; ++t) {
          mma(aV[t], frag_cols<DP>(sd, t, 32 * qt + 16 * sg, lane), fp);
          mma(aK[t], frag_cols<DP>(sq, t, 32 * qt + 16 * sg, lane), fs);
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if constexpr (IS_F16<L>) {
    const float undo = ldexpf(1.0f, -(int)rintf(up * c));
    scale_all<ND>(aK, undo);
    scale_all<ND>(aV, undo);
  }
  if constexpr (SPLIT > 1) {
    join_parts<ND, NW, SPLIT>(aK, (float*)smem_all, wave, part, lane);
    join_parts<ND, NW, SPLIT>(aV, (float*)smem_all, wave, part, lane);
    if (part) return;
  }
#pragma unroll
  for (int t = 0; t < ND; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) aK[t][r] *= p.scale;
  store_rows<L, DP>(dK + kw * p.dk_rs, p.dk_rs, D, aK, l31, ok, h);
  store_rows<L, DP>(dV + kw * p.dv_rs, p.dv_rs, D, aV, l31, ok, h);
  if (!__any(ok && (nonfinite<ND>(aK) || nonfinite<ND>(aV)))) return;
  // queries before the wave's last key that its first tile holds, in any head of the group
  bool bad = false;
  const int64_t f0 = kw / QB * QB, f1 = kw + 31 < pl.len ? kw + 31 : pl.len;
  for (int gh = 0; gh < group && !bad; ++gh) {
    const int head = kvh * group + gh;
    bad = any_nonfinite<L>((const uint16_t*)p.q + pl.row0 * p.q_rs + head * p.q_hs, p.q_rs, D, f0, f1, lane) ||
          any_nonfinite<L>((const uint16_t*)p.dout + pl.row0 * p.do_rs + head * p.do_hs, p.do_rs, D, f0, f1, lane);
  }
  if (!bad) return;
  for (int64_t j = kw; j < kw + 32 && j < pl.len; ++j) {                               // dk, dv of these keys from the queries that see them alone
    float ok_[2] = {0.0f, 0.0f}, ov_[2] = {0.0f, 0.0f};
    for (int gh = 0; gh < group; ++gh) {
      const int head = kvh * group + gh;
      const uint16_t* Q = (const uint16_t*)p.q + pl.row0 * p.q_rs + head * p.q_hs;
      const uint16_t* dO = (const uint16_t*)p.dout + pl.row0 * p.do_rs + head * p.do_hs;
      const int64_t at = (int64_t)head * p.rows + pl.row0;
      for (int64_t i0 = j; i0 < pl.len; i0 += 64) {
        const int n = (int)(pl.len - i0 < 64 ? pl.len - i0 : 64);
        float wv = 0.0f, wk = 0.0f;
        if (lane < n) {
          const int64_t i = i0 + lane;
          wv = __builtin_amdgcn_exp2f(fmaf(dot_rows<L>(Q + i * p.q_rs, Kp + j * p.k_rs, D), c, -p.lse[at + i]));
          wk = wv * (dot_rows<L>(dO + i * p.do_rs, V + j * p.v_rs, D) + p.delta[at + i]);       // (delta is stored negative)
        }
        add_weighted<L>(ov_, wv, dO + i0 * p.do_rs, p.do_rs, D, n, lane);
        add_weighted<L>(ok_, wk, Q + i0 * p.q_rs, p.q_rs, D, n, lane);
        if (all_nan(ov_, D, lane) && all_nan(ok_, D, lane)) break;
      }
    }
    put_row<L>(dK + j * p.dk_rs, ok_, p.scale, D, lane);
    put_row<L>(dV + j * p.dv_rs, ov_, 1.0f, D, lane);
  }
}

int check_common(const ffvc_attn_packed_desc& d, const char* who) {
  FFVC_CHECK_ARG(d.dtype == FFVC_BF16 || d.dtype == FFVC_F16, "%s: 16-bit storage only (bf16, f16)", who);
  FFVC_CHECK_ARG(d.rows > 0 && d.seqs > 0 && d.cu, "%s: needs rows > 0, seqs > 0 and the sequence offsets", who);
  FFVC_CHECK_ARG(d.rows < (1ll << 31), "%s: the row offsets are 32-bit integers: rows < 2^31", who);
  FFVC_CHECK_ARG(d.heads > 0 && d.kv_heads > 0 && d.heads % d.kv_heads == 0, "%s: heads (%d) must be a multiple of kv_heads (%d)", who, d.heads, d.kv_heads);
  FFVC_CHECK_ARG(d.head_dim >= 8 && d.head_dim <= 128 && d.head_dim % 8 == 0, "%s: head_dim %d unsupported (a multiple of 8, at most 128)", who, d.head_dim);
  FFVC_CHECK_ARG(d.scale > 0.0f && d.scale < INFINITY, "%s: scale must be positive and finite", who);
  return 0;
}
int check_tensor(const void* ptr, int64_t rs, int64_t hs, int D, const char* who, const char* what) {
  FFVC_CHECK_ARG(ptr && (uintptr_t)ptr % 16 == 0, "%s: %s must be non-null and 16-byte aligned", who, what);
  FFVC_CHECK_ARG(rs % 8 == 0 && hs % 8 == 0 && rs >= D && hs >= 0, "%s: %s strides must be multiples of 8 elements, rows at least head_dim apart (row %lld, head %lld)", who, what, (long long)rs, (long long)hs);
  FFVC_CHECK_ARG(rs < (1ll << 23), "%s: %s row stride too long", who, what);       // a tile of 64 rows stays below 2 GiB
  return 0;
}
// a tensor that is written: no element belongs to two (row, head) pairs
int check_written(const void* ptr, int64_t rs, int64_t hs, const ffvc_attn_packed_desc& d, int heads, const char* who, const char* what) {
  const int rc = check_tensor(ptr, rs, hs, d.head_dim, who, what);
  if (rc) return rc;
  FFVC_CHECK_ARG(rs >= (heads - 1) * hs + d.head_dim || hs >= (d.rows - 1) * rs + d.head_dim, "%s: rows and heads of %s overlap (strides %lld, %lld)", who,
                 what, (long long)rs, (long long)hs);
  return 0;
}

// one launch of KERNEL (a template-id in parentheses) over slots x HEADS workgroups
#define LAUNCH_PACKED(KERNEL, LDS, HEADS, THREADS)                                                                                              \
  do {                                                                                                                                          \
    static ffvc_lds_once once__;                                                                                                                \
    const int64_t blocks__ = slots * (HEADS);                                                                                                   \
    FFVC_CHECK_ARG(ffvc_launch_fits(blocks__, THREADS), "ffvc_attn_packed: too many tiles for one launch (%lld)", (long long)blocks__);         \
    const int rc__ = once__.set((const void*)KERNEL, LDS);                                                                                      \
    if (rc__) return rc__;                                                                                                                      \
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)blocks__), dim3(THREADS), LDS, st, d, slots);                                                     \
    FFVC_LAUNCH_CHECK();                                                                                                                        \
  } while (0)

// Short sequences on average: one wave per workgroup, so that a prompt does not pay for rows it has not.  Forward, four waves / one, us, 256 sequences with
// 8 heads, of 20 / 48 / 64 / 100 / 128 rows: 20 / 9.7, 28 / 17, 26 / 20, 37 / 32, 62 / 36 with 64 features; 26 / 18, 32 / 31, 35 / 35, 53 / 66, 89 / 68 with 128 (and
// 128 of 200 rows 38 / 36, 56 / 69).  Backward, dq + dk / dv, 256 sequences of 20 / 48 / 64 / 100: 43 / 24, 54 / 43, 60 / 50, 95 / 83; 61 / 44, 90 / 86, 103 / 98, 186 / 209.
// The mean says nothing about the longest sequence, and the lengths are not known here.  A long one among short or empty ones goes through one-wave
// tiles whose walks nobody splits; four waves / one, forward and backward, 8 heads: one of 2048 rows and 63 of 10 39 / 39 and 66 / 104 (128 features 53 / 56,
// 155 / 165); one of 4096 and 127 of 10 73 / 75, 183 / 200 (103 / 120, 327 / 338; with 16 / 4 heads of 64 85 / 90, 226 / 539); one of 8000 in 256 slots 130 / 164,
// 348 / 398 (192 / 241, 634 / 841).  The rule stands for what it serves, prompts of like lengths, which the four-wave form takes twice as long for.
inline bool short_rows(const ffvc_attn_packed_desc& d, int rows) { return d.rows <= rows * (int64_t)d.seqs; }

template <typename L, int DP>
int run_fwd(const ffvc_attn_packed_desc& d, hipStream_t st) {
  if (short_rows(d, DP == 64 ? 128 : 64)) {
    const int64_t slots = d.rows / 32 + d.seqs + 2;
    LAUNCH_PACKED((attn_packed_fwd_kernel<L, DP, 1, 1, 64>), 2 * 64 * DP * 2, d.heads, 64);
  } else {
    constexpr int NW = 4, NST = 2, KB = 64;
    const int64_t slots = d.rows / (32 * NW) + d.seqs + 2;
    LAUNCH_PACKED((attn_packed_fwd_kernel<L, DP, NW, NST, KB>), NST * 2 * KB * DP * 2, d.heads, 64 * NW);
  }
  return 0;
}

// bytes of LDS of the dk / dv kernel
constexpr int dkv_lds(int DP, int NW, int NST, int QB, bool VLDS, int SPLIT) {
  return SPLIT * NST * (2 * QB * DP * 2 + 2 * 64 * 4) + (VLDS ? 32 * NW * DP * 2 : 0);
}
template <typename L, int DP>
int run_bwd(const ffvc_attn_packed_desc& d, hipStream_t st) {
  constexpr bool VLDS = DP == 128;
  if (short_rows(d, 64)) {
    const int64_t slots = d.rows / 32 + d.seqs + 2;
    LAUNCH_PACKED((attn_packed_dq_kernel<L, DP, 1, 2, 32, 1>), 2 * 2 * 32 * DP * 2, d.heads, 64);
    LAUNCH_PACKED((attn_packed_dkv_kernel<L, DP, 1, 2, 32, VLDS, 1>), dkv_lds(DP, 1, 2, 32, VLDS, 1), d.kv_heads, 64);
  } else {
    constexpr int NW = 4, NST = 2, KB = 64, QB = DP == 64 ? 64 : 32;
    const int64_t slots = d.rows / (32 * NW) + d.seqs + 2;
    // (Tiles are counted as rows / 128 + seqs + 1 per head.)  Few query tiles for the chip's places: each split over two halves of its keys, tiles of 64
    // queries.  Measured (1 / 2 parts), us: 560 tiles, 8 ragged sequences with 16 heads 28 / 22, 128 features 42 / 37; 288 tiles, one of 2048 rows 39 / 30,
    // 62 / 43; but 1056 tiles, one of 8192 198 / 217, 380 / 394; 2064 tiles, 24 ragged ones 72 / 90, 128 / 157 (the halves fetch every key and value
    // twice as often).
    if ((slots - 1) * d.heads < 768) {
      const int64_t slots = d.rows / 64 + d.seqs + 2;
      LAUNCH_PACKED((attn_packed_dq_kernel<L, DP, 2, 2, 32, 2>), 2 * 2 * 2 * 32 * DP * 2, d.heads, 256);
    } else {
      LAUNCH_PACKED((attn_packed_dq_kernel<L, DP, 4, NST, KB, 1>), NST * 2 * KB * DP * 2, d.heads, 256);
    }
    // A key tile's walk is as long as its sequence times the group: while the tiles are few for the chip's 512 places the longest walk alone decides,
    // so it is split over the workgroup's waves.  Measured (1 / 2 / 4 parts; the last with tiles of 64 keys), us:
    //   520 tiles, 24 ragged sequences of up to 2100 rows, 64 features: 208 / 143 / 108; 128 features: 397 / 248 / 236; one sequence, 264 tiles: 1520 / 935 / 614
    //   884 tiles, 40 ragged sequences: 247 / 213 / 229; 128 features: 424 / 316 / 434; 12 sequences of 2048 rows, 820 tiles: 233 / 252 / 276
    //   1056 tiles, one sequence of 8192 rows: 298 / 311 / 347; 128 features: 540 / 562 / 757
    if ((slots - 1) * d.kv_heads < 768) {
      const int64_t slots = d.rows / 64 + d.seqs + 2;
      LAUNCH_PACKED((attn_packed_dkv_kernel<L, DP, 2, NST, QB, VLDS, 4>), dkv_lds(DP, 2, NST, QB, VLDS, 4), d.kv_heads, 512);
    } else if ((slots - 1) * d.kv_heads < 1024) {
      LAUNCH_PACKED((attn_packed_dkv_kernel<L, DP, 4, NST, QB, VLDS, 2>), dkv_lds(DP, 4, NST, QB, VLDS, 2), d.kv_heads, 512);
    } else {
      LAUNCH_PACKED((attn_packed_dkv_kernel<L, DP, 4, NST, QB, VLDS, 1>), dkv_lds(DP, 4, NST, QB, VLDS, 1), d.kv_heads, 256);
    }
  }
  return 0;
}

}  // namespace

extern "C" int ffvc_attn_packed_fwd(const ffvc_attn_packed_desc* dp, void* stream) {
  FFVC_CHECK_ARG(dp, "ffvc_attn_packed_fwd: null descriptor");
  const ffvc_attn_packed_desc& d = *dp;
  const char* who = "ffvc_attn_packed_fwd";
  int rc = check_common(d, who);
  if (!rc) rc = check_tensor(d.q, d.q_rs, d.q_hs, d.head_dim, who, "q");
  if (!rc) rc = check_tensor(d.k, d.k_rs, d.k_hs, d.head_dim, who, "k");
  if (!rc) rc = check_tensor(d.v, d.v_rs, d.v_hs, d.head_dim, who, "v");
  if (!rc) rc = check_written(d.out, d.o_rs, d.o_hs, d, d.heads, who, "out");
  if (rc) return rc;
  hipStream_t st = (hipStream_t)stream;
  if (d.head_dim <= 64) return d.dtype == FFVC_F16 ? run_fwd<f16_t, 64>(d, st) : run_fwd<uint16_t, 64>(d, st);
  return d.dtype == FFVC_F16 ? run_fwd<f16_t, 128>(d, st) : run_fwd<uint16_t, 128>(d, st);
}

extern "C" int ffvc_attn_packed_bwd(const ffvc_attn_packed_desc* dp, void* stream) {
  FFVC_CHECK_ARG(dp, "ffvc_attn_packed_bwd: null descriptor");
  const ffvc_attn_packed_desc& d = *dp;
  const char* who = "ffvc_attn_packed_bwd";
  int rc = check_common(d, who);
  if (!rc) rc = check_tensor(d.q, d.q_rs, d.q_hs, d.head_dim, who, "q");
  if (!rc) rc = check_tensor(d.k, d.k_rs, d.k_hs, d.head_dim, who, "k");
  if (!rc) rc = check_tensor(d.v, d.v_rs, d.v_hs, d.head_dim, who, "v");
  if (!rc) rc = check_tensor(d.out, d.o_rs, d.o_hs, d.head_dim, who, "out");
  if (!rc) rc = check_tensor(d.dout, d.do_rs, d.do_hs, d.head_dim, who, "dout");
  if (!rc) rc = check_written(d.dq, d.dq_rs, d.dq_hs, d, d.heads, who, "dq");
  if (!rc) rc = check_written(d.dk, d.dk_rs, d.dk_hs, d, d.kv_heads, who, "dk");
  if (!rc) rc = check_written(d.dv, d.dv_rs, d.dv_hs, d, d.kv_heads, who, "dv");
  if (rc) return rc;
  FFVC_CHECK_ARG(d.lse && d.delta, "ffvc_attn_packed_bwd: needs the forward's lse and the delta workspace");
  hipStream_t st = (hipStream_t)stream;
  if (d.head_dim <= 64) return d.dtype == FFVC_F16 ? run_bwd<f16_t, 64>(d, st) : run_bwd<uint16_t, 64>(d, st);
  return d.dtype == FFVC_F16 ? run_bwd<f16_t, 128>(d, st) : run_bwd<uint16_t, 128>(d, st);
}
