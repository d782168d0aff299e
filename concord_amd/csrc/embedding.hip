// embedding.hip -- rows of a table by token, scaled, and the table's gradient by
// sorted tokens.
//
//   y[i] = s W[t_i];   dW[v] = s sum over { i : t_i = v } of dy[i]
//
// Both passes are bound by memory: the forward reads the rows it names and
// writes the result, the backward reads dy and writes the whole table's gradient,
// zeros included.
//
// The backward sorts (token, position) pairs by token, stably, with a radix sort
// of up to 9 bits a pass; a token's rows then stand one after another, in the
// order of their positions.  The sorted pairs are cut into pieces of equal
// length, whatever the tokens' counts, and each wave adds the rows of a piece for
// one slab of columns in registers.  A token inside one piece is stored at once;
// one that crosses pieces leaves its sums in the workspace, and a second kernel
// adds those in order.  No sum depends on the order in which waves run: there are
// no atomics on floating point numbers.
//
// Kernel times, 32768 tokens of 50257, 4096 wide, bf16: forward 75 us (268 MB written and
// as much read, a third of it from memory), sort 21 us in four launches, sums and zeros
// 136 us (680 MB, 5.0 TB/s), join 12 us.  16384 tokens of 65, 384 wide, fp32: 7.8, 7.8, 7.9
// and 5.1 us, near the cost of the launches and their latencies.
#include "elem.h"

namespace concord {

constexpr int kMaxBits = 9, kMaxBins = 1 << kMaxBits;
// pairs a block of the sort takes: few where the tokens are, since a wave ranks its pairs
// one after another
static int emb_tile(int64_t n) { return n <= 65536 ? 1024 : 4096; }
constexpr int kOneBlock = 4096;      // pairs that one block sorts alone
// Up to this many blocks each sums the counts of all of them for itself; past it, where that
// work would grow with the square of the tokens, a kernel of its own sums them up once a pass
// (whole backward of tokens of 511, 8 wide, bf16: 2^19 tokens 79 to 90 us without it, 89 to
// 92 with; 2^20 128 to 138 and 133 to 137; 2^21 224 to 233 and 211; 2^24 3045 and 1450).
constexpr unsigned kScanBlocks = 256;

struct EmbArgs {
  const void* tokens;
  int idx64;
  int64_t n;            // < 2^31
  uint32_t V;
  int64_t C;
  float scale;
  const void* src;      // the table, or dy
  int64_t lds;
  void* dst;            // y, or dW
  int64_t ldd;
  const uint32_t* keys; // sorted tokens, V for those outside the table
  const uint32_t* pos;  // their positions
  float* part;          // [pieces][2][C]: sums of a run's head (it began earlier), of its first rows
  int piece;            // pairs a wave adds
  int64_t pieces;
  int64_t slabs;        // of 64 lanes' columns
  int64_t fill_at;      // first block of those that write zeros
};

CONCORD_DEV uint32_t token_key(const void* tokens, int idx64, int64_t i, uint32_t V) {
  const int64_t t = idx64 ? ((const int64_t*)tokens)[i] : (int64_t)((const int32_t*)tokens)[i];
  return (uint64_t)t < V ? (uint32_t)t : V;
}

// VEC columns of a row as they lie in memory: on their size, or (AL false) where an element
// may begin, which this GPU takes for wide accesses too.  Rows whose length VEC does not
// divide end in a step that is moved back to end with them: it gives the columns that it
// shares with the one before the same values again.
template <class T, int VEC, bool AL>
struct alignas(AL ? sizeof(T) * VEC : sizeof(T)) Cols {
  T v[VEC];
};
template <int VEC>
CONCORD_DEV int64_t last_step(int64_t c, int64_t C) { return min(c, C - VEC); }
template <bool AL, class V>
CONCORD_DEV void store_cols(void* p, const V& v) {
  if constexpr (AL) store_stream((V*)p, v);
  else *(V*)p = v;
}

// ---- forward ------------------------------------------------------------------
// 2^lg threads a row, VEC columns a thread and step.  (Four rows at once, their loads
// out together: no change.  The stores go past the caches: 16384 x 384 in fp32 9.1 -> 7.4
// us, 32768 x 4096 in bf16 72 -> 75.)
template <class TW, class TO, int VEC, bool AL>
__global__ __launch_bounds__(256) void emb_fwd_kernel(EmbArgs a, int lg) {
  const int64_t step = (int64_t)gridDim.x << (8 - lg);
  for (int64_t row = ((int64_t)blockIdx.x << (8 - lg)) + (threadIdx.x >> lg); row < a.n; row += step) {
    const uint32_t t = token_key(a.tokens, a.idx64, row, a.V);
    const bool there = t < a.V;
    const TW* src = (const TW*)a.src + (int64_t)(there ? t : 0) * a.lds;
    TO* dst = (TO*)a.dst + row * a.ldd;
    for (int64_t c = (int64_t)(threadIdx.x & ((1 << lg) - 1)) * VEC; c < a.C; c += (int64_t)VEC << lg) {
      const int64_t at = last_step<VEC>(c, a.C);
      Cols<TW, VEC, AL> v = {};
      if (there) v = *(const Cols<TW, VEC, AL>*)(src + at);
      Cols<TO, VEC, AL> r;
#pragma unroll
      for (int e = 0; e < VEC; ++e) r.v[e] = from_f32<TO>(to_f32(v.v[e]) * a.scale);
      store_cols<AL>(dst + at, r);
    }
  }
}

// ---- sort -----------------------------------------------------------------------
// lanes of the wave whose digit of `bits` bits is this lane's
CONCORD_DEV uint64_t same_digit(uint32_t d, int bits) {
  uint64_t m = ~0ull;
  for (int b = 0; b < bits; ++b) {
    const bool bit = (d >> b) & 1;
    const uint64_t set = __builtin_amdgcn_ballot_w64(bit);
    m &= bit ? set : ~set;
  }
  return m;
}
// how many of the wave's earlier pairs have the digit d: counts, one for each digit, goes on from step to step
CONCORD_DEV uint32_t digit_rank(uint32_t* counts, uint32_t d, int bits) {
  const uint64_t m = same_digit(d, bits);
  const uint32_t before = __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
  const uint32_t prior = counts[d];
  __builtin_amdgcn_wave_barrier();
  if (before == 0) counts[d] = prior + (uint32_t)__builtin_popcountll(m);
  __builtin_amdgcn_wave_barrier();
  return prior + before;
}

// exclusive sums over the block's first `bins` threads' values (W waves; all threads call)
template <int W>
CONCORD_DEV uint32_t block_exclusive(uint32_t v, uint32_t (&sums)[W]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t s = v;
#pragma unroll
  for (int h = 1; h < 64; h <<= 1) {
    const uint32_t o = __shfl_up(s, h, 64);
    if (lane >= h) s += o;
  }
  if (lane == 63) sums[wave] = s;
  __syncthreads();
  uint32_t base = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) base += w < wave ? sums[w] : 0;
  return base + s - v;
}

// All of up to IT * 1024 pairs in one block: pair e belongs to wave e / (64 IT).
template <int IT>
__global__ __launch_bounds__(1024) void emb_sort_block_kernel(EmbArgs a, int passes, int bits, uint32_t* keys,
                                                             uint32_t* pos) {
  __shared__ uint32_t lk[IT * 1024], lp[IT * 1024], cnt[16][kMaxBins], sums[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << bits;
  const int e0 = wave * IT * 64 + lane, n = (int)a.n;
  uint32_t k[IT], p[IT], rank[IT];
#pragma unroll
  for (int j = 0; j < IT; ++j) {
    const int e = e0 + j * 64;
    // (behind the last pair: the largest digits, so they stay behind it)
    k[j] = e < n ? token_key(a.tokens, a.idx64, e, a.V) : 0xFFFFFFFFu;
    p[j] = (uint32_t)e;
  }
  for (int pass = 0; pass < passes; ++pass) {
    for (int i = lane; i < bins; i += 64) cnt[wave][i] = 0;
    __builtin_amdgcn_wave_barrier();
    const int shift = pass * bits;
#pragma unroll
    for (int j = 0; j < IT; ++j) rank[j] = digit_rank(cnt[wave], (k[j] >> shift) & (bins - 1), bits);
    __syncthreads();
    uint32_t total = 0;
    if ((int)threadIdx.x < bins) {
#pragma unroll
      for (int w = 0; w < 16; ++w) total += cnt[w][threadIdx.x];
    }
    uint32_t at = block_exclusive<16>(total, sums);
    if ((int)threadIdx.x < bins) {
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        const uint32_t c = cnt[w][threadIdx.x];
        cnt[w][threadIdx.x] = at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < IT; ++j) {
      const uint32_t dst = cnt[wave][(k[j] >> shift) & (bins - 1)] + rank[j];
      lk[dst] = k[j];
      lp[dst] = p[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < IT; ++j) {
      k[j] = lk[e0 + j * 64];
      p[j] = lp[e0 + j * 64];
    }
  }
#pragma unroll
  for (int j = 0; j < IT; ++j)
    if (e0 + j * 64 < n) {
      keys[e0 + j * 64] = k[j];
      pos[e0 + j * 64] = p[j];
    }
}

// One pass over many blocks of 512 IT pairs each: the digits' counts of each block ...
struct SortPass {
  const uint32_t *keys, *pos;   // NULL in the first pass: the tokens
  uint32_t *out_keys, *out_pos;
  uint32_t* counts;             // [blocks][bins]
  uint32_t* totals;             // [bins] where the counts are summed up before, else NULL
  int shift, bits;
};
template <int IT>
__global__ __launch_bounds__(512) void emb_count_kernel(EmbArgs a, SortPass s) {
  __shared__ uint32_t cnt[kMaxBins];
  const int bins = 1 << s.bits;
  if ((int)threadIdx.x < bins) cnt[threadIdx.x] = 0;
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * (IT * 512);
#pragma unroll
  for (int j = 0; j < IT; ++j) {
    const int64_t i = first + j * 512 + threadIdx.x;
    if (i < a.n) {
      const uint32_t k = s.keys ? s.keys[i] : token_key(a.tokens, a.idx64, i, a.V);
      atomicAdd(&cnt[(k >> s.shift) & (bins - 1)], 1u);
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < bins) s.counts[(int64_t)blockIdx.x * bins + threadIdx.x] = cnt[threadIdx.x];
}
// ... the counts' exclusive sums over the blocks, in place, and their totals: a wave a
// sixteenth of the blocks, its sum first, then the running sums behind those of the waves before it ...
__global__ __launch_bounds__(1024) void emb_scan_kernel(SortPass s, uint32_t blocks) {
  constexpr int B = 16;
  __shared__ uint32_t sums[16][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << s.bits;
  const int bin = blockIdx.x * 64 + lane;
  const uint32_t per = (blocks + 15) / 16, first = min(wave * per, blocks), last = min(first + per, blocks);
  uint32_t* c = s.counts + min(bin, bins - 1);
  uint32_t v[B], sum = 0;
  auto load = [&](uint32_t b) {
#pragma unroll
    for (int i = 0; i < B; ++i) v[i] = b + i < last ? c[(int64_t)(b + i) * bins] : 0;
  };
  for (uint32_t b = first; b < last; b += B) {
    load(b);
#pragma unroll
    for (int i = 0; i < B; ++i) sum += v[i];
  }
  sums[wave][lane] = sum;
  __syncthreads();
  uint32_t at = 0;
  for (int w = 0; w < wave; ++w) at += sums[w][lane];
  if (bin >= bins) return;
  if (wave == 15) s.totals[bin] = at + sum;
  for (uint32_t b = first; b < last; b += B) {
    load(b);
#pragma unroll
    for (int i = 0; i < B; ++i) {
      if (b + i < last) c[(int64_t)(b + i) * bins] = at;
      at += v[i];
    }
  }
}
// ... and the pairs to their places: behind all smaller digits, behind the same digit of earlier blocks
template <int IT>
__global__ __launch_bounds__(512) void emb_scatter_kernel(EmbArgs a, SortPass s) {
  __shared__ uint32_t cnt[8][kMaxBins], sums[8];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << s.bits;
  const int64_t e0 = (int64_t)blockIdx.x * (IT * 512) + wave * IT * 64 + lane;
  uint32_t k[IT], p[IT], rank[IT];
#pragma unroll
  for (int j = 0; j < IT; ++j) {
    const int64_t i = e0 + j * 64;
    const bool in = i < a.n;
    k[j] = !in ? 0xFFFFFFFFu : s.keys ? s.keys[i] : token_key(a.tokens, a.idx64, i, a.V);
    p[j] = in && s.pos ? s.pos[i] : (uint32_t)i;
  }
  uint32_t before = 0, all = 0;
  if (s.totals) {
    if ((int)threadIdx.x < bins) {
      before = s.counts[(int64_t)blockIdx.x * bins + threadIdx.x];
      all = s.totals[threadIdx.x];
    }
  } else if ((int)threadIdx.x < bins) {
    // sixteen blocks' counts in flight: another XCD wrote them, so each load is a long one
    constexpr int B = 16;
    const uint32_t* c = s.counts + threadIdx.x;
    for (uint32_t b = 0; b < gridDim.x; b += B) {
      uint32_t v[B];
#pragma unroll
      for (int i = 0; i < B; ++i) v[i] = c[(int64_t)min(b + i, gridDim.x - 1) * bins];
#pragma unroll
      for (int i = 0; i < B; ++i) {
        before += b + i < blockIdx.x ? v[i] : 0;
        all += b + i < gridDim.x ? v[i] : 0;
      }
    }
  }
  for (int i = lane; i < bins; i += 64) cnt[wave][i] = 0;
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < IT; ++j) rank[j] = digit_rank(cnt[wave], (k[j] >> s.shift) & (bins - 1), s.bits);
  uint32_t at = block_exclusive<8>(all, sums) + before;   // (its barrier stands between the counts and their use)
  if ((int)threadIdx.x < bins) {
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const uint32_t c = cnt[w][threadIdx.x];
      cnt[w][threadIdx.x] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < IT; ++j) {
    // (what stands for no pair is counted last of the last block: nothing comes after it)
    if (e0 + j * 64 >= a.n) continue;
    const uint32_t dst = cnt[wave][(k[j] >> s.shift) & (bins - 1)] + rank[j];
    s.out_keys[dst] = k[j];
    s.out_pos[dst] = p[j];
  }
}

// ---- sums -------------------------------------------------------------------------
// one row of the gradient, or zeros
template <class TW, int VEC, bool AL>
CONCORD_DEV void store_row(const EmbArgs& a, uint32_t v, int64_t c, const float (&s)[VEC]) {
  if (c >= a.C) return;
  Cols<TW, VEC, AL> r;
#pragma unroll
  for (int e = 0; e < VEC; ++e) r.v[e] = from_f32<TW>(s[e] * a.scale);
  store_cols<AL>((TW*)a.dst + (int64_t)v * a.ldd + last_step<VEC>(c, a.C), r);
}
template <int VEC>
CONCORD_DEV void store_part(const EmbArgs& a, int64_t piece, int which, int64_t c, const float (&s)[VEC]) {
  if (c >= a.C) return;
  float* p = a.part + (piece * 2 + which) * a.C + last_step<VEC>(c, a.C);
#pragma unroll
  for (int e = 0; e < VEC; ++e) p[e] = s[e];
}

// First of keys[lo, hi) that is not less than v, found by a wave: 64 places at once, so
// three rounds of loads find one among a quarter of a million.
CONCORD_DEV int64_t first_not_less(const uint32_t* keys, int64_t lo, int64_t hi, uint32_t v) {
  const int lane = threadIdx.x & 63;
  while (hi > lo) {
    const int64_t step = (hi - lo + 63) >> 6, at = lo + lane * step;
    const int less = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at < hi && keys[at] < v));
    // keys at the first `less` places are less than v, the next is not
    hi = min(hi, lo + less * step);
    lo = less ? lo + (less - 1) * step + 1 : hi;
  }
  return lo;
}

constexpr int kFillRows = 8;   // rows of the table that a wave looks at for zeros

template <class TG, class TW, int VEC, bool AL>
__global__ __launch_bounds__(256) void emb_sum_kernel(EmbArgs a) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int64_t)blockIdx.x >= a.fill_at) {
    // rows of the table without a token
    const int64_t v0 = (((int64_t)blockIdx.x - a.fill_at) * 4 + wave) * kFillRows;
    if (v0 >= a.V) return;
    const int64_t lo = first_not_less(a.keys, 0, a.n, (uint32_t)v0);
    const int64_t hi = first_not_less(a.keys, lo, a.n, (uint32_t)min(v0 + kFillRows, (int64_t)a.V));
    const float zero[VEC] = {};
    for (int64_t v = v0; v < min(v0 + kFillRows, (int64_t)a.V); ++v) {
      const int64_t at = hi > lo ? first_not_less(a.keys, lo, hi, (uint32_t)v) : hi;
      if (at < hi && a.keys[at] == (uint32_t)v) continue;
      for (int64_t c = (int64_t)lane * VEC; c < a.C; c += 64 * VEC) store_row<TW, VEC, AL>(a, (uint32_t)v, c, zero);
    }
    return;
  }
  const int64_t item = (int64_t)blockIdx.x * 4 + wave, piece = item / a.slabs;
  if (piece >= a.pieces) return;
  // the piece's pairs, one a lane; their rows are loaded U at a time, the next U while
  // these are added, and no load is behind a branch (a lane past the last column loads the
  // first, a step past the last pair its row again)
  const int64_t p0 = piece * a.piece, p1 = min(p0 + a.piece, a.n), at = min(p0 + lane, p1 - 1);
  const uint32_t key = a.keys[at], pos = a.pos[at];
  const uint32_t earlier = p0 > 0 ? a.keys[p0 - 1] : ~0u, later = p1 < a.n ? a.keys[p1] : ~0u;
  const int m = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < p1 - p0 && key < a.V));
  if (m == 0) return;   // (tokens outside the table stand last)
  const int64_t c = ((item - piece * a.slabs) * 64 + lane) * VEC;
  const TG* src = (const TG*)a.src + (c < a.C ? last_step<VEC>(c, a.C) : 0);
  constexpr int U = 8;
  Cols<TG, VEC, AL> r[2][U];
  auto load = [&](Cols<TG, VEC, AL> (&t)[U], int i) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      t[u] = *(const Cols<TG, VEC, AL>*)(src + (int64_t)(uint32_t)__builtin_amdgcn_readlane(pos, min(i + u, m - 1)) * a.lds);
  };
  uint32_t cur = __builtin_amdgcn_readlane(key, 0);
  bool head = earlier == cur;
  float s[VEC] = {};
  auto add = [&](const Cols<TG, VEC, AL> (&t)[U], int i) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i + u >= m) break;
      const uint32_t k = __builtin_amdgcn_readlane(key, i + u);
      if (k != cur) {
        if (head) store_part<VEC>(a, piece, 0, c, s);
        else store_row<TW, VEC, AL>(a, cur, c, s);
        head = false;
        cur = k;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] = 0.0f;
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] += to_f32(t[u].v[e]);
    }
  };
  load(r[0], 0);
  for (int i = 0; i < m; i += 2 * U) {
    load(r[1], i + U);
    add(r[0], i);
    if (i + U >= m) break;
    load(r[0], i + 2 * U);
    add(r[1], i + U);
  }
  if (head) store_part<VEC>(a, piece, 0, c, s);
  else if (later == cur) store_part<VEC>(a, piece, 1, c, s);
  else store_row<TW, VEC, AL>(a, cur, c, s);
}

// Tokens that cross pieces: the block of the piece that such a run begins in
// adds its sums, each wave every eighth of them, then the waves' sums in order.
template <class TW, int VEC, bool AL>
__global__ __launch_bounds__(512) void emb_join_kernel(EmbArgs a) {
  constexpr int W = 8, U = 4;
  __shared__ float part[W][64 * VEC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t piece = blockIdx.x / a.slabs, p0 = piece * a.piece, p1 = p0 + a.piece;
  if (p1 >= a.n) return;
  const uint32_t cur = a.keys[p1 - 1];
  if (cur >= a.V || a.keys[p1] != cur) return;
  if (p0 > 0 && a.keys[p0 - 1] == cur) return;   // it began earlier
  const int64_t last = (first_not_less(a.keys, p1, a.n, cur + 1) - 1) / a.piece;
  const int64_t c = ((blockIdx.x - piece * a.slabs) * 64 + lane) * VEC;
  float s[VEC] = {};
  if (c < a.C) {
    const float* h = a.part + last_step<VEC>(c, a.C);
    const int64_t row = 2 * a.C;
    int64_t q = piece + 1 + wave;
    for (; q + (U - 1) * W <= last; q += U * W) {
      float v[U][VEC];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[u][e] = h[(q + u * W) * row + e];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[e] += v[u][e];
    }
    for (; q <= last; q += W)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] += h[q * row + e];
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) part[wave][lane * VEC + e] = s[e];
  __syncthreads();
  if (wave == 0 && c < a.C) {
    const float* t = a.part + (piece * 2 + 1) * a.C + last_step<VEC>(c, a.C);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      s[e] = t[e];
#pragma unroll
      for (int w = 0; w < W; ++w) s[e] += part[w][lane * VEC + e];
    }
    store_row<TW, VEC, AL>(a, cur, c, s);
  }
}

// ---- host -------------------------------------------------------------------
static bool emb_dtype_ok(int t) { return t == CONCORD_F32 || t == CONCORD_BF16 || t == CONCORD_F16; }
static size_t emb_size(int t) { return t == CONCORD_F32 ? 4 : 2; }

// Pairs a wave adds.  A lane's worth each: fewer cost the join more than they save here
// (16384 tokens of 65, 384 wide: 8.5 + 4.6 us by 64, 10.6 + 5.7 by 16; 32768 of 50257,
// 4096 wide: 134 + 11 and 134 + 34).  Among few tokens the chain of loads counts (4000 of
// 65, 384 wide: 6.7 + 4.3 by 16, 9.4 + 4.0 by 64).
static int emb_piece(int64_t n) { return n <= 4096 ? 16 : 64; }

struct EmbWorkspace {
  size_t keys[2], pos[2], counts, totals, part, bytes;
};
static EmbWorkspace emb_workspace(int64_t n, int64_t C) {
  EmbWorkspace w{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += (bytes + 255) & ~(size_t)255;
    return r;
  };
  for (int i = 0; i < 2; ++i) {
    w.keys[i] = take((size_t)n * 4);
    w.pos[i] = take((size_t)n * 4);
  }
  w.counts = take((size_t)cdiv(n, emb_tile(n)) * kMaxBins * 4);
  w.totals = take(kMaxBins * 4);
  w.part = take((size_t)cdiv(n, emb_piece(n)) * 2 * (size_t)C * 4);
  w.bytes = at;
  return w;
}

static bool emb_chunked(const void* p, int64_t ld, size_t bytes, size_t es) {
  return ((uintptr_t)p & (bytes - 1)) == 0 && (ld * es) % bytes == 0;
}

// columns of a lane and step: 16 bytes of the narrower type, or one of a row shorter than that
template <class TA, class TB>
struct EmbVec {
  static constexpr int V = sizeof(TA) == 2 || sizeof(TB) == 2 ? 8 : 4;
};
struct EmbColumns {
  int n;
  bool aligned;
};
static EmbColumns emb_columns(const EmbArgs& a, int src_type, int dst_type) {
  const int v = emb_size(src_type) == 2 || emb_size(dst_type) == 2 ? 8 : 4;
  if (a.C < v) return {1, true};
  return {v, a.C % v == 0 && emb_chunked(a.src, a.lds, 16, emb_size(src_type)) &&
                 emb_chunked(a.dst, a.ldd, 16, emb_size(dst_type))};
}

template <class TW, class TO>
static void emb_fwd(const EmbArgs& a, EmbColumns columns, hipStream_t st) {
  constexpr int V = EmbVec<TW, TO>::V;
  const int64_t steps = cdiv(a.C, columns.n);
  int lg = 0;
  while (lg < 8 && (1 << lg) < steps) ++lg;
  const dim3 grid((unsigned)std::min<int64_t>(cdiv(a.n, 256 >> lg), 1 << 20));
  if (columns.n == 1) hipLaunchKernelGGL((emb_fwd_kernel<TW, TO, 1, true>), grid, dim3(256), 0, st, a, lg);
  else if (columns.aligned) hipLaunchKernelGGL((emb_fwd_kernel<TW, TO, V, true>), grid, dim3(256), 0, st, a, lg);
  else hipLaunchKernelGGL((emb_fwd_kernel<TW, TO, V, false>), grid, dim3(256), 0, st, a, lg);
}

template <class TG, class TW, int V, bool AL>
static void emb_sums(EmbArgs& a, hipStream_t st) {
  a.fill_at = cdiv(a.pieces * a.slabs, 4);
  hipLaunchKernelGGL((emb_sum_kernel<TG, TW, V, AL>), dim3((unsigned)(a.fill_at + cdiv(a.V, 4 * kFillRows))), dim3(256), 0, st,
                     a);
  if (a.pieces > 1)
    hipLaunchKernelGGL((emb_join_kernel<TW, V, AL>), dim3((unsigned)(a.pieces * a.slabs)), dim3(512), 0, st, a);
}
template <class TG, class TW>
static void emb_bwd(EmbArgs& a, EmbColumns columns, hipStream_t st) {
  constexpr int V = EmbVec<TG, TW>::V;
  if (columns.n == 1) emb_sums<TG, TW, 1, true>(a, st);
  else if (columns.aligned) emb_sums<TG, TW, V, true>(a, st);
  else emb_sums<TG, TW, V, false>(a, st);
}

// f<A, B>() for two of the three types
template <class A, class F>
static void emb_type2(int b, F&& f) {
  if (b == CONCORD_F32) f(A{}, float{});
  else if (b == CONCORD_BF16) f(A{}, BF16{});
  else f(A{}, (_Float16)0);
}
template <class F>
static void emb_types(int a, int b, F&& f) {
  if (a == CONCORD_F32) emb_type2<float>(b, f);
  else if (a == CONCORD_BF16) emb_type2<BF16>(b, f);
  else emb_type2<_Float16>(b, f);
}

static bool emb_sizes_ok(int64_t n, int64_t V, int64_t C) {
  return n >= 0 && V >= 0 && C >= 1 && n < (1LL << 31) && V < (1LL << 31) - 1 && C < (1LL << 21);
}

}  // namespace concord

using namespace concord;

extern "C" int concord_embedding_fwd(const void* tokens, int index64, int64_t n, const void* table, int64_t ld_t,
                                     int wdtype, int64_t V, int64_t C, float scale, void* out, int64_t ld_o, int dtype,
                                     void* stream) {
  CONCORD_CHECK(emb_sizes_ok(n, V, C), "concord_embedding_fwd: bad size");
  CONCORD_CHECK(emb_dtype_ok(dtype) && emb_dtype_ok(wdtype), "concord_embedding_fwd: bad type");
  CONCORD_CHECK(__builtin_isfinite(scale), "concord_embedding_fwd: the scale must be finite");
  CONCORD_CHECK(ld_t >= C && ld_o >= C, "concord_embedding_fwd: leading dimension < C");
  if (n == 0) return CONCORD_OK;
  CONCORD_CHECK(tokens && out && (table || V == 0), "concord_embedding_fwd: NULL argument");
  EmbArgs a{};
  a.tokens = tokens, a.idx64 = index64, a.n = n, a.V = (uint32_t)V, a.C = C, a.scale = scale;
  a.src = table, a.lds = ld_t, a.dst = out, a.ldd = ld_o;
  const EmbColumns columns = emb_columns(a, wdtype, dtype);
  emb_types(wdtype, dtype, [&](auto w, auto o) { emb_fwd<decltype(w), decltype(o)>(a, columns, (hipStream_t)stream); });
  return launch_status("embedding_fwd");
}

extern "C" size_t concord_embedding_workspace_bytes(int64_t n, int64_t V, int64_t C) {
  if (!emb_sizes_ok(n, V, C) || n == 0 || V == 0) return 0;
  return emb_workspace(n, C).bytes;
}

extern "C" int concord_embedding_bwd(const void* tokens, int index64, int64_t n, const void* dy, int64_t ld_dy, int dtype,
                                     int64_t V, int64_t C, float scale, void* dtable, int64_t ld_dt, int wdtype,
                                     void* workspace, size_t workspace_bytes, void* stream) {
  CONCORD_CHECK(emb_sizes_ok(n, V, C), "concord_embedding_bwd: bad size");
  CONCORD_CHECK(emb_dtype_ok(dtype) && emb_dtype_ok(wdtype), "concord_embedding_bwd: bad type");
  CONCORD_CHECK(__builtin_isfinite(scale), "concord_embedding_bwd: the scale must be finite");
  CONCORD_CHECK(ld_dy >= C && ld_dt >= C, "concord_embedding_bwd: leading dimension < C");
  if (V == 0) return CONCORD_OK;
  CONCORD_CHECK(dtable && (n == 0 || (tokens && dy)), "concord_embedding_bwd: NULL argument");
  const EmbWorkspace w = emb_workspace(n, C);
  if (n > 0 && (!workspace || workspace_bytes < w.bytes)) {
    set_error("concord_embedding_bwd: workspace of %zu bytes needed", w.bytes);
    return CONCORD_EWORKSPACE;
  }
  CONCORD_CHECK(((uintptr_t)workspace & 15) == 0, "concord_embedding_bwd: the workspace is not on 16 bytes");
  hipStream_t st = (hipStream_t)stream;
  EmbArgs a{};
  a.tokens = tokens, a.idx64 = index64, a.n = n, a.V = (uint32_t)V, a.C = C, a.scale = scale;
  a.src = dy, a.lds = ld_dy, a.dst = dtable, a.ldd = ld_dt;
  a.piece = emb_piece(n), a.pieces = cdiv(n, a.piece);
  const EmbColumns columns = emb_columns(a, dtype, wdtype);
  a.slabs = cdiv(C, 64 * columns.n);
  CONCORD_CHECK(grid_fits(cdiv(a.pieces * a.slabs, 4) + cdiv(V, 4 * kFillRows), 256) && grid_fits(a.pieces * a.slabs, 512),
                "concord_embedding_bwd: too many tokens or rows");
  uint32_t *keys[2] = {}, *pos[2] = {};
  int at = 0;
  if (n > 0) {
    char* base = (char*)workspace;
    for (int i = 0; i < 2; ++i) {
      keys[i] = (uint32_t*)(base + w.keys[i]);
      pos[i] = (uint32_t*)(base + w.pos[i]);
    }
    a.part = (float*)(base + w.part);
    int bits = 1;
    while (V >> bits) ++bits;   // (V itself stands for what is outside)
    const int passes = (bits + kMaxBits - 1) / kMaxBits, each = (bits + passes - 1) / passes;
    if (n <= kOneBlock) {
      if (n <= 1024) hipLaunchKernelGGL((emb_sort_block_kernel<1>), dim3(1), dim3(1024), 0, st, a, passes, each, keys[0], pos[0]);
      else hipLaunchKernelGGL((emb_sort_block_kernel<kOneBlock / 1024>), dim3(1), dim3(1024), 0, st, a, passes, each, keys[0], pos[0]);
    } else {
      const int tile = emb_tile(n);
      const dim3 grid((unsigned)cdiv(n, tile));
      const bool scan = grid.x > kScanBlocks;
      for (int p = 0; p < passes; ++p) {
        SortPass s{};
        if (p) s.keys = keys[at ^ 1], s.pos = pos[at ^ 1];
        s.out_keys = keys[at], s.out_pos = pos[at], s.counts = (uint32_t*)(base + w.counts);
        if (scan) s.totals = (uint32_t*)(base + w.totals);
        s.shift = p * each, s.bits = each;
        if (tile == 1024) {
          hipLaunchKernelGGL((emb_count_kernel<2>), grid, dim3(512), 0, st, a, s);
          hipLaunchKernelGGL((emb_scatter_kernel<2>), grid, dim3(512), 0, st, a, s);
        } else {
          hipLaunchKernelGGL((emb_count_kernel<8>), grid, dim3(512), 0, st, a, s);
          if (scan) hipLaunchKernelGGL(emb_scan_kernel, dim3((unsigned)cdiv(1 << each, 64)), dim3(1024), 0, st, s, grid.x);
          hipLaunchKernelGGL((emb_scatter_kernel<8>), grid, dim3(512), 0, st, a, s);
        }
        at ^= 1;
      }
      at ^= 1;
    }
  }
  a.keys = keys[at], a.pos = pos[at];
  emb_types(dtype, wdtype, [&](auto g, auto t) { emb_bwd<decltype(g), decltype(t)>(a, columns, st); });
  return launch_status("embedding_bwd");
}
