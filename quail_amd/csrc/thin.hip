// Thinning of kept keys: of each (layer, sequence, KV head) the rows of most
// weight stay, in place.
//
// With u = used rows and k = min(u, keep), the first `sinks` rows, the last
// `recent` and the heaviest of the others stay, k in all (ties: the lowest row;
// a NaN is heavier than every number). A row that moves leaves the order of the
// tokens, so the last rows of a sequence that was thinned before are its newest
// tokens only if it grew by as many since: by token, each row's number goes with
// it, and the tokens below `sinks` and the newest stay instead, wherever their
// rows lie. Kept rows below k stay where they are;
// the j-th dropped slot below k takes the j-th kept row at or past k. So every
// row that is read for a move lies at or past k and every one that is written
// below it: the moves need no order among them, and only what has to move
// does (a sequence that grew by 64 rows moves at most 64 a head, where keeping
// the rows' order would move all behind the first gap).
#include "qx_common.h"
#include "qx_status.h"

namespace qx {
namespace {

constexpr int kPage = 16;
constexpr int kMaxKeys = 2560 * kPage;  // as the paged attention's

struct ThinArgs {
  uint8_t* pools;  // K and V of layer 0, K of layer 1, ...
  int64_t pool_stride;
  uint8_t* scales;
  int64_t scale_stride;
  const float* w;
  int64_t w_layer, w_seq, w_head;
  const int *used, *table;
  int64_t table_ld;
  int seqs, HK, bound, cols, keep, slots, sinks, recent;
  int* kept;   // (layers, seqs, HK, slots)
  float* out;  // (layers, seqs, HK, cols)
  // by token: each row's number (negative: appended since the last thinning), the
  // tokens so far of a sequence, and the numbers left, (layers, seqs, HK, cols);
  // `recent` counts the newest tokens then
  const int* tokens;
  int64_t t_layer, t_seq, t_head;
  const int* total;
  int* left;
};

// A float's rank as an unsigned number; -0 ranks as 0, NaN above all
__device__ __forceinline__ uint32_t rank_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  if (f != f) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// the sum of v over the lanes up to this one, on vector operands (through LDS
// permutes the three scans took a third of a short call's time)
__device__ __forceinline__ int wave_sum_to(int v) {
#define QX_STEP(CTRL, ROWS) v += __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false)
  QX_STEP(0x111, 0xf);  // from 1, 2, 4 and 8 lanes below in the row of 16
  QX_STEP(0x112, 0xf);
  QX_STEP(0x114, 0xf);
  QX_STEP(0x118, 0xf);
  QX_STEP(0x142, 0xa);  // the row's last lane into the next row, of rows 1 and 3
  QX_STEP(0x143, 0xc);  // lane 31 into the upper rows
#undef QX_STEP
  return v;
}

// the sum of v over the threads before, and over all of W waves; sums: W in LDS
template <int W>
__device__ __forceinline__ int block_sum_before(int v, int lane, int wave, int* sums, int* total) {
  const int to = wave_sum_to(v);
  if (lane == 63) sums[wave] = to;
  __syncthreads();
  const int waves = wave_sum_to(lane < W ? sums[lane] : 0);
  *total = __builtin_amdgcn_readlane(waves, W - 1);
  return to - v + (wave ? __builtin_amdgcn_readlane(waves, wave - 1) : 0);
}

__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// bits [lo, hi) of a word whose first bit is number `base`
__device__ __forceinline__ uint64_t bits(int lo, int hi, int base) {
  const int a = min(max(lo - base, 0), 64), b = min(max(hi - base, 0), 64);
  const uint64_t below_b = b == 64 ? ~0ull : (1ull << b) - 1;
  return a >= b ? 0 : below_b & ~((1ull << a) - 1);
}

// One (layer, sequence, head) per workgroup, its weights' ranks in registers,
// E a thread (row e * NT + thread); 0 stands for a row that is protected or not
// there (no weight ranks so low). BY_TOKEN protects rows anywhere: they rank above
// all others instead (a NaN just below them) and count among the k, so that k rows
// stay whatever numbers a caller gives. The border, the rank of the last row kept, is
// found 11, 11 and 10 bits at a time from histograms in LDS, of which the second
// and third count few rows, if they are needed at all. What stays is then a bit a row, in words of 64 rows
// (a wave's ballots), and dropped slots and movers are numbered by words. Bound
// by instructions (some 60 a row) and, where rows are few, by the barriers
// between these steps; 8 bytes a row from and to memory, 16 by token (2304 heads of
// 1088 rows 23 us either way, 288 of 8003 rows 16.0 and 18.1, of 39,990 50 and 59).
template <int NT, int E, bool BY_TOKEN>
__global__ __launch_bounds__(NT, NT == 1024 ? 8 : 4) void thin_select_kernel(ThinArgs p) {
  constexpr int W = NT / 64, WORDS = E * W, BINS = 2048, PER = BINS / NT;
  __shared__ int hist[BINS];
  __shared__ uint64_t stays[WORDS];
  __shared__ int before[WORDS];  // flagged rows before a word's
  __shared__ int sums[W];
  __shared__ int found[3];  // bin, rows above it, rows in it
  __shared__ uint16_t movers[NT * E / 2];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t row = blockIdx.x;
  const int h = (int)(row % p.HK);
  const int64_t ls = row / p.HK;
  const int s = (int)(ls % p.seqs);
  const float* w = p.w + ls / p.seqs * p.w_layer + s * p.w_seq + h * p.w_head;
  int* kept = p.kept + row * p.slots;
  float* out = p.out + row * p.cols;
  const int used = min(max(p.used[s], 0), p.bound);
  const int* tokens = nullptr;
  int* left = nullptr;
  int newer = 0;                // the number of row i is i + newer where none is given
  int first_token = 0, fresh = 0;  // tokens [first_token, fresh) may leave
  if constexpr (BY_TOKEN) {
    tokens = p.tokens + ls / p.seqs * p.t_layer + s * p.t_seq + h * p.t_head;
    left = p.left + row * p.cols;
    const int total = max(p.total[s], used);
    newer = total - used;
    first_token = p.sinks;
    fresh = total - p.recent;
  }
  auto number_at = [&](int i, int given) { return given < 0 ? i + newer : given; };
  if (used <= p.keep) {
    for (int i = tid; i < p.cols; i += NT) out[i] = i < used ? w[i] : 0.f;
    for (int i = tid; i < p.slots; i += NT) kept[i] = i < used ? i : -1;
    if constexpr (BY_TOKEN)
      for (int i = tid; i < p.cols; i += NT) left[i] = i < used ? number_at(i, tokens[i]) : -1;
    return;
  }
  const int k = p.keep;
  const int early = BY_TOKEN ? 0 : p.sinks, late = BY_TOKEN ? used : used - p.recent;
  int want = BY_TOKEN ? k : k - p.sinks - p.recent;  // of the rows [early, late), which are more
  const bool none = want == 0;
  uint32_t rank[E];
  uint32_t border = 0;
  int equal = 0;
  auto count = [&](int bin) {
    // a wave whose rows are all of one bin counts them at once (weights of
    // keys that never had any are all 0)
    const int first = __builtin_amdgcn_readfirstlane(bin);
    if (__ballot(bin != first) == 0) {
      const uint64_t active = __ballot(1);
      if (lanes_before(active) == 0) atomicAdd(&hist[bin], (int)__popcll(active));
    } else {
      atomicAdd(&hist[bin], 1);
    }
  };
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    // (all of the border's bin stay: its last bits do not matter)
    if (pass > 0 && (none || want == equal)) continue;
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, width = pass == 2 ? 10 : 11;
    for (int i = tid; i < BINS; i += NT) hist[i] = 0;
    __syncthreads();
    if (pass == 0) {
      constexpr int AT_ONCE = E < 8 ? E : 8;  // loads in flight
#pragma unroll
      for (int e0 = 0; e0 < E; e0 += AT_ONCE) {
        const int t = opaque(tid);
        int given[BY_TOKEN ? AT_ONCE : 1];
#pragma unroll
        for (int e = e0; e < e0 + AT_ONCE; ++e) {
          rank[e] = __float_as_uint(w[min(e * NT + t, used - 1)]);
          if constexpr (BY_TOKEN) given[e - e0] = tokens[min(e * NT + t, used - 1)];
        }
#pragma unroll
        for (int e = e0; e < e0 + AT_ONCE; ++e) {
          const int first = e * NT + wave * 64;
          rank[e] = rank_of(__uint_as_float(rank[e]));
          if constexpr (BY_TOKEN) {
            const int token = number_at(e * NT + t, given[e - e0]);
            const bool stays = token < first_token || token >= fresh;
            rank[e] = stays ? 0xffffffffu : min(rank[e], 0xfffffffeu);
          }
          if (first >= early && first + 64 <= late) {
            count(rank[e] >> 21);
          } else {
            const int i = e * NT + t;
            if (i >= early && i < late) count(rank[e] >> 21); else rank[e] = 0;
          }
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (rank[e] >> (shift + width) == border >> (shift + width))
          count((rank[e] >> shift) & ((1 << width) - 1));
    }
    __syncthreads();
    // bins from the top, PER a thread
    int bins[PER], mine = 0;
#pragma unroll
    for (int b = 0; b < PER; ++b) mine += bins[b] = hist[BINS - 1 - (tid * PER + b)];
    int total;
    int above = block_sum_before<W>(mine, lane, wave, sums, &total);
    if (above < want && want <= above + mine) {
#pragma unroll
      for (int b = 0; b < PER; ++b) {
        if (above < want && want <= above + bins[b]) {
          found[0] = BINS - 1 - (tid * PER + b);
          found[1] = above;
          found[2] = bins[b];
        }
        above += bins[b];
      }
    }
    __syncthreads();
    if (!none) {
      border |= (uint32_t)__builtin_amdgcn_readfirstlane(found[0]) << shift;
      want -= __builtin_amdgcn_readfirstlane(found[1]);
      equal = __builtin_amdgcn_readfirstlane(found[2]);
    }
  }
  // Word c holds rows [64 c, 64 c + 64); wave v has the words v, v + W, ...
  // number(flags): the set bits of the words before each word, and of all
  const int words = (used + NT - 1) / NT * W;
  auto number = [&](auto flags) {
    int total;
    static_assert(WORDS <= NT, "a word a thread");
    const int n = block_sum_before<W>(tid < words ? (int)__popcll(flags(tid)) : 0, lane, wave, sums, &total);
    if (tid < words) before[tid] = n;
    __syncthreads();
    return total;
  };
  const bool ties = want != equal;  // not all of the border's rank stay
  if (ties) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t m = __ballot(rank[e] == border);
      if (lane == 0) stays[e * W + wave] = m;
    }
    __syncthreads();
    number([&](int c) { return stays[c]; });
  }
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int c = e * W + wave;
    uint64_t m = __ballot(ties ? rank[e] > border : rank[e] >= border);
    if (ties) {
      const uint64_t same = stays[c];
      m |= __ballot((same >> lane & 1) && before[c] + lanes_before(same) < want);
    }
    if (none) m = 0;
    if constexpr (!BY_TOKEN)
      if (64 * c < early || 64 * c + 64 > late) m |= bits(0, early, 64 * c) | bits(late, used, 64 * c);
    if (lane == 0) stays[c] = m;
  }
  __syncthreads();
  // dropped slots below k, then (numbered behind them) movers from k on
  auto flagged = [&](int c) {
    const uint64_t m = stays[c];
    if (64 * c + 64 <= k) return ~m;
    return 64 * c >= k ? m : m ^ bits(0, k, 64 * c);
  };
  const int holes = number(flagged) / 2;
  // row 64 c + lane's number among the flagged ones, or -1
  auto number_of = [&](int c) {
    const uint64_t m = flagged(c);
    const int n = before[c] + lanes_before(m);
    return m >> lane & 1 ? n : -1;
  };
  constexpr int AT_ONCE = 4;  // words of a wave in flight
  for (int c0 = k / 64; c0 < words; c0 += AT_ONCE * W) {
    int n[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int c = c0 + j * W + wave;
      n[j] = c < words ? number_of(c) : -1;
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j)
      if (n[j] >= holes) movers[n[j] - holes] = (uint16_t)((c0 + j * W + wave) * 64 + lane);
  }
  __syncthreads();
  for (int c0 = 0; c0 * 64 < k; c0 += AT_ONCE * W) {
    int src[AT_ONCE], given[BY_TOKEN ? AT_ONCE : 1];
    float f[AT_ONCE];
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int c = min(c0 + j * W + wave, (k - 1) / 64), n = number_of(c);
      src[j] = n < 0 ? c * 64 + lane : n < holes ? movers[n] : 0;  // (0: past k)
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      f[j] = w[min(src[j], used - 1)];
      if constexpr (BY_TOKEN) given[j] = tokens[min(src[j], used - 1)];
    }
#pragma unroll
    for (int j = 0; j < AT_ONCE; ++j) {
      const int i = (c0 + j * W + wave) * 64 + lane;
      if (i < k) {
        kept[i] = src[j];
        out[i] = f[j];
        if constexpr (BY_TOKEN) left[i] = number_at(src[j], given[j]);
      }
    }
  }
  for (int i = k + tid; i < p.cols; i += NT) {
    out[i] = 0.f;
    if constexpr (BY_TOKEN) left[i] = -1;
  }
}

// The moves of a wave: 64 slots of a (layer, sequence, head), one a lane. Those
// whose row moves are listed in LDS. (256 slots a wave, for more moves in each:
// 8 to 10% slower, with few moves among the slots or many.)
struct Place {
  int h;
  int64_t layer, head;  // head: of kept
  const int* table;
  int slot;
};

__device__ __forceinline__ Place place_of(const ThinArgs& p, int64_t wid, int parts, int lane) {
  Place x;
  x.h = (int)(wid % p.HK);
  const int64_t ls = wid / p.HK / parts;
  x.layer = ls / p.seqs;
  x.head = ls * p.HK + x.h;
  x.table = p.table + ls % p.seqs * p.table_ld;
  x.slot = (int)(wid / p.HK % parts) * 64 + lane;
  return x;
}

__device__ __forceinline__ int source(const ThinArgs& p, const Place& x) {
  return x.slot < p.slots ? p.kept[x.head * p.slots + x.slot] : -1;
}

// A row of D values goes by D * 2 / 16 lanes, 16 bytes each, K and V of kBatch
// rows a lane in flight, past the caches (each is read and written once; 4%).
// Bound by HBM, in pieces of a head's row: 8003 rows to 2000 in 36 layers of 8 heads
// of 128, both launches 110 us, 91 at a copy's rate.
template <int D>
__global__ __launch_bounds__(256) void thin_move_kernel(ThinArgs p, int64_t waves, int parts) {
  constexpr int LPR = D / 8, RPP = 64 / LPR, kBatch = 4;
  __shared__ int64_t list[4][64][2];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t wid = (int64_t)blockIdx.x * 4 + wave;
  if (wid >= waves) return;
  const Place x = place_of(p, wid, parts, lane);
  const int src = source(p, x);
  const bool moves = src >= 0 && src != x.slot;
  const uint64_t mask = __ballot(moves);
  const int n = __popcll(mask);
  if (moves) {
    int64_t* to = list[wave][lanes_before(mask)];
    to[0] = (int64_t)x.table[x.slot / kPage] * kPage + x.slot % kPage;
    to[1] = (int64_t)x.table[src / kPage] * kPage + src % kPage;
  }
  if (n == 0) return;
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own list
  uint8_t* k_pool = p.pools + 2 * x.layer * p.pool_stride + (int64_t)x.h * D * 2;
  uint8_t* v_pool = k_pool + p.pool_stride;
  const int64_t row_bytes = (int64_t)p.HK * D * 2;
  const int at = lane % LPR * 16;
  for (int m0 = lane / LPR; m0 < n; m0 += RPP * kBatch) {
    v4i kv[kBatch][2];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = min(m0 + b * RPP, n - 1);  // a row again: no branch between the loads
      const int64_t from = list[wave][m][1] * row_bytes + at;
      kv[b][0] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(k_pool + from));
      kv[b][1] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(v_pool + from));
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = m0 + b * RPP;
      if (m >= n) continue;
      const int64_t to = list[wave][m][0] * row_bytes + at;
      __builtin_nontemporal_store(kv[b][0], reinterpret_cast<v4i*>(k_pool + to));
      __builtin_nontemporal_store(kv[b][1], reinterpret_cast<v4i*>(v_pool + to));
    }
  }
}

// The 8 codes of a word pair times 2^shift, shift <= 0 (exact unless they
// become subnormal)
__device__ __forceinline__ uint2 shifted8(uint2 c, int shift) {
  float y[8] = {__builtin_amdgcn_cvt_f32_fp8(c.x, 0), __builtin_amdgcn_cvt_f32_fp8(c.x, 1),
                __builtin_amdgcn_cvt_f32_fp8(c.x, 2), __builtin_amdgcn_cvt_f32_fp8(c.x, 3),
                __builtin_amdgcn_cvt_f32_fp8(c.y, 0), __builtin_amdgcn_cvt_f32_fp8(c.y, 1),
                __builtin_amdgcn_cvt_f32_fp8(c.y, 2), __builtin_amdgcn_cvt_f32_fp8(c.y, 3)};
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __builtin_ldexpf(y[i], shift);
  return make_uint2(pack4_fp8(y[0], y[1], y[2], y[3]), pack4_fp8(y[4], y[5], y[6], y[7]));
}
__device__ __forceinline__ v4i shifted16(v4i c, int shift) {
  if (shift == 0) return c;
  const uint2 a = shifted8(make_uint2(c[0], c[1]), shift), b = shifted8(make_uint2(c[2], c[3]), shift);
  return v4i{(int)a.x, (int)a.y, (int)b.x, (int)b.y};
}

// The same over 8-bit pages. A page that a row moves into gets the largest
// scale of those its rows come with (its own among them, where a row stays);
// the codes of the others are shifted down to it, those of rows that stay too.
// `keep` is whole pages, so no page is both read for a move and written.
// A scale outlives the large row that it was for and goes with the page's other
// rows, but never passes the largest that a row of the head was written with; over
// any number of thinnings a value is off by less than 2^-9 of the scale it has then
// (half a subnormal step each time the scale rises, by a factor of 2 or more).
template <int D>
__global__ __launch_bounds__(256) void thin_move8_kernel(ThinArgs p, int64_t waves, int parts) {
  constexpr int LPR = D / 16, RPP = 64 / LPR, kBatch = 4;
  __shared__ int64_t list[4][64][2];
  __shared__ int shifts[4][64];  // K's and V's, 16 bits each
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t wid = (int64_t)blockIdx.x * 4 + wave;
  if (wid >= waves) return;
  const Place x = place_of(p, wid, parts, lane);
  const int src = source(p, x);
  const bool moves = src >= 0 && src != x.slot;
  const uint64_t moving = __ballot(moves);
  if (moving == 0) return;
  uint8_t* scales = p.scales + x.layer * p.scale_stride;
  // whether a row moves into the lane's page; then all 16 of its slots hold rows
  const bool page_moves = (moving >> (lane & 48) & 0xffff) != 0;
  int64_t to = 0, from = 0;
  int bk = 0, bv = 0;
  if (page_moves) {
    to = x.table[x.slot / kPage];
    from = x.table[src / kPage];
    const uint16_t b = *reinterpret_cast<const uint16_t*>(scales + (from * p.HK + x.h) * 2);
    bk = b & 0xff;
    bv = b >> 8;
  }
  int top_k = bk, top_v = bv;
#pragma unroll
  for (int o = kPage / 2; o > 0; o >>= 1) {
    top_k = max(top_k, __shfl_xor(top_k, o, 64));
    top_v = max(top_v, __shfl_xor(top_v, o, 64));
  }
  const bool write = page_moves && (moves || bk != top_k || bv != top_v);
  const uint64_t mask = __ballot(write);
  const int n = __popcll(mask);
  if (write) {
    const int m = lanes_before(mask);
    list[wave][m][0] = to * kPage + x.slot % kPage;
    list[wave][m][1] = from * kPage + src % kPage;
    shifts[wave][m] = (top_k - bk) | (top_v - bv) << 16;
  }
  if (page_moves && lane % kPage == 0)
    *reinterpret_cast<uint16_t*>(scales + (to * p.HK + x.h) * 2) = (uint16_t)(top_k | top_v << 8);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the wave's own list
  uint8_t* k_pool = p.pools + 2 * x.layer * p.pool_stride + (int64_t)x.h * D;
  uint8_t* v_pool = k_pool + p.pool_stride;
  const int64_t row_bytes = (int64_t)p.HK * D;
  const int at = lane % LPR * 16;
  for (int m0 = lane / LPR; m0 < n; m0 += RPP * kBatch) {
    v4i kv[kBatch][2];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = min(m0 + b * RPP, n - 1);
      const int64_t row = list[wave][m][1] * row_bytes + at;
      kv[b][0] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(k_pool + row));
      kv[b][1] = __builtin_nontemporal_load(reinterpret_cast<const v4i*>(v_pool + row));
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = m0 + b * RPP;
      if (m >= n) continue;
      const int64_t row = list[wave][m][0] * row_bytes + at;
      const int shift = shifts[wave][m];
      __builtin_nontemporal_store(shifted16(kv[b][0], -(shift & 0xffff)), reinterpret_cast<v4i*>(k_pool + row));
      __builtin_nontemporal_store(shifted16(kv[b][1], -(shift >> 16)), reinterpret_cast<v4i*>(v_pool + row));
    }
  }
}

struct ByToken {
  const int* tokens;
  int64_t layer, seq, head;
  const int* total;
  int* left;
};

int thin_rows(void* pools, int64_t pool_stride, int64_t element_bytes, void* scales,
              int64_t scale_stride, const float* weights, int64_t w_layer, int64_t w_seq,
              int64_t w_head, const ByToken* by, const int* used, const int* table, int64_t table_ld,
              int64_t layers, int64_t seqs, int64_t HK, int64_t D, int64_t page, int64_t max_used,
              int64_t cols, int64_t keep, int64_t sinks, int64_t recent, int* kept, float* out,
              hipStream_t stream) {
  QX_CHECK(D == 64 || D == 128, "thin_rows: head_dim %lld (64 or 128)", (long long)D);
  QX_CHECK(page == kPage, "thin_rows: page of %lld tokens (16)", (long long)page);
  QX_CHECK(element_bytes == 2 || (element_bytes == 1 && scales),
           "thin_rows: rows of 2-byte values, or of codes with scales");
  QX_CHECK(layers >= 0 && seqs >= 0 && HK > 0 && cols >= 0 && cols < (1LL << 30),
           "thin_rows: %lld layers, %lld sequences, %lld heads, %lld columns", (long long)layers,
           (long long)seqs, (long long)HK, (long long)cols);
  QX_CHECK(max_used >= 0 && max_used <= cols && max_used <= kMaxKeys,
           "thin_rows: up to %lld rows (%lld columns of weights; at most %d)", (long long)max_used,
           (long long)cols, kMaxKeys);
  QX_CHECK(sinks >= 0 && recent >= 0 && keep >= 0 && sinks + recent <= keep,
           "thin_rows: %lld first and %lld last rows of %lld that stay", (long long)sinks,
           (long long)recent, (long long)keep);
  QX_CHECK(element_bytes == 2 || keep % kPage == 0,
           "thin_rows: 8-bit pages are kept whole, not %lld rows", (long long)keep);
  QX_CHECK(pool_stride % 16 == 0 && ((uintptr_t)pools & 15) == 0, "thin_rows: alignment");
  const int64_t rows = layers * seqs * HK;
  if (rows == 0 || cols == 0) return QX_OK;
  const int64_t slots = keep < cols ? keep : cols;
  QX_CHECK(pools && weights && used && out && (kept || slots == 0) && (table || max_used == 0),
           "thin_rows: null pointer");
  QX_CHECK(!by || (by->tokens && by->total && by->left), "thin_rows: null pointer");
  QX_CHECK(rows < (1LL << 21), "thin_rows: %lld heads exceed one launch", (long long)rows);
  const int parts = (int)((slots + 63) / 64);
  const int64_t waves = rows * parts;
  QX_CHECK(waves <= (1LL << 26) - 4, "thin_rows: %lld rows of %lld heads exceed one launch",
           (long long)slots, (long long)rows);
  ThinArgs a{(uint8_t*)pools, pool_stride, (uint8_t*)scales, scale_stride, weights, w_layer, w_seq,
             w_head, used, table, table_ld, (int)seqs, (int)HK, (int)max_used, (int)cols,
             (int)(keep < kMaxKeys ? keep : kMaxKeys), (int)slots, (int)sinks, (int)recent, kept, out,
             nullptr, 0, 0, 0, nullptr, nullptr};
  if (by) {
    a.tokens = by->tokens;
    a.t_layer = by->layer, a.t_seq = by->seq, a.t_head = by->head;
    a.total = by->total;
    a.left = by->left;
  }
  // A thread's rows as few as the bound allows (each step is done for all E), in
  // as few waves as hold them in registers, since barriers among many cost more:
  // of 2304 heads 1088 rows 26.5 us, by 16 waves 51; 4000 rows 49.5 and 65, 8000
  // rows 80 and 93 (by 4 waves 49.5 and 82.5). 288 heads leave CUs to spare: 4000
  // rows 16.8 and 17.1, 8000 rows 24.0 and 23.7 (by 4 waves 18.5 and 29). Of 20,000
  // rows 24 a thread 46, 40 56.
#define QX_SELECT(NT, E, B) \
  hipLaunchKernelGGL((thin_select_kernel<NT, E, B>), dim3((unsigned)rows), dim3(NT), 0, stream, a)
#define QX_THIN(NT, E) \
  if (by) QX_SELECT(NT, E, true); else QX_SELECT(NT, E, false)
  if (max_used <= 1024) {
    QX_THIN(256, 4);
  } else if (max_used <= 2048) {
    QX_THIN(256, 8);
  } else if (max_used <= 4096) {
    QX_THIN(512, 8);
  } else if (max_used <= 8192) {
    QX_THIN(512, 16);
  } else if (max_used <= 16384) {
    QX_THIN(1024, 16);
  } else if (max_used <= 24576) {
    QX_THIN(1024, 24);
  } else {
    QX_THIN(1024, 40);
  }
#undef QX_THIN
#undef QX_SELECT
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (max_used <= keep) return QX_OK;  // no row moves
  const dim3 grid((unsigned)((waves + 3) / 4)), block(256);
#define QX_MOVE(K, DD) hipLaunchKernelGGL((K<DD>), grid, block, 0, stream, a, waves, parts)
  if (waves) {
    if (element_bytes == 2) {
      if (D == 128) QX_MOVE(thin_move_kernel, 128); else QX_MOVE(thin_move_kernel, 64);
    } else {
      if (D == 128) QX_MOVE(thin_move8_kernel, 128); else QX_MOVE(thin_move8_kernel, 64);
    }
  }
#undef QX_MOVE
  QX_LAUNCH_STATUS();
}

}  // namespace
}  // namespace qx

using namespace qx;

extern "C" {

int qx_thin_rows(void* pools, int64_t pool_stride, int64_t element_bytes, void* scales,
                 int64_t scale_stride, const float* weights, int64_t w_layer, int64_t w_seq,
                 int64_t w_head, const int* used, const int* table, int64_t table_ld,
                 int64_t layers, int64_t seqs, int64_t HK, int64_t D, int64_t page,
                 int64_t max_used, int64_t cols, int64_t keep, int64_t sinks, int64_t recent,
                 int* kept, float* out, hipStream_t stream) {
  return thin_rows(pools, pool_stride, element_bytes, scales, scale_stride, weights, w_layer, w_seq,
                   w_head, nullptr, used, table, table_ld, layers, seqs, HK, D, page, max_used, cols,
                   keep, sinks, recent, kept, out, stream);
}

int qx_thin_rows_by_token(void* pools, int64_t pool_stride, int64_t element_bytes, void* scales,
                          int64_t scale_stride, const float* weights, int64_t w_layer, int64_t w_seq,
                          int64_t w_head, const int* tokens, int64_t t_layer, int64_t t_seq,
                          int64_t t_head, const int* total, const int* used, const int* table,
                          int64_t table_ld, int64_t layers, int64_t seqs, int64_t HK, int64_t D,
                          int64_t page, int64_t max_used, int64_t cols, int64_t keep, int64_t sinks,
                          int64_t newest, int* kept, float* out, int* left, hipStream_t stream) {
  const ByToken by{tokens, t_layer, t_seq, t_head, total, left};
  return thin_rows(pools, pool_stride, element_bytes, scales, scale_stride, weights, w_layer, w_seq,
                   w_head, &by, used, table, table_ld, layers, seqs, HK, D, page, max_used, cols,
                   keep, sinks, newest, kept, out, stream);
}

}  // extern "C"
