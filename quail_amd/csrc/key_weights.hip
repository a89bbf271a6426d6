// The attention weight that each key has gathered: for sequence s, KV head h
// and key j
//   out[s, h, j] = base[s, h, j] + sum over rows i that see j and heads g of h's group of
//                  exp(scale q[i, g] . k[j, h] - lse[g, i])
// over pages of 16 rows, bf16 or e4m3 codes with a scale per (page, head).
//
// A wave holds 32 KT keys of one KV head in registers, as the A operand of
// v_mfma_f32_32x32x16_bf16, and the (row, head of the group) pairs of the
// sequence stream past it as its columns, kCols of them a step, through LDS
// (four waves share them). Rows are keys, so a column's log-sum-exp is one value
// a lane and a key's sum stays in one register across the steps: a score costs
// one multiply-add, one exponential and one addition, and lanes are added up
// once, at the end. Sums are fp32, in an order that the call's lengths fix: no
// atomics.
//
// Few rows (a token or a question a sequence): a workgroup for each (sequence,
// head, key tile) reads its keys once and writes the result itself; the keys' bytes
// bound it. Many rows: 512 workgroups, two a CU, share the groups of rows of all tiles
// evenly, whatever the sequences' lengths; a tile's parts go to scratch memory
// and a second launch adds them up in the order of the rows. There a step of 64
// columns with a wave's 64 keys is 32 MFMAs of 32 cycles (8003 rows of 32 heads,
// causal, 218 us at the rate of a large product), and the 64 exponentials a lane
// cost the vector unit as long, so that the two have to run side by side
// (item_sums). 8003 rows of 32/8 heads of 128 take 261-278 us on several cards, an
// AI.IF pack of 46 sequences over a kept prefix 71-74.
#include "qx_common.h"
#include "qx_status.h"

#include <algorithm>
#include <type_traits>

namespace qx {
namespace {

constexpr int kPage = 16;
constexpr int kMaxKeys = 2560 * kPage;
constexpr int kCols = 64;            // (row, head) columns of a step
constexpr int kSeqs = 2048;          // sequences of one launch (their bounds in LDS)
constexpr int kShares = 512;         // workgroups that the work is shared by: two a CU
constexpr int kStart = 8;            // groups that a key tile's start takes as long as (0: 8003 rows 332 us, 8: 288)
constexpr int kFirst = 40;           // of 64: the part of a pair's groups that its first workgroup has
constexpr int kMinShare = 2;         // groups of a share, at least
constexpr float kLog2e = 1.4426950408889634f;

struct WeightsArgs {
  const uint16_t* q;
  int64_t q_ld;
  const float* lse;
  int64_t lse_ld;
  const uint8_t *k, *scales;
  const int *cu_q, *used, *table;
  int64_t table_ld;
  const float* base;
  int64_t base_s, base_h;
  float* out;
  int64_t out_s, out_h;
  float* part;
  int* bound;
  int seqs, HK, G, rows, max_q, max_used, cols, tiles;
  int step_rows, blocks;  // rows of a step; steps that a row's heads take (G > kCols)
  int start;              // groups that a tile's start is counted as
  int drop;               // groups that a tile has fewer than the one before
  int row_limit;          // rows whose elements 32 bits of bytes reach
  float scale_log2;
  int causal;
};

// Keys of a workgroup whose waves hold KT tiles of 32
constexpr int tile_keys(int KT) { return 4 * 32 * KT; }

// A sequence: its first row, rows, keys
struct Seq {
  int q0, n, used;
};

__device__ __forceinline__ Seq seq_of(const WeightsArgs& p, int s) {
  Seq x;
  x.q0 = min(max(p.cu_q[s], 0), p.rows);
  x.n = min(min(max(p.cu_q[s + 1] - x.q0, 0), p.rows - x.q0), p.max_q);
  x.used = min(max(p.used[s], 0), p.max_used);
  return x;
}

// keys that row i of the sequence sees: [0, seen)
__device__ __forceinline__ int seen_by(const WeightsArgs& p, const Seq& x, int i) {
  return p.causal ? x.used - x.n + i + 1 : x.used;
}

// the first row that sees key k0 (k0 < used)
__device__ __forceinline__ int first_row(const WeightsArgs& p, const Seq& x, int k0) {
  return p.causal ? max(0, k0 - (x.used - x.n)) : 0;
}

// The work of a sequence, in groups of step_rows rows: its key tiles, those that
// every row sees (`full` groups each), and of the others the first one's groups;
// each next one has p.drop fewer (or up to one less than that where step_rows does
// not divide a tile: the last groups then hold no row).
struct Work {
  int tiles, seen, full, rest;
};

__device__ __forceinline__ Work work_of(const WeightsArgs& p, const Seq& x, int tile) {
  Work w{0, 0, 0, 0};
  if (x.n == 0 || x.used == 0) return w;
  w.tiles = (x.used + tile - 1) / tile;
  w.full = p.start + (x.n + p.step_rows - 1) / p.step_rows;
  const int older = x.used - x.n;  // keys that every row sees, and one more
  w.seen = !p.causal ? w.tiles : older < 0 ? 0 : min(older / tile + 1, w.tiles);
  if (w.seen < w.tiles) w.rest = p.start + (x.used - w.seen * tile + p.step_rows - 1) / p.step_rows;
  return w;
}

// groups of tile t, and of the tiles before it
__device__ __forceinline__ int groups_of(const Work& w, int drop, int t) {
  return t < w.seen ? w.full : w.rest - (t - w.seen) * drop;
}
__device__ __forceinline__ int groups_before(const Work& w, int drop, int t) {
  const int m = max(t - w.seen, 0);
  return min(t, w.seen) * w.full + m * w.rest - drop * (m * (m - 1) / 2);
}

// acc[i], i < N, summed over the 32 lanes of a half wave: lane l's is
// i = l & (N - 1). Lanes O apart exchange halves of what is left (each O its own
// function: as one loop, the registers' numbers became selects)
template <int O, int N>
__device__ __forceinline__ void sum_lanes(float (&acc)[N], int lane) {
  if constexpr (O >= N) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += __shfl_xor(acc[i], O, 64);
  } else {
    const bool up = lane & O;
#pragma unroll
    for (int i = 0; i < O; ++i) {
      const float send = up ? acc[i] : acc[i + O], own = up ? acc[i + O] : acc[i];
      acc[i] = own + __shfl_xor(send, O, 64);
    }
  }
  if constexpr (O > 1) sum_lanes<O / 2>(acc, lane);
}

// 16 bytes per lane (4 for dma4) to LDS from a uniform base and a lane's own
// offset in bytes, as lds_dma16
__device__ __forceinline__ void dma16(const void* base, uint32_t offset, const uint8_t* lds) {
  const uint32_t addr = (uint32_t)(uintptr_t)(lds_u8*)lds;
  asm volatile(
      "s_nop 1\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "{m0}"(addr), "v"(offset), "s"(base)
      : "memory");
}

// the key, within its wave's, whose sum a lane gets
__device__ __forceinline__ int lane_key(int lane) {
  return ((lane & 31) >> 4) * 32 + ((lane & 15) >> 2) * 8 + (lane >> 5) * 4 + (lane & 3);
}

// LDS of a workgroup: three stages of a step's rows, and their log-sum-exps.
// The waves' keys come in through the last two stages.
constexpr int kStage = kCols * 256;
constexpr int kLds = 3 * kStage + 3 * kCols * 4;

// The sums of one item: keys [k0, k0 + tile_keys(KT)) of head h over rows
// [lo, hi) of the sequence. Lane l of wave w returns that of key k0 +
// w * 32 KT + lane_key(l) (KT 1: of lanes with l & 16 nothing new).
template <int D, bool F8, int KT>
__device__ __forceinline__ float item_sums(const WeightsArgs& p, const Seq& x, int s, int h, int k0,
                                           int lo, int hi, uint8_t* lds) {
  constexpr int CH = D / 8;  // 16-byte chunks of a query row
  constexpr int C = D / 16;  // MFMAs of a dot product
  constexpr int LOADS = kCols * CH / 256;
  const int tid = opaque(threadIdx.x), lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int kw = k0 + wave * 32 * KT;
  const int steps = (hi - lo + p.step_rows - 1) / p.step_rows * p.blocks;
  const uint16_t* q = p.q + (int64_t)(x.q0 + lo) * p.q_ld + (int64_t)h * p.G * D;
  const float* lse = p.lse + (int64_t)h * p.G * p.lse_ld + x.q0 + lo;
  // Column c of a step: row c / heads of it, head c % heads of the block; past
  // the rows or heads there are, the last ones again, with weight 0.
  const int heads = min(p.G, kCols);
  // a row's chunks lie in LDS at c ^ swizzle, so that the 16 rows that a
  // quarter wave reads together lie in different banks
  auto swizzle = [](int r) { return D == 128 ? r & 15 : (r >> 1) & 7; };
  const int q_bytes = (int)p.q_ld * 2;
  auto place = [&](int c) { return min(c / heads, p.step_rows - 1) << 16 | c % heads; };
  int slot[LOADS];  // rows and heads of the columns this lane loads
#pragma unroll
  for (int j = 0; j < LOADS; ++j) slot[j] = place(j * (256 / CH) + tid / CH);
  const int chunk = (tid % CH ^ swizzle(tid / CH)) * 16;  // the same for all (their distance is whole 16s)
  const int lse_slot = place(wave * 16 + (lane & 15));
  auto load = [&](int step) {
    const int r0 = p.blocks == 1 ? step * p.step_rows : step / p.blocks;  // blocks > 1: a row a step
    const int g0 = p.blocks == 1 ? 0 : step % p.blocks * kCols;
    const int buffer = step % 3, last = hi - lo - 1;
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      int at = (slot[j] & 0xffff) * (2 * D) + chunk;
      if (p.blocks > 1) at = min((slot[j] & 0xffff) + g0, p.G - 1) * (2 * D) + chunk;
      // (an item's rows and their bytes are below 2^24, and together below 2^31)
      dma16(q, __umul24(min(r0 + (slot[j] >> 16), last), q_bytes) + at,
            lds + buffer * kStage + (j * 256 + wave * 64) * 16);
    }
    if (lane < 16)
      lds_dma4(lse + min((lse_slot & 0xffff) + g0, p.G - 1) * p.lse_ld + min(r0 + (lse_slot >> 16), last),
               lds + 3 * kStage + buffer * kCols * 4 + wave * 64);
  };
  __syncthreads();  // an earlier item's reads of the stages
  load(0);
  // The wave's keys; past the last one, the last again (their sums are
  // dropped). They come through LDS, whole rows a request: read from memory as
  // the fragments lie, 32 bytes of each of 32 rows, a row's lines came several
  // times (two contexts of 40,000 keys 97 us)
  v8bf kf[KT][C];
  {
    constexpr int RB = F8 ? D : 2 * D, RCH = RB / 16;  // bytes and chunks of a key's row
    constexpr int RPL = 64 / RCH;                      // rows of one request
    constexpr int ROUND = RB == 256 ? 32 : 32 * KT;    // keys at a time, in 8 KiB
    auto key_swizzle = [](int r) { return RB == 256 ? r & 15 : RB == 128 ? (r >> 1) & 7 : (r >> 2) & 3; };
    uint8_t* mine = lds + kStage + wave * 8192;
    const int* table = p.table + s * p.table_ld;
#pragma unroll
    for (int t0 = 0; t0 < KT; t0 += ROUND / 32) {
      int64_t row[ROUND / RPL];
#pragma unroll
      for (int j = 0; j < ROUND / RPL; ++j) {
        const int key = min(kw + t0 * 32 + j * RPL + lane / RCH, x.used - 1);
        row[j] = (int64_t)table[key / kPage] * kPage + key % kPage;
      }
#pragma unroll
      for (int j = 0; j < ROUND / RPL; ++j) {
        const int c = lane % RCH ^ key_swizzle(j * RPL + lane / RCH);
        lds_dma16(p.k + (row[j] * p.HK + h) * RB + c * 16, mine + j * 1024);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int t = 0; t < ROUND / 32; ++t) {
        const int r = t * 32 + col;
        if constexpr (F8) {
          const int key = min(kw + (t0 + t) * 32 + col, x.used - 1);
          const uint32_t b = p.scales[((int64_t)table[key / kPage] * p.HK + h) * 2];
          const float scale = __uint_as_float(max(b, 1u) << 23);
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const uint2 w = *reinterpret_cast<const uint2*>(mine + r * RB + (c ^ key_swizzle(r)) * 16 + half * 8);
            const uint4 f = make_uint4(
                pack2_bf16(__builtin_amdgcn_cvt_f32_fp8(w.x, 0) * scale, __builtin_amdgcn_cvt_f32_fp8(w.x, 1) * scale),
                pack2_bf16(__builtin_amdgcn_cvt_f32_fp8(w.x, 2) * scale, __builtin_amdgcn_cvt_f32_fp8(w.x, 3) * scale),
                pack2_bf16(__builtin_amdgcn_cvt_f32_fp8(w.y, 0) * scale, __builtin_amdgcn_cvt_f32_fp8(w.y, 1) * scale),
                pack2_bf16(__builtin_amdgcn_cvt_f32_fp8(w.y, 2) * scale, __builtin_amdgcn_cvt_f32_fp8(w.y, 3) * scale));
            kf[t0 + t][c] = __builtin_bit_cast(v8bf, f);
          }
        } else {
#pragma unroll
          for (int c = 0; c < C; ++c)
            kf[t0 + t][c] = *reinterpret_cast<const v8bf*>(mine + r * RB + ((2 * c + half) ^ key_swizzle(r)) * 16);
        }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
  }
  lds_barrier();  // every wave has its keys
  if (steps > 1) load(1);
  float acc[16 * KT];
#pragma unroll
  for (int i = 0; i < 16 * KT; ++i) acc[i] = 0.f;
  const int end = min(kw + 32 * KT, x.used);  // past the wave's last key
  // rows and heads of the lane's columns; a step's last columns may be none
  int at_col[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int c = t * 32 + col;
    at_col[t] = c / heads < p.step_rows ? place(c) : -1;
  }
  const int frag = col * D * 2 + (half ^ swizzle(col)) * 16;  // of chunk `half`; 2 c + half is at ^ 32 c
  // this step's rows have landed (the next one's may be on their way), and the
  // last step's are read
  auto arrive = [&](int step) {
    if (step + 1 < steps) {
      wait_vmcnt<LOADS + 1>();
    } else {
      wait_vmcnt<0>();
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (step + 2 < steps) load(step + 2);
  };
  auto first_of = [&](int step) { return p.blocks == 1 ? step * p.step_rows : step / p.blocks; };
  auto is_live = [&](int t, int step, int left) {
    const int g0 = p.blocks == 1 ? 0 : step % p.blocks * kCols;
    return (uint32_t)(at_col[t] >> 16) < (uint32_t)left && (at_col[t] & 0xffff) + g0 < p.G;
  };
  const float* all_lse = reinterpret_cast<const float*>(lds + 3 * kStage);
  // (rounded once, at the size of the log-sum-exp: 2^-24 of it of a weight)
  auto bias_of = [&](int t, int step, bool live) {
    const float v = all_lse[step % 3 * kCols + t * 32 + col] * -kLog2e;
    return live ? v : -__builtin_inff();
  };
  constexpr int AHEAD = 3;
  auto fragment = [&](int step, int t, int c) {
    return *reinterpret_cast<const v8bf*>(lds + step % 3 * kStage + t * 64 * D + (frag ^ c * 32));
  };
  // steps whose first row does not see all of the wave's keys: each score
  // against the keys that its column sees
  int step = 0;
  for (; step < steps; ++step) {
    const int r0 = first_of(step), left = hi - lo - r0;  // rows from the step's first on
    if (seen_by(p, x, lo + r0) >= end) break;
    arrive(step);
    if (kw >= seen_by(p, x, lo + r0 + min(left, p.step_rows) - 1)) continue;
#pragma unroll 1
    for (int t = 0; t < 2 && t * 32 < left * heads; ++t) {
      const bool live = is_live(t, step, left);
      const float bias = bias_of(t, step, live);
      const int last = (live ? seen_by(p, x, lo + r0 + (at_col[t] >> 16)) : 0) - kw - 4 * half;
      v16f sc[KT] = {};
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const v8bf qf = fragment(step, t, c);
#pragma unroll
        for (int u = 0; u < KT; ++u)
          sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u][c], qf, sc[u], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 16 * KT; ++i) {
        const int key = (i >> 4) * 32 + ((i & 15) >> 2) * 8 + (i & 3);
        const float w = __builtin_amdgcn_exp2f(fmaf(sc[i >> 4][i & 15], p.scale_log2, bias));
        acc[i] += key < last ? w : 0.f;
      }
    }
  }
  if (step < steps && kw < x.used) {
    // The rest: the products of 32 columns with the wave's keys, and behind each
    // of them a share of the exponentials of the 32 columns before. (The waves of
    // a SIMD run the same steps at about the same time, so the matrix core and
    // the vector unit overlap only within a wave.)
    struct Scores {
      v16f sc[KT];
      float bias;
    } s0, s1;
    auto add = [&](const Scores& y, int i0, int i1) {
#pragma unroll
      for (int i = i0; i < i1; ++i)
        acc[i] += __builtin_amdgcn_exp2f(fmaf(y.sc[i >> 4][i & 15], p.scale_log2, y.bias));
    };
    auto products = [&](int t, Scores& y, const Scores& old) {
      v8bf qf[AHEAD];
#pragma unroll
      for (int c = 0; c < AHEAD; ++c) qf[c] = fragment(step, t, c);
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int u = 0; u < KT; ++u)
          y.sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[u][c], qf[c % AHEAD],
                                                             c == 0 ? v16f{} : y.sc[u], 0, 0, 0);
        if (c + AHEAD < C) qf[c % AHEAD] = fragment(step, t, c + AHEAD);
        add(old, c * 16 * KT / C, (c + 1) * 16 * KT / C);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    s1.bias = -__builtin_inff();  // nothing is left of the steps before
#pragma unroll
    for (int u = 0; u < KT; ++u) s1.sc[u] = v16f{};
    for (; step < steps; ++step) {
      const int left = hi - lo - first_of(step);
      arrive(step);
      // (no branch between the two: the exponentials would move behind it)
      const float bias = bias_of(1, step, is_live(1, step, left));
      s0.bias = bias_of(0, step, is_live(0, step, left));
      products(0, s0, s1);
      s1.bias = bias;
      products(1, s1, s0);
    }
    add(s1, 0, 16 * KT);
  } else {
    for (; step < steps; ++step) arrive(step);
  }
  sum_lanes<16>(acc, lane);
  return acc[0];
}

// One workgroup per (key tile, sequence, head), heads fastest (a page's heads lie
// side by side, and neighbouring workgroups read them at about the same time).
// Two contexts of 40,000 keys, 8 heads of 128, weights there before: 45 us, 41 by
// itself; their 169 MB take 33 at the rate of a copy.
template <int D, bool F8, int KT>
__global__ __launch_bounds__(256, 2) void key_weights_direct_kernel(WeightsArgs p) {
  __shared__ __align__(16) uint8_t lds[kLds];
  const int id = blockIdx.x;
  const int h = id % p.HK, s = id / p.HK % p.seqs, k0 = id / p.HK / p.seqs * tile_keys(KT);
  const Seq x = seq_of(p, s);
  const int lane = threadIdx.x & 63;
  const int j = k0 + (threadIdx.x >> 6) * 32 * KT + lane_key(lane & (KT == 1 ? 47 : 63));
  // (read ahead: behind the sums it would be one more way to memory)
  const float prior = p.base && j < p.cols ? p.base[s * p.base_s + h * p.base_h + j] : 0.f;
  float sum = 0.f;
  const int lo = first_row(p, x, k0);
  if (k0 < x.used && lo < x.n) {
    const float v = item_sums<D, F8, KT>(p, x, s, h, k0, lo, x.n, lds);
    sum = j < x.used ? v : 0.f;
  }
  if (j >= p.cols || (KT == 1 && (lane & 16))) return;
  p.out[s * p.out_s + h * p.out_h + j] = p.base ? sum + prior : sum;
}

// Groups of a head from each sequence on (bound[s], s <= seqs), by one wave
__device__ __forceinline__ void bounds(const WeightsArgs& p, int lane, int tile, int* bound) {
  int carry = 0;
  for (int s0 = 0; s0 < p.seqs; s0 += 64) {
    const int s = s0 + lane;
    int sum = 0;
    if (s < p.seqs) {
      const Work w = work_of(p, seq_of(p, s), tile);
      sum = groups_before(w, p.drop, w.tiles);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(sum, o, 64);
      if (lane >= o) sum += y;
    }
    if (s < p.seqs) bound[s + 1] = carry + sum;
    carry += __shfl(sum, 63, 64);
  }
  if (lane == 0) bound[0] = 0;
}

// Shares go in pairs, one for each of the two workgroups that run on a CU: of
// their waves the older issue first, so that the one which started first took
// 203 us for half of 8003 rows and the other 275. It gets the larger share (of
// 64ths 32: 286 us, an AI.IF pack 85; 36: 275 and 76; 40: 267 and 71; 44 on another
// card 4% more than 40).
struct Shares {
  int first, both;  // groups of the first of a pair, and of the two
};
__device__ __forceinline__ Shares shares_of(int total) {
  const int both = max(2 * kMinShare, (total + kShares / 2 - 1) / (kShares / 2));
  return {(int)((int64_t)both * kFirst / 64), both};
}

// Many rows: the groups of all heads' sequences' key tiles, in that order, in
// equal shares, one a workgroup (items of a tile and some of its rows, taken in
// turn: an AI.IF pack 110 us where the shares took 88). A share begins and ends
// anywhere; each tile's part of it goes to scratch memory, at the tile's number
// plus the workgroup's (both only rise along the order).
template <int D, bool F8>
__global__ __launch_bounds__(256, 2) void key_weights_share_kernel(WeightsArgs p) {
  constexpr int KT = 2, TILE = tile_keys(KT);
  __shared__ __align__(16) uint8_t lds[kLds];
  __shared__ int bound[kSeqs + 1];
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid < 64) bounds(p, lane, TILE, bound);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int s = tid; s <= p.seqs; s += 256) p.bound[s] = bound[s];
  auto uniform = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
  const int of_head = uniform(bound[p.seqs]);
  const int total = of_head * p.HK;
  const Shares share = shares_of(total);
  // workgroups i, i + 8, ... run on one XCD, half of them first on their CUs: it
  // takes neighbouring pairs, whose query rows are the same
  const int nth = blockIdx.x / 8, half = kShares / 16;
  const int pair = blockIdx.x % 8 * half + nth % half, w = 2 * pair + nth / half;
  int at = min(pair * share.both + nth / half * share.first, total);
  const int end = uniform(min(at + (nth / half ? share.both - share.first : share.first), total));
  if (at == end) return;
  int h = at / of_head, in = at % of_head, s;
  {
    int a = 0, b = p.seqs;  // bound[a] <= in < bound[b]
    while (b - a > 1) {
      const int m = (a + b) / 2;
      if (bound[m] <= in) a = m; else b = m;
    }
    s = uniform(a);
  }
  in -= uniform(bound[s]);
  Seq x = seq_of(p, s);
  Work work = work_of(p, x, TILE);
  int t = min(in / work.full, work.seen);
  while (in >= groups_before(work, p.drop, t + 1)) ++t;
  in -= groups_before(work, p.drop, t);
  for (;;) {
    // (the same in every lane, found by way of LDS)
    h = uniform(h), s = uniform(s), t = uniform(t), in = uniform(in), at = uniform(at);
    x = seq_of(p, s);
    work = work_of(p, x, TILE);
    const int groups = groups_of(work, p.drop, t);
    const int here = min(groups - in, end - at);
    const int k0 = t * TILE, first = first_row(p, x, k0);
    const int lo = first + max(in - p.start, 0) * p.step_rows;
    const int hi = min(first + max(in + here - p.start, 0) * p.step_rows, x.n);
    float v = 0.f;
    for (int l = lo; l < hi; l += p.row_limit)
      v += item_sums<D, F8, KT>(p, x, s, h, k0, l, min(l + p.row_limit, hi), lds);
    const int64_t part = ((int64_t)h * p.seqs + s) * p.tiles + t + w;
    p.part[part * TILE + (tid >> 6) * 32 * KT + lane_key(lane)] = v;
    at += here;
    if (at == end) return;
    in = 0;
    if (++t < work.tiles) continue;
    t = 0;
    do {
      if (++s == p.seqs) s = 0, ++h;
      x = seq_of(p, s);
      work = work_of(p, x, TILE);
    } while (work.tiles == 0);
  }
}

__global__ __launch_bounds__(256) void key_weights_join_kernel(WeightsArgs p) {
  constexpr int TILE = tile_keys(2);
  const int h = blockIdx.y % p.HK, s = blockIdx.y / p.HK;
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= p.cols) return;
  const Seq x = seq_of(p, s);
  const Work work = work_of(p, x, TILE);
  const int t = j / TILE;
  const float prior = p.base ? p.base[s * p.base_s + h * p.base_h + j] : 0.f;
  float sum = 0.f;
  if (j < x.used && t < work.tiles) {
    const int of_head = p.bound[p.seqs];
    const Shares share = shares_of(of_head * p.HK);
    auto share_at = [&](int group) {
      const int pair = group / share.both;
      return 2 * pair + (group - pair * share.both >= share.first);
    };
    const int at = of_head * h + p.bound[s] + groups_before(work, p.drop, t);
    const int last = share_at(at + groups_of(work, p.drop, t) - 1);
    const float* part = p.part + (((int64_t)h * p.seqs + s) * p.tiles + t) * TILE + j % TILE;
    for (int w = share_at(at); w <= last; ++w) sum += part[(int64_t)w * TILE];
  }
  p.out[s * p.out_s + h * p.out_h + j] = p.base ? sum + prior : sum;
}

int64_t tiles_of(int64_t keys, int KT) { return (keys + tile_keys(KT) - 1) / tile_keys(KT); }

// Whether the rows go in shares. Up to two steps a tile's workgroup has no more
// to do than read its keys. Up to 12 and where its tiles are few, the shares' start
// (bounds, a search, the second launch) costs more than they even out, in us by
// tiles and shares: 8 contexts of up to 1600 keys (832 tiles), 64 rows of 4 heads a
// group 14.8 and 22.2, 128 rows 23.6 and 29.8, 200 rows 31.6 and 38.5 (500: 61 and
// 56); 60 of up to 900 (3840), 64 rows 47.6 and 51.2. Many tiles: 24 contexts of
// up to 8000 (12096), 64 rows 147 and 132, 128 rows 236 and 201.
bool shared_rows(int64_t seqs, int64_t max_q, int64_t max_used, int64_t HK, int64_t G) {
  return max_q * G > 2 * kCols && (max_q * G > 12 * kCols || tiles_of(max_used, 1) * seqs * HK > 4000);
}

// Scratch memory of a pair of launches over shares: the sequences' bounds, then
// the parts of (tile, workgroup)
constexpr int kBoundBytes = (kSeqs + 64) * 4;
int64_t part_bytes(int64_t seqs, int64_t max_used, int64_t HK) {
  return kBoundBytes + (seqs * HK * tiles_of(max_used, 2) + kShares) * tile_keys(2) * 4;
}

// Sequences of one pair of launches: within kScratch of scratch memory, and
// groups that are counted in 31 bits
constexpr int64_t kScratch = 128 << 20;
int64_t batch_of(int64_t seqs, int64_t max_q, int64_t max_used, int64_t HQ, int64_t HK) {
  const int64_t G = HQ / HK, rows = std::max<int64_t>(1, kCols / G);
  const int64_t groups = std::max<int64_t>(1, ((max_q + rows - 1) / rows + kStart) * tiles_of(max_used, 2) * HK);
  int64_t n = std::min<int64_t>({seqs, kSeqs, (1LL << 30) / groups});
  const int64_t fixed = part_bytes(0, max_used, HK), each = part_bytes(1, max_used, HK) - fixed;
  n = std::min({n, (kScratch - fixed) / std::max<int64_t>(each, 1), 65535 / HK});
  return std::max<int64_t>(n, 1);
}

}  // namespace
}  // namespace qx

using namespace qx;

extern "C" {

int64_t qx_key_weights_workspace(int64_t seqs, int64_t max_q, int64_t max_used, int64_t HQ,
                                 int64_t HK) {
  QX_CHECK(seqs >= 0 && max_q >= 0 && max_used >= 0 && HQ > 0 && HK > 0 && HQ % HK == 0,
           "key_weights_workspace: sizes");
  if (!shared_rows(seqs, max_q, max_used, HK, HQ / HK)) return 0;
  return part_bytes(batch_of(seqs, max_q, max_used, HQ, HK), max_used, HK);
}

int qx_key_weights(const void* q, int64_t q_ld, const float* lse, int64_t lse_ld,
                   const void* k_pool, const void* scales, const int* cu_q, const int* used,
                   const int* table, int64_t table_ld, int64_t seqs, int64_t rows, int64_t max_q,
                   int64_t max_used, int64_t HQ, int64_t HK, int64_t D, int64_t page, float scale,
                   int causal, const float* base, int64_t base_seq, int64_t base_head, float* out,
                   int64_t out_seq, int64_t out_head, int64_t cols, void* workspace,
                   int64_t workspace_bytes, hipStream_t stream) {
  QX_CHECK(D == 64 || D == 128, "key_weights: head_dim %lld (64 or 128)", (long long)D);
  QX_CHECK(HQ > 0 && HK > 0 && HQ % HK == 0 && HQ <= 4096, "key_weights: heads %lld/%lld",
           (long long)HQ, (long long)HK);
  QX_CHECK(page == kPage, "key_weights: page of %lld tokens (16)", (long long)page);
  QX_CHECK(seqs >= 0 && rows >= 0 && rows < (1LL << 31) && max_q >= 0 && max_used >= 0 &&
               max_used <= kMaxKeys && max_used <= cols && cols < (1LL << 30),
           "key_weights: %lld rows, up to %lld keys of %lld columns (at most %d)", (long long)rows,
           (long long)max_used, (long long)cols, kMaxKeys);
  QX_CHECK(max_q < (1LL << 28) && max_q * (HQ / HK) < (1LL << 31), "key_weights: a sequence of %lld rows",
           (long long)max_q);
  QX_CHECK(q_ld >= 0 && q_ld < (1LL << 19), "key_weights: rows %lld elements apart (below 2^19)",
           (long long)q_ld);
  QX_CHECK(q_ld % 8 == 0 && (((uintptr_t)q | (uintptr_t)k_pool) & 15) == 0 && lse_ld >= rows,
           "key_weights: strides or alignment");
  QX_CHECK(scale * kLog2e - scale * kLog2e == 0.f, "key_weights: scale %g", (double)scale);
  if (seqs == 0 || cols == 0) return QX_OK;
  QX_CHECK(cu_q && used && out && (rows == 0 || max_used == 0 || (q && lse && k_pool && table)),
           "key_weights: null pointer");
  const int64_t need = qx_key_weights_workspace(seqs, max_q, max_used, HQ, HK);
  QX_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
           "key_weights: a workspace of %lld bytes, %lld given", (long long)need,
           (long long)workspace_bytes);
  const int64_t G = HQ / HK;
  const bool shares = shared_rows(seqs, max_q, max_used, HK, G);
  // few rows: smaller tiles, so that more workgroups read the keys (8 sequences
  // of 700 keys 13.3 us, with the larger ones 22; two contexts of 40,000 41.8 and
  // 41.2)
  const int KT = shares ? 2 : 1;
  const int64_t tiles = tiles_of(shares ? max_used : cols, KT);
  const int64_t step_rows = G > kCols ? 1 : kCols / G;
  const int64_t batch = shares ? batch_of(seqs, max_q, max_used, HQ, HK)
                               : std::min<int64_t>({seqs, kSeqs, ((1LL << 24) - 1) / (tiles * HK)});
  QX_CHECK(batch > 0, "key_weights: %lld columns of %lld heads exceed one launch", (long long)cols,
           (long long)HK);
  QX_CHECK(!shares || ((max_q + step_rows - 1) / step_rows + kStart) * tiles * HK < (1LL << 30),
           "key_weights: %lld rows of %lld heads over %lld keys exceed one launch", (long long)max_q,
           (long long)HQ, (long long)max_used);
  for (int64_t s0 = 0; s0 < seqs; s0 += batch) {
    const int64_t n = std::min(seqs - s0, batch);
    WeightsArgs a{(const uint16_t*)q, q_ld, lse, lse_ld, (const uint8_t*)k_pool,
                  (const uint8_t*)scales, cu_q + s0, used + s0, table + s0 * table_ld, table_ld,
                  base ? base + s0 * base_seq : nullptr, base_seq, base_head, out + s0 * out_seq,
                  out_seq, out_head, (float*)((char*)workspace + kBoundBytes), (int*)workspace, (int)n,
                  (int)HK, (int)G, (int)rows, (int)max_q, rows ? (int)max_used : 0, (int)cols,
                  (int)tiles, (int)step_rows, (int)((G + kCols - 1) / kCols),
                  kStart, (int)(tile_keys(KT) / step_rows),
                  (int)((1LL << 31) / std::max<int64_t>(2 * q_ld, 1 << 16) / step_rows * step_rows),
                  scale * kLog2e, causal};
#define QX_KEYS(K, grid, ...)                                                                    \
  if (scales) {                                                                                  \
    if (D == 128) hipLaunchKernelGGL((K<128, true __VA_ARGS__>), grid, dim3(256), 0, stream, a); \
    else hipLaunchKernelGGL((K<64, true __VA_ARGS__>), grid, dim3(256), 0, stream, a);           \
  } else {                                                                                       \
    if (D == 128) hipLaunchKernelGGL((K<128, false __VA_ARGS__>), grid, dim3(256), 0, stream, a); \
    else hipLaunchKernelGGL((K<64, false __VA_ARGS__>), grid, dim3(256), 0, stream, a);          \
  }
    if (!shares) {
      const dim3 grid((unsigned)(tiles * n * HK));
      QX_KEYS(key_weights_direct_kernel, grid, , 1)
    } else {
      QX_KEYS(key_weights_share_kernel, dim3(kShares))
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return (int)e;
      hipLaunchKernelGGL(key_weights_join_kernel, dim3((unsigned)((cols + 255) / 256), (unsigned)(n * HK)),
                         dim3(256), 0, stream, a);
    }
#undef QX_KEYS
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return QX_OK;
}

}  // extern "C"
