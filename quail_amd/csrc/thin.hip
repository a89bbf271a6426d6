// Thinning of kept keys: of each (layer, sequence, KV head) the rows of most
// weight stay, in place.
//
// With u = used rows and k = min(u, keep), the first `sinks` rows, the last
// `recent` and the heaviest of the others stay, k in all (ties: the lowest row;
// a NaN is heavier than every number). Kept rows below k stay where they are;
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
};

// A float's rank as an unsigned number; -0 ranks as 0, NaN above all
__device__ __forceinline__ uint32_t rank_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.0f);
  if (f != f) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int wave_sum_before(int v, int lane, int* total) {
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  *total = __shfl(x, 63, 64);
  return x - v;
}

__device__ __forceinline__ int lanes_before(uint64_t mask) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32),
                                   __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// One (layer, sequence, head) per workgroup, its weights' ranks in registers,
// E a thread (row e * NT + thread). The border, the rank of the last row kept, is
// found 11, 11 and 10 bits at a time from histograms in LDS; rows are then
// numbered by counting ballots, equal ranks, dropped slots and movers alike.
// Bound by latency: a few passes over registers with barriers between, 4 bytes
// a row from memory.
template <int NT, int E>
__global__ __launch_bounds__(NT) void thin_select_kernel(ThinArgs p) {
  constexpr int W = NT / 64, CELLS = E * W, BINS = 2048, PER = BINS / NT;
  __shared__ int hist[BINS];
  __shared__ int cell[CELLS + 1];
  __shared__ int sums[W];
  __shared__ int found[3];  // bin, rows above it, rows in it
  __shared__ uint16_t movers[NT * E / 2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const int h = (int)(row % p.HK);
  const int64_t ls = row / p.HK;
  const int s = (int)(ls % p.seqs);
  const float* w = p.w + ls / p.seqs * p.w_layer + s * p.w_seq + h * p.w_head;
  int* kept = p.kept + row * p.slots;
  float* out = p.out + row * p.cols;
  const int used = min(max(p.used[s], 0), p.bound);
  if (used <= p.keep) {
    for (int i = tid; i < p.cols; i += NT) out[i] = i < used ? w[i] : 0.f;
    for (int i = tid; i < p.slots; i += NT) kept[i] = i < used ? i : -1;
    return;
  }
  const int k = p.keep, late = used - p.recent;
  uint32_t rank[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * NT + tid;
    rank[e] = i >= p.sinks && i < late ? rank_of(w[i]) : 0;
  }
  int want = k - p.sinks - p.recent;  // of the rows [sinks, late), which are more
  uint32_t border = 0;
  int equal = 0;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    for (int i = tid; i < BINS; i += NT) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = e * NT + tid;
      const bool in = i >= p.sinks && i < late &&
                      (pass == 0 || (rank[e] >> (shift + bits)) == (border >> (shift + bits)));
      if (!in) continue;
      const int bin = (rank[e] >> shift) & ((1 << bits) - 1);
      // a wave whose rows are all of one bin counts them at once (weights of
      // keys that never had any are all 0)
      const int first = __builtin_amdgcn_readfirstlane(bin);
      const uint64_t active = __ballot(1);
      if (__ballot(bin == first) == active) {
        if (lanes_before(active) == 0) atomicAdd(&hist[bin], (int)__popcll(active));
      } else {
        atomicAdd(&hist[bin], 1);
      }
    }
    __syncthreads();
    // bins from the top, PER a thread
    int mine = 0;
#pragma unroll
    for (int b = 0; b < PER; ++b) mine += hist[BINS - 1 - (tid * PER + b)];
    int total;
    int before = wave_sum_before(mine, lane, &total);
    if (lane == 0) sums[wave] = total;
    __syncthreads();
    for (int v = 0; v < wave; ++v) before += sums[v];
    if (before < want && want <= before + mine) {
#pragma unroll
      for (int b = 0; b < PER; ++b) {
        const int bin = BINS - 1 - (tid * PER + b), n = hist[bin];
        if (before < want && want <= before + n) {
          found[0] = bin;
          found[1] = before;
          found[2] = n;
        }
        before += n;
      }
    }
    __syncthreads();
    if (want > 0) {
      border |= (uint32_t)found[0] << shift;
      want -= found[1];
      equal = found[2];
    }
  }
  const bool none = k == p.sinks + p.recent;  // no other row stays
  // numbers a flag's rows: cell[c] = rows before wave cell c
  auto number = [&](auto flag) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint64_t m = __ballot(flag(e));
      if (lane == 0) cell[e * W + wave] = __popcll(m);
    }
    __syncthreads();
    if (wave == 0) {
      int carry = 0;
      for (int c = 0; c < CELLS; c += 64) {
        const int v = c + lane < CELLS ? cell[c + lane] : 0;
        int total;
        const int before = wave_sum_before(v, lane, &total);
        if (c + lane < CELLS) cell[c + lane] = carry + before;
        carry += total;
      }
      if (lane == 0) cell[CELLS] = carry;
    }
    __syncthreads();
  };
  // bit e: row e * NT + tid stays
  uint64_t stays = 0;
  const bool all_equal = want == equal;
  if (!none && !all_equal)
    number([&](int e) {
      const int i = e * NT + tid;
      return i >= p.sinks && i < late && rank[e] == border;
    });
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * NT + tid;
    const bool middle = i >= p.sinks && i < late;
    bool stay = i < used && !middle;
    if (!none) {
      bool tie = middle && rank[e] == border;
      if (!all_equal) {
        const uint64_t m = __ballot(tie);
        tie = tie && cell[e * W + wave] + lanes_before(m) < want;
      }
      stay = stay || tie || (middle && rank[e] > border);
    }
    stays |= (uint64_t)stay << e;
  }
  __syncthreads();
  // dropped slots come before all movers
  auto flag = [&](int e) {
    const int i = e * NT + tid;
    const bool stay = stays >> e & 1;
    return i < k ? !stay : stay;
  };
  number(flag);
  const int holes = cell[CELLS] / 2;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * NT + tid;
    const bool f = flag(e);
    const uint64_t m = __ballot(f);
    if (f && i >= k) movers[cell[e * W + wave] + lanes_before(m) - holes] = (uint16_t)i;
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = e * NT + tid;
    const bool f = flag(e);
    const uint64_t m = __ballot(f);
    if (i < k) {
      const int src = f ? movers[cell[e * W + wave] + lanes_before(m)] : i;
      kept[i] = src;
      out[i] = w[src];
    }
  }
  for (int i = k + tid; i < p.cols; i += NT) out[i] = 0.f;
}

// 64 slots of a (layer, sequence, head) per wave: those whose row moves are
// listed in LDS, then a row of D values goes by D * 2 / 16 lanes, 16 bytes each,
// K and V of kBatch rows a lane in flight. Bound by HBM, in pieces of a head's
// row.
template <int D>
__global__ __launch_bounds__(256) void thin_move_kernel(ThinArgs p, int64_t waves, int parts) {
  constexpr int LPR = D / 8, RPP = 64 / LPR, kBatch = 4;
  __shared__ int64_t list[4][64][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t wid = (int64_t)blockIdx.x * 4 + wave;
  int n = 0;
  int h = 0;
  int64_t layer = 0;
  if (wid < waves) {
    h = (int)(wid % p.HK);
    const int part = (int)(wid / p.HK % parts);
    const int64_t ls = wid / p.HK / parts;
    layer = ls / p.seqs;
    const int* table = p.table + ls % p.seqs * p.table_ld;
    const int slot = part * 64 + lane;
    const int src = slot < p.slots ? p.kept[(ls * p.HK + h) * p.slots + slot] : -1;
    const bool moves = src >= 0 && src != slot;
    const uint64_t mask = __ballot(moves);
    n = __popcll(mask);
    if (moves) {
      int64_t* to = list[wave][lanes_before(mask)];
      to[0] = (int64_t)table[slot / kPage] * kPage + slot % kPage;
      to[1] = (int64_t)table[src / kPage] * kPage + src % kPage;
    }
  }
  __syncthreads();
  if (n == 0) return;
  uint8_t* k_pool = p.pools + 2 * layer * p.pool_stride + (int64_t)h * D * 2;
  uint8_t* v_pool = k_pool + p.pool_stride;
  const int64_t row_bytes = (int64_t)p.HK * D * 2;
  const int at = lane % LPR * 16;
  for (int m0 = lane / LPR; m0 < n; m0 += RPP * kBatch) {
    uint4 kv[kBatch][2];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = min(m0 + b * RPP, n - 1);  // a row again: no branch between the loads
      const int64_t from = list[wave][m][1] * row_bytes + at;
      kv[b][0] = *reinterpret_cast<const uint4*>(k_pool + from);
      kv[b][1] = *reinterpret_cast<const uint4*>(v_pool + from);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = m0 + b * RPP;
      if (m >= n) continue;
      const int64_t to = list[wave][m][0] * row_bytes + at;
      *reinterpret_cast<uint4*>(k_pool + to) = kv[b][0];
      *reinterpret_cast<uint4*>(v_pool + to) = kv[b][1];
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
__device__ __forceinline__ uint4 shifted16(uint4 c, int shift) {
  if (shift == 0) return c;
  const uint2 a = shifted8(make_uint2(c.x, c.y), shift), b = shifted8(make_uint2(c.z, c.w), shift);
  return make_uint4(a.x, a.y, b.x, b.y);
}

// The same over 8-bit pages. A page that a row moves into gets the largest
// scale of those its rows come with (its own among them, where a row stays);
// the codes of the others are shifted down to it, those of rows that stay too.
// `keep` is whole pages, so no page is both read for a move and written.
template <int D>
__global__ __launch_bounds__(256) void thin_move8_kernel(ThinArgs p, int64_t waves, int parts) {
  constexpr int LPR = D / 16, RPP = 64 / LPR, kBatch = 4;
  __shared__ int64_t list[4][64][2];
  __shared__ int shifts[4][64];  // K's and V's, 16 bits each
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t wid = (int64_t)blockIdx.x * 4 + wave;
  int n = 0;
  int h = 0;
  int64_t layer = 0;
  if (wid < waves) {
    h = (int)(wid % p.HK);
    const int part = (int)(wid / p.HK % parts);
    const int64_t ls = wid / p.HK / parts;
    layer = ls / p.seqs;
    const int* table = p.table + ls % p.seqs * p.table_ld;
    const int slot = part * 64 + lane;
    const int src = slot < p.slots ? p.kept[(ls * p.HK + h) * p.slots + slot] : -1;
    const bool moves = src >= 0 && src != slot;
    const uint64_t moving = __ballot(moves);
    if (moving) {
      uint8_t* scales = p.scales + layer * p.scale_stride;
      const bool page_moves = (moving >> (lane & 48) & 0xffff) != 0;
      int64_t to = 0, from = 0;
      int bk = 0, bv = 0;
      if (page_moves) {  // then all 16 of its slots hold rows
        to = table[slot / kPage];
        from = table[src / kPage];
        const uint8_t* b = scales + (from * p.HK + h) * 2;
        bk = b[0];
        bv = b[1];
      }
      int top_k = bk, top_v = bv;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
        top_k = max(top_k, __shfl_xor(top_k, o, 64));
        top_v = max(top_v, __shfl_xor(top_v, o, 64));
      }
      const bool write = page_moves && (moves || bk != top_k || bv != top_v);
      const uint64_t mask = __ballot(write);
      n = __popcll(mask);
      if (write) {
        const int m = lanes_before(mask);
        list[wave][m][0] = to * kPage + slot % kPage;
        list[wave][m][1] = from * kPage + src % kPage;
        shifts[wave][m] = ((top_k - bk) & 0xffff) | (top_v - bv) << 16;
      }
      if (page_moves && lane % kPage == 0) {
        uint8_t* b = scales + (to * p.HK + h) * 2;
        b[0] = (uint8_t)top_k;
        b[1] = (uint8_t)top_v;
      }
    }
  }
  __syncthreads();
  if (n == 0) return;
  uint8_t* k_pool = p.pools + 2 * layer * p.pool_stride + (int64_t)h * D;
  uint8_t* v_pool = k_pool + p.pool_stride;
  const int64_t row_bytes = (int64_t)p.HK * D;
  const int at = lane % LPR * 16;
  for (int m0 = lane / LPR; m0 < n; m0 += RPP * kBatch) {
    uint4 kv[kBatch][2];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = min(m0 + b * RPP, n - 1);  // a row again: no branch between the loads
      const int64_t from = list[wave][m][1] * row_bytes + at;
      kv[b][0] = *reinterpret_cast<const uint4*>(k_pool + from);
      kv[b][1] = *reinterpret_cast<const uint4*>(v_pool + from);
    }
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int m = m0 + b * RPP;
      if (m >= n) continue;
      const int64_t to = list[wave][m][0] * row_bytes + at;
      const int shift = shifts[wave][m];
      *reinterpret_cast<uint4*>(k_pool + to) = shifted16(kv[b][0], -(shift & 0xffff));
      *reinterpret_cast<uint4*>(v_pool + to) = shifted16(kv[b][1], -(shift >> 16));
    }
  }
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
  QX_CHECK(rows < (1LL << 21), "thin_rows: %lld heads exceed one launch", (long long)rows);
  ThinArgs a{(uint8_t*)pools, pool_stride, (uint8_t*)scales, scale_stride, weights, w_layer, w_seq,
             w_head, used, table, table_ld, (int)seqs, (int)HK, (int)max_used, (int)cols,
             (int)(keep < kMaxKeys ? keep : kMaxKeys), (int)slots, (int)sinks, (int)recent, kept, out};
#define QX_THIN(NT, E) \
  hipLaunchKernelGGL((thin_select_kernel<NT, E>), dim3((unsigned)rows), dim3(NT), 0, stream, a)
  if (max_used <= 1024) QX_THIN(256, 4);
  else if (max_used <= 2048) QX_THIN(256, 8);
  else if (max_used <= 4096) QX_THIN(1024, 4);
  else if (max_used <= 8192) QX_THIN(1024, 8);
  else if (max_used <= 16384) QX_THIN(1024, 16);
  else if (max_used <= 24576) QX_THIN(1024, 24);
  else QX_THIN(1024, 40);
#undef QX_THIN
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  if (max_used <= keep) return QX_OK;  // no row moves
  const int parts = (int)((slots + 63) / 64);
  const int64_t waves = rows * parts;
  QX_CHECK(waves <= (1LL << 26) - 4, "thin_rows: %lld rows of %lld heads exceed one launch",
           (long long)slots, (long long)rows);
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

}  // extern "C"
