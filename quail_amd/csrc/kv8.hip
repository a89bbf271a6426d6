// The 8-bit KV arena's writes, and copies of whole pages of any arena.
//
// An 8-bit pool holds e4m3 codes, (pages * 16, HK, D) bytes, K and V apart,
// and one power-of-two scale per (page, KV head), an E8M0 byte b that stands
// for 2^(b - 127), at scales[(page * HK + head) * 2 + (0 for K, 1 for V)].
#include <algorithm>
#include <new>
#include <vector>

#include "qx_common.h"
#include "qx_status.h"

namespace qx {
namespace {

constexpr int kPage = 16;  // tokens per arena page
// The last scale (2^120, for values past 448 * 2^119) holds codes up to 240
// alone: 256 would stand for 2^128, which bf16 and fp32 do not have, and a
// reader's weight of 0 times infinity is NaN. 240 for a value up to 256 is off
// by at most 2^-4 of it, as a code's rounding is.
constexpr int kLastScale = 247;
constexpr float kLargest = 240.f * 0x1p120f;

// The E8M0 byte of the least power of two s with amax <= 448 s, at least 1:
// with amax = 1.m * 2^e that is 2^(e - 8), and twice that where 1.m > 1.75.
// Adding the distance from the fraction of 1.75 to the next power of two
// carries into the exponent exactly where the fraction is past it. (An infinity:
// 247, as the largest float.)
__device__ __forceinline__ int scale_byte(float amax) {
  return max((int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 8, 1);
}

// v of lane ^ 4: within a row of 16 lanes, the banks of four 0 and 2 take the
// next bank's, 1 and 3 the one's before
__device__ __forceinline__ float xor4(float v) {
  const int x = __float_as_int(v);
  const int a = __builtin_amdgcn_update_dpp(x, x, 0x104, 0xf, 0x5, false);  // row_shl:4
  return __int_as_float(__builtin_amdgcn_update_dpp(a, x, 0x114, 0xf, 0xa, false));  // row_shr:4
}

// group_sum<width>'s sums in its order (width 8 or 4), on vector operands
// instead of LDS permutes
template <int width>
__device__ __forceinline__ float row_sum(float v) {
  if (width == 8) v += xor4(v);
  v += dpp_f32<0x4e>(v);  // lane ^ 2
  return v + dpp_f32<0xb1>(v);  // lane ^ 1
}

// the maximum over the wave, likewise
__device__ __forceinline__ float wave_max(float v) {
  v = group_max<16>(v);
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return max_halves(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// e4m3 codes of 8 values times 2^shift
__device__ __forceinline__ uint2 codes8(const float* x, int shift) {
  float y[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) y[k] = __builtin_ldexpf(x[k], shift);
  return make_uint2(pack4_fp8(y[0], y[1], y[2], y[3]), pack4_fp8(y[4], y[5], y[6], y[7]));
}

__device__ __forceinline__ void bf16x8_to_f32(uint4 w, float* x) {
  x[0] = lo_bf16(w.x); x[1] = hi_bf16(w.x); x[2] = lo_bf16(w.y); x[3] = hi_bf16(w.y);
  x[4] = lo_bf16(w.z); x[5] = hi_bf16(w.z); x[6] = lo_bf16(w.w); x[7] = hi_bf16(w.w);
}

// 16 bytes that nobody reads again (past the caches: 4% of a pack's write)
__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const v4i*>(p)));
}

// One page of `heads` heads per wave. Item i of `items` is (destination page,
// source page, kept rows, first row, rows): the page's rows [0, keep) are
// the source page's, the next `count` are fresh rows row0, row0 + 1, ...; the
// rest of the page stays as it is. The scale is the fresh rows' own, or the
// larger of that and the source page's where rows are kept: the kept codes
// then move by a power of two, exactly unless they become subnormal.
// Slots of an item: HK of K, HK of V, then (QKV, with a q output) HQ of q;
// an item of page -1 has the last ones alone.
// QKV: rows are the qkv projection's; q and K go through their norm and RoPE
// (the sums and products of norm_part4 and norm_rope4, in their order) and K
// from fp32 to its code in one rounding. Otherwise k and v are rows as the
// pool takes them.
// Streams 2 * (2 HK + HQ) * D bytes a row in and (2 HK + 2 HQ) * D out. A
// lane holds 16 columns of a row (8 of each half where they are rotated, so
// that every load is 16 bytes wide), D / 16 lanes a row, and the wave a
// head's 16 rows in registers between their maximum and their codes; the
// next head's rows load meanwhile, and a row's cos and sin serve every head.
// Sums and maxima over lanes run on vector operands (through LDS permutes
// they took 8% of a pack's write). A pack of 15,654 rows (32 + 8 + 8 heads of
// 128, 353 MB) 71 us, 4.9 TB/s (a large copy on the same card: 4.8); one token
// each for 8 sequences 4.6 us.
struct WriteArgs {
  const uint16_t *x, *v;  // qkv rows, or K rows and V rows
  int64_t x_ld, v_ld;
  uint16_t* qo;
  int64_t qo_ld;
  uint8_t *kp, *vp, *scales;
  const int* items;
  const void* cs;
  const int64_t* pos;
  const uint16_t *qw, *kw;
  float eps;
  int64_t waves;
  int groups, heads, slots, HQ, HK;  // waves per item, slots per wave
};

template <int D, bool QKV, bool CS_F32>
__global__ __launch_bounds__(256) void kv8_write_kernel(WriteArgs p) {
  constexpr int LPR = D / 16;      // lanes per row, 16 columns each
  constexpr int RPP = 64 / LPR;    // rows per pass
  constexpr int PASSES = kPage / RPP;
  constexpr int HALF = D / 2;
  const int lane = threadIdx.x & 63;
  const int64_t wid = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wid >= p.waves) return;
  const int* item = p.items + wid / p.groups * 5;
  const int dst = item[0], src = item[1], keep = item[2], row0 = item[3], count = item[4];
  const int head0 = (int)(wid % p.groups) * p.heads;
  const int first = max(head0, dst < 0 ? 2 * p.HK : 0);  // rows of no page: their q alone
  const int last = min(head0 + p.heads, p.slots);
  if (first >= last) return;
  const int j = lane % LPR;
  const int64_t kv_row = (int64_t)p.HK * D;
  // this lane's rows of the page, clamped to fresh ones for the loads
  int64_t row[PASSES];
  bool fresh[PASSES];
#pragma unroll
  for (int t = 0; t < PASSES; ++t) {
    const int r = t * RPP + lane / LPR;
    fresh[t] = r >= keep && r < keep + count;
    row[t] = (int64_t)row0 + min(max(r - keep, 0), max(count - 1, 0));
  }
  uint4 cs[PASSES][CS_F32 ? 4 : 2];  // cos and sin of columns 8 j .. 8 j + 8, as they lie
  auto is_v = [&](int slot) { return slot >= p.HK && slot < 2 * p.HK; };
  if (QKV && count > 0) {
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      const int64_t at = p.pos[row[t]] * D + 8 * j;
      if constexpr (CS_F32) {
        const uint4* c = reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p.cs) + at);
        cs[t][0] = c[0];
        cs[t][1] = c[1];
        cs[t][2] = c[HALF / 4];
        cs[t][3] = c[HALF / 4 + 1];
      } else {
        const uint4* c = reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.cs) + at);
        cs[t][0] = c[0];
        cs[t][1] = c[HALF / 8];
      }
    }
  }
  auto load = [&](int slot, uint4 (&w)[PASSES][2]) {
    const bool v = is_v(slot), q = QKV && slot >= 2 * p.HK;
    const int head = q ? slot - 2 * p.HK : v ? slot - p.HK : slot;
    const uint16_t* x = QKV || !v ? p.x : p.v;
    const int64_t ld = QKV || !v ? p.x_ld : p.v_ld;
    const int64_t col = (int64_t)D * (!QKV || q ? head : v ? p.HQ + p.HK + head : p.HQ + head);
    const bool rotate = QKV && !v;
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      if (count == 0) continue;
      const uint16_t* at = x + row[t] * ld + col;
      w[t][0] = load_once(at + (rotate ? 8 * j : 16 * j));
      w[t][1] = load_once(at + (rotate ? HALF + 8 * j : 16 * j + 8));
    }
  };
  uint4 w[PASSES][2] = {}, next[PASSES][2] = {};
  load(first, w);
  for (int slot = first; slot < last; ++slot) {
    if (slot + 1 < last) load(slot + 1, next);
    const bool v = is_v(slot), q = QKV && slot >= 2 * p.HK;
    const bool rotate = QKV && !v;
    const int head = q ? slot - 2 * p.HK : v ? slot - p.HK : slot;
    const int side = v ? 1 : 0;
    int b_old = 0;
    if (!q && keep > 0) b_old = p.scales[((int64_t)src * p.HK + head) * 2 + side];
    float y[PASSES][16];
    float wa[2][4], wb[2][4];
    if (rotate) {
      const uint16_t* g = q ? p.qw : p.kw;
      const uint4 a = *reinterpret_cast<const uint4*>(g + 8 * j);
      const uint4 b = *reinterpret_cast<const uint4*>(g + HALF + 8 * j);
      bf16x4_to_f32(make_uint2(a.x, a.y), wa[0]);
      bf16x4_to_f32(make_uint2(a.z, a.w), wa[1]);
      bf16x4_to_f32(make_uint2(b.x, b.y), wb[0]);
      bf16x4_to_f32(make_uint2(b.z, b.w), wb[1]);
    }
    float amax = 0.f;
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      if (rotate) {
        float a[2][4], b[2][4], s[2];
        const uint4 lo = w[t][0], hi = w[t][1];
        bf16x4_to_f32(make_uint2(lo.x, lo.y), a[0]);
        bf16x4_to_f32(make_uint2(lo.z, lo.w), a[1]);
        bf16x4_to_f32(make_uint2(hi.x, hi.y), b[0]);
        bf16x4_to_f32(make_uint2(hi.z, hi.w), b[1]);
        // the qk-norm-rope pass's tree over 4-column groups: its last level
        // pairs the lane's own two
#pragma unroll
        for (int e = 0; e < 2; ++e) s[e] = row_sum<LPR>(norm_part4(a[e], b[e]));
        const float rstd = norm_rstd<D>(s[0] + s[1], p.eps);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float cosv[4], sinv[4], oa[4], ob[4];
          if constexpr (CS_F32) {
            const uint4 c = cs[t][e], n = cs[t][2 + e];
            cosv[0] = __uint_as_float(c.x); cosv[1] = __uint_as_float(c.y);
            cosv[2] = __uint_as_float(c.z); cosv[3] = __uint_as_float(c.w);
            sinv[0] = __uint_as_float(n.x); sinv[1] = __uint_as_float(n.y);
            sinv[2] = __uint_as_float(n.z); sinv[3] = __uint_as_float(n.w);
          } else {
            const uint4 c = cs[t][0], n = cs[t][1];
            bf16x4_to_f32(e ? make_uint2(c.z, c.w) : make_uint2(c.x, c.y), cosv);
            bf16x4_to_f32(e ? make_uint2(n.z, n.w) : make_uint2(n.x, n.y), sinv);
          }
          norm_rope4(a[e], b[e], wa[e], wb[e], cosv, sinv, rstd, oa, ob);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            y[t][4 * e + k] = oa[k];
            y[t][8 + 4 * e + k] = ob[k];
          }
        }
      } else {
        bf16x8_to_f32(w[t][0], y[t]);
        bf16x8_to_f32(w[t][1], y[t] + 8);
      }
      if (q) {
        if (fresh[t]) {
          uint16_t* out = p.qo + row[t] * p.qo_ld + head * D + 8 * j;
          *reinterpret_cast<uint4*>(out) =
              make_uint4(pack2_bf16(y[t][0], y[t][1]), pack2_bf16(y[t][2], y[t][3]),
                         pack2_bf16(y[t][4], y[t][5]), pack2_bf16(y[t][6], y[t][7]));
          *reinterpret_cast<uint4*>(out + HALF) =
              make_uint4(pack2_bf16(y[t][8], y[t][9]), pack2_bf16(y[t][10], y[t][11]),
                         pack2_bf16(y[t][12], y[t][13]), pack2_bf16(y[t][14], y[t][15]));
        }
      } else if (fresh[t]) {
#pragma unroll
        for (int k = 0; k < 16; ++k) amax = fmaxf(amax, fabsf(y[t][k]));
      }
    }
    if (!q) {
      amax = wave_max(amax);
      const int need = scale_byte(amax);
      if (need == kLastScale) {  // infinities (e4m3 has none) and what they share a page with; NaN stays
#pragma unroll
        for (int t = 0; t < PASSES; ++t)
#pragma unroll
          for (int k = 0; k < 16; ++k)
            y[t][k] = y[t][k] != y[t][k] ? y[t][k] : fminf(fmaxf(y[t][k], -kLargest), kLargest);
      }
      const int b = keep > 0 ? max(b_old, need) : need;
      const bool move = src != dst || b != b_old;  // the kept rows change
      uint8_t* pool = v ? p.vp : p.kp;
      const int c0 = rotate ? 8 * j : 16 * j, c1 = rotate ? HALF + 8 * j : 16 * j + 8;
#pragma unroll
      for (int t = 0; t < PASSES; ++t) {
        const int r = t * RPP + lane / LPR;
        uint8_t* out = pool + ((int64_t)dst * kPage + r) * kv_row + head * D;
        int shift = 127 - b;
        if (r < keep) {
          if (!move) continue;
          const uint8_t* in = pool + ((int64_t)src * kPage + r) * kv_row + head * D;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const uint2 old = *reinterpret_cast<const uint2*>(in + (e ? c1 : c0));
            y[t][8 * e + 0] = __builtin_amdgcn_cvt_f32_fp8(old.x, 0);
            y[t][8 * e + 1] = __builtin_amdgcn_cvt_f32_fp8(old.x, 1);
            y[t][8 * e + 2] = __builtin_amdgcn_cvt_f32_fp8(old.x, 2);
            y[t][8 * e + 3] = __builtin_amdgcn_cvt_f32_fp8(old.x, 3);
            y[t][8 * e + 4] = __builtin_amdgcn_cvt_f32_fp8(old.y, 0);
            y[t][8 * e + 5] = __builtin_amdgcn_cvt_f32_fp8(old.y, 1);
            y[t][8 * e + 6] = __builtin_amdgcn_cvt_f32_fp8(old.y, 2);
            y[t][8 * e + 7] = __builtin_amdgcn_cvt_f32_fp8(old.y, 3);
          }
          shift = b_old - b;
        } else if (!fresh[t]) {
          continue;
        }
        *reinterpret_cast<uint2*>(out + c0) = codes8(y[t], shift);
        *reinterpret_cast<uint2*>(out + c1) = codes8(y[t] + 8, shift);
      }
      if (lane == 0) p.scales[((int64_t)dst * p.HK + head) * 2 + side] = (uint8_t)b;
    }
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      w[t][0] = next[t][0];
      w[t][1] = next[t][1];
    }
  }
}

int kv8_write_launch(WriteArgs& a, bool qkv, int64_t n_items, int64_t HK, int64_t D, int cs_is_f32,
                     hipStream_t stream) {
  QX_CHECK(D == 64 || D == 128, "kv8_write: head_dim %lld (64 or 128)", (long long)D);
  QX_CHECK(HK > 0 && n_items >= 0, "kv8_write: heads %lld, items %lld", (long long)HK,
           (long long)n_items);
  if (n_items == 0) return QX_OK;
  // heads per wave: as many as leave 6144 waves (twice what the card holds of
  // these at once). The pack above, with q (48 slots) 1: 79.2 us, 2: 72.9, 4: 71.3;
  // its K and V alone (16 slots) 31.1, 28.5, 30.8
  for (a.heads = 4; a.heads > 1 && n_items * a.slots / a.heads < 6144;) a.heads /= 2;
  a.groups = (a.slots + a.heads - 1) / a.heads;
  a.waves = n_items * a.groups;
  QX_CHECK(a.waves <= (1LL << 26) - 4, "kv8_write: %lld items of %d heads exceed one launch",
           (long long)n_items, a.slots);  // 2^32 threads
  const dim3 grid((unsigned)((a.waves + 3) / 4)), block(256);
#define QX_KV8(DD, Q, F) hipLaunchKernelGGL((kv8_write_kernel<DD, Q, F>), grid, block, 0, stream, a)
  if (!qkv) {
    if (D == 128) QX_KV8(128, false, false); else QX_KV8(64, false, false);
  } else if (cs_is_f32) {
    if (D == 128) QX_KV8(128, true, true); else QX_KV8(64, true, true);
  } else {
    if (D == 128) QX_KV8(128, true, false); else QX_KV8(64, true, false);
  }
#undef QX_KV8
  QX_LAUNCH_STATUS();
}

// Pages src[i] -> dst[i] of every pool: the page ids travel in the kernel's
// arguments, so a copy needs no upload and nothing of the caller's stays in
// use after the call.
constexpr int kCopyIds = 440;
struct CopyIds {
  int src[kCopyIds], dst[kCopyIds];
};
struct CopyRegion {
  uint8_t* base;
  int64_t pool_stride, page_bytes;
  int pools;
};

// blockIdx.x: page of the list; blockIdx.y: pool (the codes' pools, then the
// scales'); blockIdx.z: part of the page. Bound by HBM: 1000 pages of 36
// layers (16 KiB of codes each for K and V, 2.36 GB read and written) 480 us,
// 4.9 TB/s, a large copy's rate; 37 pages (87 MB) 18 us.
__global__ __launch_bounds__(256) void copy_pages_kernel(CopyRegion big, CopyRegion small,
                                                         CopyIds ids) {
  const int pool = blockIdx.y;
  const bool tail = pool >= big.pools;
  if (tail && blockIdx.z) return;
  const CopyRegion r = tail ? small : big;
  uint8_t* at = r.base + (tail ? pool - big.pools : pool) * r.pool_stride;
  const uint8_t* s = at + ids.src[blockIdx.x] * r.page_bytes;
  uint8_t* d = at + ids.dst[blockIdx.x] * r.page_bytes;
  if (tail) {
    for (int64_t c = threadIdx.x; c < r.page_bytes / 2; c += 256)
      reinterpret_cast<uint16_t*>(d)[c] = reinterpret_cast<const uint16_t*>(s)[c];
    return;
  }
  const int64_t chunks = r.page_bytes / 16;
  for (int64_t c = blockIdx.z * 256 + threadIdx.x; c < chunks; c += 256 * gridDim.z)
    reinterpret_cast<uint4*>(d)[c] = reinterpret_cast<const uint4*>(s)[c];
}

bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace
}  // namespace qx

using namespace qx;

extern "C" {

int qx_qk_norm_rope_kv8(const void* qkv, int64_t qkv_ld, void* q_out, int64_t q_ld, void* k_pool,
                        void* v_pool, void* scales, const int* items, int64_t n_items,
                        const void* cos_sin, int cs_is_f32, const int64_t* positions,
                        const void* q_w, const void* k_w, int64_t HQ, int64_t HK, int64_t D,
                        float eps, hipStream_t stream) {
  QX_CHECK(qkv && k_pool && v_pool && scales && cos_sin && positions && q_w && k_w &&
               (items || n_items == 0),
           "qk_norm_rope_kv8: null pointer");
  QX_CHECK(HQ > 0, "qk_norm_rope_kv8: heads");
  QX_CHECK(qkv_ld % 8 == 0 && q_ld % 8 == 0 && aligned(qkv, 16) && aligned(q_out, 16) &&
               aligned(k_pool, 8) && aligned(v_pool, 8) && aligned(cos_sin, 16) &&
               aligned(q_w, 16) && aligned(k_w, 16),
           "qk_norm_rope_kv8: strides or alignment");
  WriteArgs a{(const uint16_t*)qkv, nullptr, qkv_ld, 0, (uint16_t*)q_out, q_ld,
              (uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)scales, items, cos_sin, positions,
              (const uint16_t*)q_w, (const uint16_t*)k_w, eps, 0, 0, 0,
              (int)(2 * HK + (q_out ? HQ : 0)), (int)HQ, (int)HK};
  return kv8_write_launch(a, true, n_items, HK, D, cs_is_f32, stream);
}

int qx_kv8_write(const void* k, int64_t k_ld, const void* v, int64_t v_ld, void* k_pool,
                 void* v_pool, void* scales, const int* items, int64_t n_items, int64_t HK,
                 int64_t D, hipStream_t stream) {
  QX_CHECK(k && v && k_pool && v_pool && scales && (items || n_items == 0),
           "kv8_write: null pointer");
  QX_CHECK(k_ld % 8 == 0 && v_ld % 8 == 0 && aligned(k, 16) && aligned(v, 16) &&
               aligned(k_pool, 8) && aligned(v_pool, 8),
           "kv8_write: strides or alignment");
  WriteArgs a{(const uint16_t*)k, (const uint16_t*)v, k_ld, v_ld, nullptr, 0,
              (uint8_t*)k_pool, (uint8_t*)v_pool, (uint8_t*)scales, items, nullptr, nullptr,
              nullptr, nullptr, 0.f, 0, 0, 0, (int)(2 * HK), 0, (int)HK};
  return kv8_write_launch(a, false, n_items, HK, D, 0, stream);
}

static int copy_pages(void* pools, int64_t n_pools, int64_t pool_stride, int64_t page_bytes,
                      void* scales, int64_t n_scale_pools, int64_t scale_stride,
                      int64_t scale_bytes, const int* src, const int* dst, int64_t count,
                      int64_t num_pages, hipStream_t stream) {
  QX_CHECK(pools && (scales || n_scale_pools == 0) && (count == 0 || (src && dst)),
           "copy_pages: null pointer");
  QX_CHECK(n_pools > 0 && n_scale_pools >= 0 && n_pools + n_scale_pools < 65536 && count >= 0 &&
               num_pages >= 0,
           "copy_pages: %lld + %lld pools, %lld pages", (long long)n_pools,
           (long long)n_scale_pools, (long long)count);
  QX_CHECK(page_bytes > 0 && page_bytes % 16 == 0 && pool_stride % 16 == 0 && aligned(pools, 16) &&
               (n_scale_pools == 0 || (scale_bytes > 0 && scale_bytes % 2 == 0 &&
                                       scale_stride % 2 == 0 && aligned(scales, 2))),
           "copy_pages: page sizes or alignment");
  std::vector<uint8_t> role(num_pages, 0);  // 1: a source, 2: a destination
  for (int64_t i = 0; i < count; ++i) {
    QX_CHECK(src[i] >= 0 && src[i] < num_pages && dst[i] >= 0 && dst[i] < num_pages,
             "copy_pages: page %d -> %d of %lld", src[i], dst[i], (long long)num_pages);
    QX_CHECK(!(role[src[i]] & 2), "copy_pages: page %d is a source and a destination", src[i]);
    QX_CHECK(!role[dst[i]], "copy_pages: page %d is a destination twice, or also a source",
             dst[i]);
    if (src[i] == dst[i]) QX_CHECK(false, "copy_pages: page %d onto itself", src[i]);
    role[src[i]] = 1;
    role[dst[i]] = 2;
  }
  const CopyRegion big{(uint8_t*)pools, pool_stride, page_bytes, (int)n_pools};
  const CopyRegion small{(uint8_t*)scales, scale_stride, scale_bytes, (int)n_scale_pools};
  for (int64_t first = 0; first < count; first += kCopyIds) {
    CopyIds ids;
    const int n = (int)std::min<int64_t>(kCopyIds, count - first);
    for (int i = 0; i < n; ++i) {
      ids.src[i] = src[first + i];
      ids.dst[i] = dst[first + i];
    }
    const int64_t parts = std::min<int64_t>((page_bytes / 16 + 1023) / 1024, 64);
    hipLaunchKernelGGL(copy_pages_kernel,
                       dim3((unsigned)n, (unsigned)(n_pools + n_scale_pools), (unsigned)parts),
                       dim3(256), 0, stream, big, small, ids);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  return QX_OK;
}

int qx_copy_pages(void* pools, int64_t n_pools, int64_t pool_stride, int64_t page_bytes,
                  void* scales, int64_t n_scale_pools, int64_t scale_stride, int64_t scale_bytes,
                  const int* src, const int* dst, int64_t count, int64_t num_pages,
                  hipStream_t stream) {
  try {
    return copy_pages(pools, n_pools, pool_stride, page_bytes, scales, n_scale_pools,
                      scale_stride, scale_bytes, src, dst, count, num_pages, stream);
  } catch (const std::bad_alloc&) {
    qx::set_error("copy_pages: out of host memory");
    return QX_EINVAL;
  }
}

}  // extern "C"
