// Paged varlen GQA attention over an arena that keeps K and V in 8 bits.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j
//   k_j = kc_j * 2^(bk - 127),  v_j = vc_j * 2^(bv - 127)
//
// with e4m3 codes kc, vc and one E8M0 byte for K and one for V per (page,
// KV head) at scales[(page * HK + head) * 2 + (0, 1)]. Sequences, block
// table, causal alignment and GQA are those of paged_attention_kernel
// (attention.hip). Codes are exact in bf16, so both products run on the bf16
// matrix cores over the codes themselves: K's scale multiplies a page's 16
// scores and V's its 16 probabilities, both in fp32 (a power of two each).
// P is rounded to bf16 in query tiles (at most 2^-8 of a weight, what the
// bf16 output rounds by); few rows, whose matrix cores wait for memory, take
// what that rounding left as a second product (2^-16; rows then are off by
// 0.0015 to 0.0017 of their size where one product gave 0.0019 to 0.0024;
// 0.5 to 3% of a call's time). Scores, maxima, sums and outputs stay in fp32.
// (P in fp16 with V's scales in the softmax's exponent keeps 11 bits, but
// loses the weights of pages whose scale is far below another's; 3% slower on
// long documents.)
#include <algorithm>
#include <new>
#include <type_traits>
#include <unordered_map>
#include <utility>
#include <vector>

#include "q_norm.h"
#include "qx_common.h"
#include "qx_status.h"

namespace qx {
namespace {

constexpr int kPage = 16;  // tokens per arena page
constexpr int kMaxKeys = 2560 * kPage;  // per sequence, as the 16-bit call takes
constexpr int kMaxChunk = 2048;         // keys per split
typedef __attribute__((address_space(3))) v2i lds_v2i;

struct Attn8Args {
  const uint16_t* q;
  int64_t q_ld;
  const int64_t* q_index;
  const uint8_t *kp, *vp;
  const uint16_t* scales;  // (pages, HK) pairs of bytes
  const int *cu_q, *used, *table;
  int64_t table_ld;
  int max_used, HQ, HK, causal;
  float scale_log2;
  uint16_t* out16;
  uint8_t* out8;
  int64_t o_ld;
  float* oscales;
  int64_t os_ld;
  float* lse;
  int64_t lse_ld;
  // keys per split (0: whole sequences), the most splits of a sequence, the
  // query rows of a tile (0: few rows), and the splits' partial results: rows
  // of HQ heads. Without slots split i of query row r has row i * rows + r;
  // with them a split item has its own rows from slots[item] on, one for each
  // of its query rows, out of `rows` in all.
  int chunk, splits, tile_rows;
  int64_t rows;
  float *part_o, *part_ml;
  const int *slots, *joins;
  int n_joins;
};

// Where query row `row`, the in_item-th of an item of item_rows, keeps the
// partial result of split `split`; -1: nowhere (a slot that is not the call's).
__device__ __forceinline__ int64_t part_row(const Attn8Args& p, int64_t item, int split, int64_t row,
                                            int in_item, int item_rows) {
  if (!p.slots) return split * p.rows + row;
  const int slot = p.slots[item];
  return slot < 0 || slot + item_rows > p.rows ? -1 : slot + in_item;
}

// 2^(b - 127) of an E8M0 byte b >= 1
__device__ __forceinline__ float e8m0(int b) { return __uint_as_float((uint32_t)b << 23); }

// 8 codes -> 8 bf16 (exact)
__device__ __forceinline__ v8bf codes_bf16(uint32_t lo, uint32_t hi) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
  return v8bf{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Four codes: which are NaN (0x7f or 0xff), as the bytes' top bits. A key
// that some rows of a tile see and others do not has weight 0 for the others,
// and 0 * NaN would be theirs too: in tiles that a mask cuts, V's NaN codes
// go into the products as 0, and the rows that see them get their NaN at the
// end.
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) {
  return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}
__device__ __forceinline__ uint32_t without(uint32_t w, uint32_t nans) {
  return w & ~((nans >> 7) * 0xffu);
}

// ln(sum exp) of a row from its sum against 2^m; -inf without a key, NaN for
// a NaN sum
__device__ __forceinline__ float row_lse(float sum, float m) {
  return sum == 0.f ? -INFINITY : (__log2f(sum) + m) * 0.6931471805599453f;
}

// One row of one head, 8 consecutive columns on each of its D / 8 lanes: the
// bf16 row, or (D = 128) its e4m3 codes and their scale, from the values
// rounded to bf16 as the separate quantization would see them.
template <int D>
__device__ __forceinline__ void store_row(const Attn8Args& p, int64_t row, int head, int j,
                                          const float (&y)[8]) {
  if (p.out8) {
    if constexpr (D == 128) {
      float v[8], amax = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = round_bf16(y[k]);
        amax = fmaxf(amax, fabsf(v[k]));
      }
      const float s = fp8_scale(group_max<16>(amax));
      const float r = recip(s);
      *reinterpret_cast<uint2*>(p.out8 + row * p.o_ld + head * D + 8 * j) = make_uint2(
          pack4_fp8(div_by(v[0], s, r), div_by(v[1], s, r), div_by(v[2], s, r), div_by(v[3], s, r)),
          pack4_fp8(div_by(v[4], s, r), div_by(v[5], s, r), div_by(v[6], s, r), div_by(v[7], s, r)));
      if (j == 0) p.oscales[(int64_t)head * p.os_ld + row] = s;
    }
    return;
  }
  *reinterpret_cast<uint4*>(p.out16 + row * p.o_ld + head * D + 8 * j) =
      make_uint4(pack2_bf16(y[0], y[1]), pack2_bf16(y[2], y[3]), pack2_bf16(y[4], y[5]),
                 pack2_bf16(y[6], y[7]));
}

// q-norm and RoPE of one column of the few-row kernel: the lanes of a group g4
// hold the row's columns (k / 2) * 64 + g4 * 16 + (k & 1) * 8 .. + 8, so that
// the rotation's pairs, 64 apart, are the lane's own chunks k and k + 2.
template <int QN>
__device__ __forceinline__ void q_norm_columns(v8bf (&qf)[4], const QNormArgs& qn, int64_t pos,
                                               int g4) {
  float x[4][8], ss = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[k][e] = (float)qf[k][e];
      ss += x[k][e] * x[k][e];
    }
  ss += __shfl_xor(ss, 16, 64);
  ss += __shfl_xor(ss, 32, 64);
  const float rstd = norm_rstd<128>(ss, qn.eps);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int c = g4 * 16 + k * 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float a[4], b[4], wa[4], wb[4], cosv[4], sinv[4], oa[4], ob[4];
      bf16x4_to_f32(*reinterpret_cast<const uint2*>(qn.qw + c + 4 * h), wa);
      bf16x4_to_f32(*reinterpret_cast<const uint2*>(qn.qw + 64 + c + 4 * h), wb);
      if constexpr (QN == 2) {
        const float* cs = reinterpret_cast<const float*>(qn.cs) + pos * 128 + c + 4 * h;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          cosv[e] = cs[e];
          sinv[e] = cs[64 + e];
        }
      } else {
        const uint16_t* cs = reinterpret_cast<const uint16_t*>(qn.cs) + pos * 128 + c + 4 * h;
        bf16x4_to_f32(*reinterpret_cast<const uint2*>(cs), cosv);
        bf16x4_to_f32(*reinterpret_cast<const uint2*>(cs + 64), sinv);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = x[k][4 * h + e];
        b[e] = x[k + 2][4 * h + e];
      }
      norm_rope4(a, b, wa, wb, cosv, sinv, rstd, oa, ob);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        qf[k][4 * h + e] = (__bf16)oa[e];
        qf[k + 2][4 * h + e] = (__bf16)ob[e];
      }
    }
  }
}

// Few query rows over long caches. The workgroup's 16 * NB columns are
// (row, head of the KV head's group) pairs of one sequence; its 4 waves take
// turns at steps of 32 keys (two pages) of the split [split * chunk, ...):
// each wave moves its own K and V rows HBM -> LDS (a ring of kRing steps, no
// barrier in the loop) and keeps its own softmax state; the four are joined
// at the end, and splits by split_merge_kernel.
//
// S^T = K Q^T by 16x16x32 MFMAs: lane l holds column l % 16 and, of each
// page, keys 4 (l / 16) + 0..3. P^T is then the PV product's B operand as it
// stands when its 32 k slots are numbered (l / 16) * 8 + page * 4 + r, and
// V^T in that order comes from the row-major codes by ds_read_b64_tr_b8.
// Both tiles are XOR-swizzled by 16-byte chunks: the rows that one LDS read
// touches land in different banks (the conflict counter reads 0).
//
// Bound by reading the codes: 200 one-row sequences of ~2100 keys (32 + 8
// heads of 128, 856 MB) 166 us, 5.2 TB/s, where a kernel that only loads in
// this pattern reaches 5.5; 2 sequences of 40,000 keys with 3 rows of 64
// heads (164 MB, 512 workgroups: one round, its start and end in the open)
// 43 us. One row over 300 keys: 7.8 us, four memory round trips.
constexpr int kRing = 2;

template <int D, int NB, int QN = 0>
__global__ __launch_bounds__(256, 2) void attention8_few_kernel(Attn8Args p, const int* work,
                                                                int seqs, QNormArgs qn) {
  static_assert(kMaxChunk / kPage <= 256, "a page id for each thread");
  constexpr int CH = D / 16;              // 16-byte chunks per code row
  constexpr int NC = D / 32;              // MFMA k-steps over the head dim
  constexpr int ND = D / 16;              // 16-row d blocks of O^T
  constexpr int TILE = 32 * D;            // bytes of one step's K (or V)
  constexpr int LOADS = TILE / 1024;      // direct loads per tile
  constexpr int KPL = 1024 / D;           // keys per direct load
  constexpr int COLS = 16 * NB;
  constexpr int LDS_RING = 4 * kRing * 2 * TILE;
  constexpr int LDS_JOIN = 4 * COLS * D * 4 + 4 * COLS * 8;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[LDS_RING > LDS_JOIN ? LDS_RING : LDS_JOIN];
  __shared__ int pages[kMaxChunk / kPage];
  __shared__ uint16_t bytes[kMaxChunk / kPage];

  // The block table's entries come in one round of loads with the sequence's
  // bounds (rows hold max_used keys' entries; those past the sequence's own
  // are not used), and the scales in one with q and the first step's K and V.
  int s, split;
  if (work) {
    s = work[2 * blockIdx.x];
    split = work[2 * blockIdx.x + 1];
    if (s < 0 || s >= seqs || split < 0 || split >= p.splits) return;  // not an item of this call
  } else {
    s = blockIdx.z;
    split = blockIdx.x;
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int k0 = split * p.chunk;
  const int* trow = p.table + (int64_t)s * p.table_ld;
  const int page = trow[min(k0 / kPage + tid, max((p.max_used - 1) / kPage, 0))];
  const int G = p.HQ / p.HK;
  const int kvh = blockIdx.y % p.HK;
  const int cgroup = blockIdx.y / p.HK;
  const int q0 = p.cu_q[s], q_len = p.cu_q[s + 1] - q0;
  const int used = min(p.used[s], p.max_used);
  const int cols = q_len * G;
  if (cgroup * COLS >= cols || (split && k0 >= used)) return;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g4 = lane >> 4;

  // keys [k0, k1) of this split that the last column of the group sees
  const int last_col = min(cgroup * COLS + COLS, cols) - 1;
  const int seen_end = p.causal ? min(used, used - q_len + last_col / G + 1) : used;
  const int k1 = min(seen_end, k0 + p.chunk);
  const int npages = k1 > k0 ? (k1 - k0 + kPage - 1) / kPage : 0;
  if (tid < npages) pages[tid] = page;
  __syncthreads();

  const int64_t kv_row = (int64_t)p.HK * D;
  const uint8_t* kbase = p.kp + kvh * D;
  const uint8_t* vbase = p.vp + kvh * D;
  uint8_t* ring = lds + wave * (kRing * 2 * TILE);
  auto kswz = [](int key) { return D == 128 ? (key >> 1) & 7 : (key >> 2) & 3; };
  auto vswz = [](int key) {
    return D == 128 ? ((key >> 1) & 3) | ((key >> 2) & 4) : ((key >> 2) & 1) | ((key >> 3) & 2);
  };
  // step t of this wave: keys [k0 + 32 (4 t + wave), + 32); lanes past the
  // split's last key read that key again
  const int nsteps = (npages * kPage + 31) / 32;
  const int mine = nsteps > wave ? (nsteps - wave + 3) / 4 : 0;
  auto issue = [&](int t) {
    const int key0 = 32 * (4 * t + wave);
    uint8_t* at = ring + (t % kRing) * (2 * TILE);
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int in_step = i * KPL + lane / CH;
        const int key = min(key0 + in_step, k1 - k0 - 1);
        const int chunk = (lane % CH) ^ (v ? vswz(in_step) : kswz(in_step));
        const int64_t row = (int64_t)pages[key / kPage] * kPage + key % kPage;
        lds_dma16((v ? vbase : kbase) + row * kv_row + chunk * 16, at + v * TILE + i * 1024);
      }
  };
  if (mine > 0) issue(0);
  if (tid < npages) bytes[tid] = p.scales[(int64_t)page * p.HK + kvh];

  // this lane's columns: their rows, heads, Q fragments and visible keys
  v8bf qf[NB][NC];
  int lim[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int c = cgroup * COLS + n * 16 + c16;
    const int cc = min(c, cols - 1);
    const int r = cc / G, head = kvh * G + cc % G;
    const int64_t row = p.q_index ? p.q_index[q0 + r] : (int64_t)(q0 + r);
    const uint16_t* q = p.q + row * p.q_ld + (int64_t)head * D;
    lim[n] = c < cols ? (p.causal ? min(used, used - q_len + r + 1) : used) : 0;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      qf[n][k] = *reinterpret_cast<const v8bf*>(q + (k >> 1) * (D == 128 ? 64 : 0) + g4 * 16 +
                                                (k & 1) * 8);
    if constexpr (QN != 0) q_norm_columns<QN>(qf[n], qn, qn.pos[row], g4);
#pragma unroll
    for (int k = 0; k < NC; ++k) asm volatile("" ::"v"(qf[n][k]));
  }

  v4f o[NB][ND];
  float m[NB], l[NB];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[n][d] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  __syncthreads();  // bytes, and nothing in flight beside the ring's loads
  // from this key of the split on, some column sees less than the last one
  const int cut = p.causal && q_len > 1
                      ? min(used, used - q_len + cgroup * COLS / G + 1) - k0 : INT32_MAX;
  uint32_t nans = 0;
  for (int t = 0; t < mine; ++t) {
    // this wave's reads of the slot that step t + 1 refills have returned
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    if (t + 1 < mine) {
      issue(t + 1);
      wait_vmcnt<2 * LOADS>();
    } else {
      wait_vmcnt<0>();
    }
    asm volatile("" ::: "memory");
    const uint8_t* kt = ring + (t % kRing) * (2 * TILE);
    const uint8_t* vt = kt + TILE;
    const int key0 = 32 * (4 * t + wave);
    const int pg = key0 / kPage;
    const int b0 = bytes[pg], b1 = bytes[min(pg + 1, npages - 1)];
    const float ks[2] = {e8m0(b0 & 255) * p.scale_log2, e8m0(b1 & 255) * p.scale_log2};
    const float vs[2] = {e8m0(b0 >> 8), e8m0(b1 >> 8)};

    v4f sc[NB][2];
#pragma unroll
    for (int n = 0; n < NB; ++n) sc[n][0] = sc[n][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int pgi = 0; pgi < 2; ++pgi) {
      const int key = pgi * 16 + c16;
#pragma unroll
      for (int k2 = 0; k2 < NC / 2; ++k2) {
        const uint4 w = *reinterpret_cast<const uint4*>(
            kt + key * D + ((k2 * 4 + g4) ^ kswz(key)) * 16);
        const v8bf lo = codes_bf16(w.x, w.y), hi = codes_bf16(w.z, w.w);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          sc[n][pgi] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, qf[n][2 * k2], sc[n][pgi], 0, 0, 0);
          sc[n][pgi] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, qf[n][2 * k2 + 1], sc[n][pgi], 0, 0, 0);
        }
      }
    }
    v8bf pf[NB], pr[NB];  // P and what its rounding to bf16 left
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      const int room = lim[n] - k0 - key0 - g4 * 4;  // key pgi * 16 + r of this lane is below it
      float z[8], top = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        z[e] = (e >> 2) * 16 + (e & 3) < room ? sc[n][e >> 2][e & 3] * ks[e >> 2] : -INFINITY;
        top = fmaxf(top, z[e]);
      }
      top = fmaxf(top, __shfl_xor(top, 16, 64));
      top = fmaxf(top, __shfl_xor(top, 32, 64));
      const float m_new = fmaxf(m[n], top);
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m[n] - m_use);
      m[n] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float pe = __builtin_amdgcn_exp2f(z[e] - m_use);
        sum += pe;
        const float pv = pe * vs[e >> 2];
        pf[n][e] = (__bf16)pv;
        pr[n][e] = (__bf16)(pv - (float)pf[n][e]);
      }
      l[n] = l[n] * alpha + sum;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][d][e] *= alpha;
    }
    const int x = lane & 15;
    const int vkey = (x >> 3) * 16 + g4 * 4 + ((x >> 1) & 3);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      v2i w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
          (lds_v2i*)(vt + vkey * D + ((d ^ vswz(vkey)) * 16) + (x & 1) * 8));
      if (key0 + 32 > cut) {
        const uint32_t n0 = nan_codes(w[0]), n1 = nan_codes(w[1]);
        w = v2i{(int)without(w[0], n0), (int)without(w[1], n1)};
        nans |= n0 | n1;
      }
      const v8bf vf = codes_bf16(w[0], w[1]);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n], o[n][d], 0, 0, 0);
        o[n][d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pr[n], o[n][d], 0, 0, 0);
      }
    }
  }
  if (__builtin_amdgcn_ballot_w64(nans != 0)) {  // rare: the keys of this wave's steps in the cut, again
    for (int t = 0; t < mine; ++t) {
      const int key0 = 32 * (4 * t + wave);
      if (key0 + 32 <= cut) continue;  // its NaN codes went into the products
      for (int key = key0; key < min(key0 + 32, k1 - k0); ++key) {
        const uint8_t* v = vbase + ((int64_t)pages[key / kPage] * kPage + key % kPage) * kv_row;
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          const uint32_t n = nan_codes(*reinterpret_cast<const uint32_t*>(v + d * 16 + g4 * 4));
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (k0 + key < lim[b] && (n >> (8 * e + 7) & 1)) o[b][d][e] = __builtin_nanf("");
        }
      }
    }
  }
  __syncthreads();  // every wave is past its ring

  // join the waves: o of (column, d = 16 blk + 4 g4 + e) as [wave][column][d]
  float* jo = reinterpret_cast<float*>(lds);
  float* jml = jo + 4 * COLS * D;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    l[n] += __shfl_xor(l[n], 16, 64);
    l[n] += __shfl_xor(l[n], 32, 64);
    float* at = jo + (wave * COLS + n * 16 + c16) * D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<v4f*>(at + ((d * 4 + g4) ^ (c16 & 7)) * 4) = o[n][d];
    if (g4 == 0) {
      jml[(wave * COLS + n * 16 + c16) * 2] = m[n];
      jml[(wave * COLS + n * 16 + c16) * 2 + 1] = l[n];
    }
  }
  __syncthreads();
  constexpr int LPC = D / 8;  // lanes per column, 8 values each
  for (int cc = tid / LPC; cc < COLS; cc += 256 / LPC) {
    const int c = cgroup * COLS + cc;
    const int j = tid % LPC;
    if (c >= cols) continue;  // whole columns leave together
    float mm = -INFINITY, ll = 0.f, y[8] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) mm = fmaxf(mm, jml[(w * COLS + cc) * 2]);
    const float m_use = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = __builtin_amdgcn_exp2f(jml[(w * COLS + cc) * 2] - m_use);
      ll += jml[(w * COLS + cc) * 2 + 1] * f;
      const float* at = jo + (w * COLS + cc) * D;
      const v4f a = *reinterpret_cast<const v4f*>(at + ((2 * j) ^ (cc & 7)) * 4);
      const v4f b = *reinterpret_cast<const v4f*>(at + ((2 * j + 1) ^ (cc & 7)) * 4);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        y[k] += a[k] * f;
        y[4 + k] += b[k] * f;
      }
    }
    const int64_t row = q0 + c / G;
    const int head = kvh * G + c % G;
    if (used > p.chunk) {
      const int64_t part = part_row(p, blockIdx.x, split, row, c / G, q_len);
      if (part < 0) continue;
      const int64_t at = part * p.HQ + head;
      if (j == 0) {
        p.part_ml[2 * at] = mm;
        p.part_ml[2 * at + 1] = ll;
      }
      if (mm != -INFINITY) {
        *reinterpret_cast<v4f*>(p.part_o + at * D + 8 * j) = v4f{y[0], y[1], y[2], y[3]};
        *reinterpret_cast<v4f*>(p.part_o + at * D + 8 * j + 4) = v4f{y[4], y[5], y[6], y[7]};
      }
      continue;
    }
    const float inv = ll == 0.f ? 0.f : 1.0f / ll;
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] *= inv;
    store_row<D>(p, row, head, j, y);
    if (p.lse && j == 0)
      p.lse[(int64_t)head * p.lse_ld + row] =
          row_lse(ll, m_use);
  }
}

// Many query rows. A workgroup is 4 waves: QSUB 32-row query tiles of one
// sequence x HPB heads that share a KV head, one wave per (tile, head); keys
// come in 64-key tiles (four pages, one per wave to move), software
// pipelined with one barrier a step. A page's codes travel HBM -> registers,
// become bf16, scaled (exact down to bf16's least number), once per workgroup, and lie in LDS as the
// 16-bit kernel's tiles do, so that both products run on the bf16 matrix
// cores. (Scores from the codes themselves on the FP8 cores, with q as the
// sum of two e4m3 numbers, take the same matrix time and no conversion, but
// those cores drop what lies 2^-12 below the largest product of a sum.)
//
// Bound by the issue of two waves a SIMD (256 registers each): two documents
// of 8000 rows (32 + 8 heads of 128, 1.07 TFLOP) 1.03 ms, 1.04 PFLOP/s (a
// large bf16 product on this card 1.21), matrix cores 48% busy and vector
// units 56%, of which half is exponentials. Short documents add what an item
// costs outside its steps: 46 of ~340 rows (107 GFLOP, 291 MB) 161 us. With
// few rows the longest item's steps count, 1.3 us each alone on a CU: 21
// rows on 60 of ~1000 keys (up to 2064) 54 us.
constexpr int kBK = 64;

// the keys that the last row of a query tile sees, which the tile visits
__host__ __device__ inline int tile_keys(int used, int q_len, int qt, int rows, int causal) {
  const int last = (qt * rows + rows < q_len ? qt * rows + rows : q_len) - 1;
  const int keys = causal ? used - q_len + last + 1 : used;
  return keys < 0 ? 0 : keys < used ? keys : used;
}

// a row's reference max moves when a tile raises its max by more than this
// many powers of two (probabilities then stay below 2^8)
constexpr float kLazyLog2 = 8.0f;
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

template <int D, int HPB, int QSUB, int QN = 0>
__global__ __launch_bounds__(256, 2) void attention8_tile_kernel(Attn8Args p, const int* work,
                                                                 int zgroups, int seqs,
                                                                 QNormArgs qn) {
  static_assert(HPB * QSUB == 4 && (QN == 0 || D == 128), "four waves; q-norm at D = 128");
  constexpr int BQ = 32 * QSUB;
  constexpr int NC = D / 16;       // MFMA k-steps of S
  constexpr int NDS = D / 32;      // 32-row d tiles of O^T
  constexpr int VROW = 2 * D;      // bytes of a bf16 V row in LDS
  constexpr int CH = D / 16;       // 16-byte chunks of a code row
  constexpr int KPL = 1024 / D;    // keys per direct load
  constexpr int LOADS = 16 / KPL;  // loads of a page's 16 rows
  __shared__ __attribute__((aligned(1024))) uint8_t k_lds[2][kBK * VROW];
  __shared__ __attribute__((aligned(1024))) uint8_t v_lds[2][kBK * VROW];
  __shared__ int pages[kMaxKeys / kPage];
  __shared__ uint16_t bytes[kMaxKeys / kPage];
  __shared__ int nans;

  int s, qt, zg, split = 0;
  if (work) {
    const int item = blockIdx.x / zgroups;
    zg = blockIdx.x % zgroups;
    s = work[2 * item];
    qt = work[2 * item + 1] & 0xffff;
    split = work[2 * item + 1] >> 16 & 0x7fff;
  } else {
    s = blockIdx.y;
    qt = gridDim.x - 1 - blockIdx.x;
    zg = blockIdx.z;
  }
  // The sequence's bounds and its pages' ids in one round of loads (rows of
  // the block table hold max_used keys' entries; those past the sequence's
  // own are not used); K, V, q and the scales in the next.
  const int tid = threadIdx.x, lane = tid & 63;
  const int sc = min(max(s, 0), seqs - 1);
  const int k0 = split * p.chunk;
  const int last_entry = max((p.max_used - 1) / kPage, 0);
  const int* trow = p.table + (int64_t)sc * p.table_ld;
  const int page = trow[min(k0 / kPage + tid, last_entry)];
  const int q0 = p.cu_q[sc], q_len = p.cu_q[sc + 1] - q0;
  const int used = min(p.used[sc], p.max_used);
  if (s < 0 || s >= seqs || (split && split >= p.splits) || qt * BQ >= q_len) return;
  const int G = p.HQ / p.HK;
  const int per_kv = G / HPB;
  const int kvh = zg / per_kv;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int head = kvh * G + (zg % per_kv) * HPB + wave % HPB;
  const int qsub = wave / HPB;
  const int half = lane >> 5, col = lane & 31;

  // keys count from the split's first one
  const int off = p.causal ? used - q_len : 0;
  const int wave_row0 = qt * BQ + qsub * 32;
  const int r = wave_row0 + col;
  const bool r_ok = r < q_len;
  const int block_end = tile_keys(used, q_len, qt, BQ, p.causal);
  const bool whole = p.chunk == 0 || block_end <= p.chunk;
  const int kv_end = max(0, whole ? block_end : min(block_end - k0, p.chunk));
  const int ntiles = (kv_end + kBK - 1) / kBK;
  const int npages = (kv_end + kPage - 1) / kPage;
  const int lim = (p.causal ? min(off + r + 1, used) : used) - k0;  // keys < lim are visible
  const int lim_min = (p.causal ? min(off + wave_row0 + 1, used) : used) - k0;
  // tiles from this one on hold keys that some row of the workgroup sees and
  // another does not
  const int cut = p.causal ? max(0, min(used, off + qt * BQ + 1) - k0) / kBK : INT32_MAX;

  int64_t q_pos = 0;  // of this lane's row, for its cos and sin
  if constexpr (QN != 0) q_pos = qn.pos[q0 + (r_ok ? r : q_len - 1)];
  if (tid < npages) pages[tid] = page;
  for (int i = tid + 256; i < npages; i += 256) pages[i] = trow[k0 / kPage + i];
  if (tid == 0) nans = 0;
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): q_pos may be on its way still
  lds_barrier();

  const int64_t kv_row = (int64_t)p.HK * D;
  const uint8_t* kbase = p.kp + kvh * D;
  const uint8_t* vbase = p.vp + kvh * D;
  // A bf16 row in LDS: the first halves of its 16-column blocks, then their
  // second halves, so that the lanes that store a row, a block each, write
  // neighbouring 16-byte chunks (with the halves side by side they wrote every
  // second chunk, and 11% of the kernel's time were bank conflicts); the
  // chunks are swizzled by the key for the reads.
  auto kswz = [](int key) { return D == 128 ? key & 15 : (key >> 1) & 7; };
  auto vswz = [](int key) { return D == 128 ? (key & 3) << 1 : ((key >> 1) & 1) << 1; };
  // Q^T fragments (B operand): lane holds row `col`, d = c * 16 + half * 8 .. + 8
  v8bf qf[NC];
  // this wave's page of a tile: lane's 16 codes of row j * KPL + lane / CH
  const int row0 = lane / CH, chunk = lane % CH;
  uint4 kreg[LOADS], vreg[LOADS];
  // this wave's page of tile t (the last one past the keys' end), and the
  // lane's bytes in it: rows past the last key read that one again
  auto slot_of = [&](int t) { return min(t * kBK + wave * kPage, kv_end - 1) / kPage; };
  auto place = [&](int t, int j) -> uint32_t {
    const int left = kv_end - 1 - slot_of(t) * kPage;
    return (uint32_t)(min(row0 + j * KPL, left) * (int)kv_row + chunk * 16);
  };
  auto load = [&](int t, const uint8_t* base, uint4 (&reg)[LOADS]) {
    const int64_t page = __builtin_amdgcn_readfirstlane(pages[slot_of(t)]);
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      reg[j] = *reinterpret_cast<const uint4*>(base + page * kPage * kv_row + place(t, j));
  };
  // the scale of this wave's page of a tile
  auto bytes_of = [&](int t) -> int { return bytes[min(t * (kBK / kPage) + wave, npages - 1)]; };
  auto scale_of = [&](int pair, bool v) -> float {
    const int b = __builtin_amdgcn_readfirstlane(pair);
    return e8m0(v ? b >> 8 : b & 255);
  };
  // where this lane's 16 codes of row row0 + j KPL go, as bf16: st_k ^ 128 j
  // (st_v) past j KPL rows, and their second half at that ^ 16 CH
  const int st_row = (wave * kPage + row0) * VROW;
  const int st_k = st_row + ((chunk ^ kswz(row0)) * 16);
  const int st_v = st_row + ((chunk ^ vswz(row0)) * 16);
  auto store = [&](uint8_t* tile, uint4 reg, int j, int at, float scale, bool v, bool check) {
    uint32_t w[4] = {reg.x, reg.y, reg.z, reg.w};
    if (check) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t n = nan_codes(w[i]);
        if (n) nans = 1;
        w[i] = without(w[i], n);
      }
    }
    uint32_t b[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, false));
      b[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, true));
    }
    uint8_t* to = tile + j * KPL * VROW + (v ? at : at ^ (128 * j));
    *reinterpret_cast<uint4*>(to) = make_uint4(b[0], b[1], b[2], b[3]);
    *reinterpret_cast<uint4*>(tile + j * KPL * VROW + ((v ? at : at ^ (128 * j)) ^ (16 * CH))) = make_uint4(b[4], b[5], b[6], b[7]);
  };
  auto store_all = [&](int t, uint8_t* tile, const uint4 (&reg)[LOADS], bool v) {
    const float scale = scale_of(bytes_of(t), v);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) store(tile, reg[j], j, v ? st_v : st_k, scale, v, v && t >= cut);
  };
  // a whole tile's rows: this wave's page, and each lane's place in it
  uint32_t in_page[LOADS];
#pragma unroll
  for (int j = 0; j < LOADS; ++j) in_page[j] = (uint32_t)((row0 + j * KPL) * (int)kv_row + chunk * 16);
  // K fragment (A operand of S^T): key `col` (+ 32), d chunk 2c + half, at
  // k_base ^ 16 c (the swizzle moves chunks within the row)
  const int k_base = col * VROW + ((CH * half ^ kswz(col)) * 16);
  // V^T fragment by transposing reads: lane 16 g + x reads 4 halfwords of key
  // 4 * half + x / 4 (+ 8) at column 16 (g & 1) + 4 (x & 3) of a 32-d tile,
  // d tile d at v_base ^ 32 d
  const int v_key = 4 * half + ((lane & 15) >> 2);
  const int v_base = v_key * VROW +
                     (((((lane >> 4) & 1) + CH * ((lane & 3) >> 1)) ^ vswz(v_key)) * 16) + 8 * (lane & 1);

  v16f o[NDS];
#pragma unroll
  for (int d = 0; d < NDS; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m_run = -INFINITY, l_run = 0.f;

  auto read_k = [&](const uint8_t* kl, int kb, int c, v8bf (&f)[2]) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
      f[ks] = *reinterpret_cast<const v8bf*>(kl + ks * 32 * VROW + (kb ^ (16 * c)));
  };
  auto read_v = [&](const uint8_t* vl, int vb, int kc, int d) -> v8bf {
    const uint8_t* at = vl + ((kc >> 1) * 32 + (kc & 1) * 16) * VROW + (vb ^ (32 * d));
    const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at);
    const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 8 * VROW));
    const v8s both = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(v8bf, both);
  };
  auto mask_tile = [&](int t, v16f (&sacc)[2]) {
    const int t0 = t * kBK;
    if (t0 + kBK <= lim_min) return;  // every row of the wave sees it whole
    const int room = lim - t0 - half * 4;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        sacc[ks][i] = ks * 32 + (i >> 2) * 8 + (i & 3) < room ? sacc[ks][i] : -INFINITY;
  };
  // the largest of scores 8 g .. 8 g + 8 of a tile
  auto part_max = [&](const v16f (&sacc)[2], int g) {
    float m = sacc[g >> 1][(g & 1) * 8];
#pragma unroll
    for (int i = 1; i < 8; ++i) m = fmaxf(m, sacc[g >> 1][(g & 1) * 8 + i]);
    return m;
  };
  auto step_end = [&]() {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    lds_barrier();
  };
  // Step t: softmax and PV of tile t beside S of tile t + 1. Tiles reach LDS
  // a step before their use: K of tile t + 2 and V of tile t + 1 are stored
  // from the registers that step t - 1 loaded, and the next ones load. The
  // new maximum and the exponentials run between the S MFMAs, the conversions
  // and stores between the PV MFMAs, in an order that sched_barrier keeps (the
  // maximum before the first MFMA: 1-2% slower).
  // FAST: no row's mask reaches tiles t and t + 1, and tiles up to t + 3 are
  // whole.
  enum { kFast, kNext, kLast };
  auto step = [&](const int t, const int cur, v16f (&s_cur)[2], v16f (&s_next)[2], auto kind_c) {
    constexpr int KIND = decltype(kind_c)::value;
    constexpr bool LAST = KIND == kLast, FAST = KIND == kFast;
    const uint8_t* kl = &k_lds[cur ^ 1][0];
    const uint8_t* vl = &v_lds[cur][0];
    // recomputed here rather than kept across the loop
    const int kb = opaque(k_base), vb = opaque(v_base);
    const int sk = opaque(st_k), sv = opaque(st_v);
    constexpr int kAhead = 1;  // chunks of K read before their MFMAs: more were as fast, and took registers
    v8bf kf[NC][2];
    int page_v = 0, page_k = 0;
    int pair_k = 0, pair_v = 0;
    if (!LAST) {
#pragma unroll
      for (int c = 0; c < kAhead; ++c) read_k(kl, kb, c, kf[c]);
    }
    if (!FAST) mask_tile(t, s_cur);
    float part[4], alpha = 1.f, m_use = 0.f, psum = 0.f;
    bool move = false;
    v8bf pf[4], vf[4][NDS];
    constexpr int LEAD = NC / 2;  // MFMAs behind which the new maximum is found
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (!LAST) {
          __builtin_amdgcn_sched_barrier(0);
          if (ks == 0 && c + kAhead < NC) read_k(kl, kb, c + kAhead, kf[c + kAhead]);
          if (c == 0 && ks == 1) {
            page_v = pages[FAST ? (t + 2) * (kBK / kPage) + wave : slot_of(t + 2)];
            page_k = pages[FAST ? (t + 3) * (kBK / kPage) + wave : slot_of(t + 3)];
          }
          if (c == 1 && ks == 1) {
            pair_v = bytes_of(t + 1);
            pair_k = bytes_of(t + 2);
          }
        }
        if (c == NC - 1) {  // V of the first 16 keys
#pragma unroll
          for (int d = ks * (NDS / 2); d < (ks + 1) * (NDS / 2); ++d) vf[0][d] = read_v(vl, vb, 0, d);
        }
        if (!LAST)
          s_next[ks] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[c][ks], qf[c], c == 0 ? v16f{} : s_next[ks], 0, 0, 0);
        const int slot = 2 * c + ks;
        if (slot < LEAD / 2) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (g * LEAD / 8 == slot) part[g] = part_max(s_cur, g);
        }
        if (slot == LEAD / 2) {
          const float tmax = max_halves(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
          const float m_cand = fmaxf(m_run, tmax);
          move = (m_cand - m_run) * p.scale_log2 > kLazyLog2;
          alpha = move ? __builtin_amdgcn_exp2f((m_run - m_cand) * p.scale_log2) : 1.0f;
          m_run = move ? m_cand : m_run;
          m_use = m_run == -INFINITY ? 0.f : m_run * p.scale_log2;
        }
        if (slot == LEAD - 1 && __builtin_amdgcn_ballot_w64(move)) {
#pragma unroll
          for (int d = 0; d < NDS; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
        }
        constexpr int REST = 2 * NC - LEAD;  // MFMAs behind which the 32 exponentials run
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          if (slot < LEAD || i < 32 * (slot - LEAD) / REST || i >= 32 * (slot - LEAD + 1) / REST) continue;
          const float pv = __builtin_amdgcn_exp2f(fmaf(s_cur[i >> 4][i & 15], p.scale_log2, -m_use));
          psum += pv;
          pf[i >> 3][i & 7] = (__bf16)pv;
        }
      }
    if (!LAST) __builtin_amdgcn_sched_barrier(0);
    l_run = l_run * alpha + sum_halves(psum);
    const float scale_v = LAST ? 1.f : scale_of(pair_v, true);
    const float scale_k = LAST ? 1.f : scale_of(pair_k, false);
    constexpr int SLOTS = 4 * NDS;  // MFMAs of PV; 2 LOADS stores go behind every few
#pragma unroll
    for (int kc = 0; kc < 4; ++kc)
#pragma unroll
      for (int d = 0; d < NDS; ++d) {
        if (kc < 3) vf[kc + 1][d] = read_v(vl, vb, kc + 1, d);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[kc][d], pf[kc], o[d], 0, 0, 0);
        if (!LAST) {
          const int slot = kc * NDS + d;
          if (slot % (SLOTS / (2 * LOADS)) == 0) {
            const int u = slot / (SLOTS / (2 * LOADS)), j = u % LOADS;
            if (u < LOADS)
              store(&v_lds[cur ^ 1][0], vreg[j], j, sv, scale_v, true, !FAST && t + 1 >= cut);
            else if (FAST || t + 2 < ntiles)
              store(&k_lds[cur][0], kreg[j], j, sk, scale_k, false, false);
            // the register's next load
            if (FAST || t + (u < LOADS ? 2 : 3) < ntiles)
              (u < LOADS ? vreg : kreg)[j] = *reinterpret_cast<const uint4*>(
                  (u < LOADS ? vbase : kbase) +
                  (int64_t)__builtin_amdgcn_readfirstlane(u < LOADS ? page_v : page_k) * kPage * kv_row +
                  (FAST ? in_page[j] : place(t + (u < LOADS ? 2 : 3), j)));
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    step_end();
  };

  v16f sa[2], sb[2];
  int checked = cut;  // the first tile whose NaN codes were left out
  if (ntiles > 0) {
    uint4 k1[LOADS];
    QNormIn<QN == 0 ? 1 : QN> qin;
    load(0, kbase, kreg);
    load(0, vbase, vreg);
    if (ntiles > 1) load(1, kbase, k1);
    uint16_t pair = 0;
    if (tid < npages) pair = p.scales[(int64_t)page * p.HK + kvh];
    {
      const int rr = r_ok ? r : q_len - 1;
      const int64_t row = p.q_index ? p.q_index[q0 + rr] : (int64_t)(q0 + rr);
      const uint16_t* q = p.q + row * p.q_ld + (int64_t)head * D;
#pragma unroll
      for (int c = 0; c < NC; ++c) qf[c] = *reinterpret_cast<const v8bf*>(q + c * 16 + half * 8);
    }
    if constexpr (QN != 0) {
      q_norm_load_weights(qin, qn, half);
      q_norm_load_row(qin, qn, q_pos, half);
    }
    if (tid < npages) bytes[tid] = pair;
    for (int i = tid + 256; i < npages; i += 256)
      bytes[i] = p.scales[(int64_t)pages[i] * p.HK + kvh];
    __builtin_amdgcn_s_waitcnt(0xc07f);
    lds_barrier();
    store_all(0, &k_lds[0][0], kreg, false);
    store_all(0, &v_lds[0][0], vreg, true);
    if (ntiles > 1) {
      store_all(1, &k_lds[1][0], k1, false);
      load(1, vbase, vreg);
      if (ntiles > 2) load(2, kbase, kreg);
    }
    if constexpr (QN != 0) {
      v8s raw[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) raw[c] = __builtin_bit_cast(v8s, qf[c]);
      q_norm_rope_apply(raw, qin, qn.eps);
#pragma unroll
      for (int c = 0; c < 8; ++c) qf[c] = __builtin_bit_cast(v8bf, raw[c]);
    }
    step_end();
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      v8bf kf[2];
      read_k(&k_lds[0][0], k_base, c, kf);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        sa[ks] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], qf[c], c == 0 ? v16f{} : sa[ks], 0, 0, 0);
    }
    step_end();
    int t = 0;
    const int whole_tiles = kv_end / kBK;
    for (; t + 4 < whole_tiles && t + 2 < cut; t += 2) {
      step(t, 0, sa, sb, std::integral_constant<int, kFast>{});
      step(t + 1, 1, sb, sa, std::integral_constant<int, kFast>{});
    }
    for (; t + 2 < ntiles; t += 2) {
      step(t, 0, sa, sb, std::integral_constant<int, kNext>{});
      step(t + 1, 1, sb, sa, std::integral_constant<int, kNext>{});
    }
    if (t + 1 < ntiles) {
      step(t, 0, sa, sb, std::integral_constant<int, kNext>{});
      step(t + 1, 1, sb, sa, std::integral_constant<int, kLast>{});
    } else {
      step(t, 0, sa, sb, std::integral_constant<int, kLast>{});
    }
  }

  if (nans) {  // rare: the keys of the tiles looked at, again
    for (int key = checked * kBK; key < kv_end; ++key) {
      const uint8_t* v = vbase + ((int64_t)pages[key / kPage] * kPage + key % kPage) * kv_row;
#pragma unroll
      for (int d = 0; d < NDS; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const uint32_t n = nan_codes(*reinterpret_cast<const uint32_t*>(v + d * 32 + g * 8 + half * 4));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (key < lim && (n >> (8 * e + 7) & 1)) o[d][g * 4 + e] = __builtin_nanf("");
        }
    }
  }

  // epilogue: lane holds row `col`, d = dt * 32 + (i / 4) * 8 + half * 4 + i % 4;
  // the wave's rows go out through LDS so that a store writes whole rows,
  // 16-byte chunks XOR-swizzled by the row
  if (!whole) {  // a split: its state as it stands
    const int64_t part = part_row(p, blockIdx.x / zgroups, split, q0 + r, r - qt * BQ,
                                  min(BQ, q_len - qt * BQ));
    const int64_t at = part * p.HQ + head;
    if (r_ok && part >= 0) {
#pragma unroll
      for (int d = 0; d < NDS; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<v4f*>(p.part_o + at * D + d * 32 + g * 8 + half * 4) =
              v4f{o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]};
      if (half == 0) {
        p.part_ml[2 * at] = m_run * p.scale_log2;
        p.part_ml[2 * at + 1] = l_run;
      }
    }
    return;
  }
  const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
  if (p.lse && r_ok && half == 0) {
    const float m_use = m_run == -INFINITY ? 0.f : m_run * p.scale_log2;
    p.lse[(int64_t)head * p.lse_ld + q0 + r] =
        row_lse(l_run, m_use);
  }
  uint8_t* stage = &v_lds[0][0] + wave * 32 * VROW;
  static_assert(4 * 32 * VROW <= sizeof(v_lds), "epilogue staging");
  constexpr int OCH = VROW / 16;
#pragma unroll
  for (int d = 0; d < NDS; ++d)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int at = 2 * (d * 32 + g * 8 + half * 4);
      *reinterpret_cast<uint2*>(stage + col * VROW + (((at >> 4) ^ (col % OCH)) << 4) + (at & 15)) =
          make_uint2(pack2_bf16(o[d][g * 4] * inv, o[d][g * 4 + 1] * inv),
                     pack2_bf16(o[d][g * 4 + 2] * inv, o[d][g * 4 + 3] * inv));
    }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  constexpr int LPC = D / 8, RPP = 64 / LPC;
  const int rows_here = min(32, q_len - wave_row0);
#pragma unroll
  for (int pass = 0; pass < 32 / RPP; ++pass) {
    const int rr = pass * RPP + lane / LPC, j = lane % LPC;
    const uint4 w = *reinterpret_cast<const uint4*>(stage + rr * VROW + ((j ^ (rr % OCH)) << 4));
    if (rr < rows_here) {  // whole rows
      const float y[8] = {lo_bf16(w.x), hi_bf16(w.x), lo_bf16(w.y), hi_bf16(w.y),
                          lo_bf16(w.z), hi_bf16(w.z), lo_bf16(w.w), hi_bf16(w.w)};
      store_row<D>(p, q0 + wave_row0 + rr, head, j, y);
    }
  }
}

// Join the splits of each (row, head), WAVES waves per pair: a lane weighs
// one split (in every wave alike), and each group of 16 lanes adds up every
// (4 WAVES)-th split's output. A split without a key has an output that
// nobody wrote: it is read and not used. A launch of 4 to 7 us
// (latency: work, then (m, l), then outputs), beside 14 to 166 us of the
// kernels that it joins.
// joins: 4 ints for each split tile (or sequence of few rows), {first query
// row, rows, first row of partial results, splits}, blockIdx.y of them; the
// grid and the partial results then cost what is split (over every sequence, a
// pack of 46 documents beside 21 rows on 40,000 keys started 323,000
// workgroups to join 21 rows). Without them: every sequence.
template <int D, int WAVES>
__global__ __launch_bounds__(256) void split_merge_kernel(Attn8Args p) {
  constexpr int PER = D / 16;  // columns per lane
  constexpr int GROUPS = 4 * WAVES;
  __shared__ v4f part[WAVES > 1 ? GROUPS * D / 4 : 1];
  const int wave = threadIdx.x >> 6;
  const int in_seq = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  const int head = in_seq % p.HQ;
  int splits;
  int64_t row, pair, step;
  if (p.joins) {
    const int* join = p.joins + 4 * blockIdx.y;
    const int rows = join[1];
    splits = join[3];
    if (in_seq >= rows * p.HQ || join[2] < 0 || join[2] + (int64_t)rows * splits > p.rows) return;
    row = join[0] + in_seq / p.HQ;
    pair = (int64_t)(join[2] + in_seq / p.HQ) * p.HQ + head;
    step = (int64_t)rows * p.HQ;
  } else {
    const int s = blockIdx.y;
    const int q0 = p.cu_q[s], q_len = p.cu_q[s + 1] - q0;
    const int used = min(p.used[s], p.max_used);
    if (in_seq >= q_len * p.HQ) return;
    const int keys = p.tile_rows
                         ? tile_keys(used, q_len, in_seq / p.HQ / p.tile_rows, p.tile_rows, p.causal)
                         : used;
    if (keys <= p.chunk) return;  // not split: its rows went out whole
    splits = (keys + p.chunk - 1) / p.chunk;
    row = q0 + in_seq / p.HQ;
    pair = row * p.HQ + head;
    step = p.rows * p.HQ;
  }
  const int lane = threadIdx.x & 63, j = lane & 15;
  const int g = (WAVES == 1 ? 0 : 4 * wave) + (lane >> 4);
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + pair;
  const float* po = p.part_o + pair * D + PER * j;
  float mm = -INFINITY, ll = 0.f, y[PER] = {};
  for (int first = 0; first < splits; first += 64) {
    const bool live = first + lane < splits;
    const float2 mine = live ? ml[(first + lane) * step] : make_float2(-INFINITY, 0.f);
    const float top = fmaxf(mm, group_max<64>(mine.x));
    const float top_use = top == -INFINITY ? 0.f : top;
    const float w = __builtin_amdgcn_exp2f(mine.x - top_use);
    const float out_w = mine.x == -INFINITY ? -1.f : w;  // no key, no output; 0 is a weight (of NaN, too)
    const float keep = __builtin_amdgcn_exp2f(mm - top_use);
    ll = ll * keep + group_sum<64>(mine.y * w);
    mm = top;
#pragma unroll
    for (int k = 0; k < PER; ++k) y[k] *= keep;
    const int n = min(64, splits - first);
    constexpr int UNROLL = 4;
    for (int i = g; i < n; i += UNROLL * GROUPS) {
      v4f a[UNROLL][PER / 4];
      float wi[UNROLL];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int at = i + u * GROUPS;
        wi[u] = __shfl(out_w, min(at, 63), 64);
        if (at >= n) wi[u] = -1.f;
#pragma unroll
        for (int k = 0; k < PER / 4; ++k)
          a[u][k] = *reinterpret_cast<const v4f*>(po + (first + min(at, n - 1)) * step * D + 4 * k);
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u)
#pragma unroll
        for (int k = 0; k < PER; ++k)
          y[k] = wi[u] < 0.f ? y[k] : fmaf(a[u][k >> 2][k & 3], wi[u], y[k]);
    }
  }
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int k = 0; k < PER / 4; ++k)
      part[g * (D / 4) + j * (PER / 4) + k] = v4f{y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]};
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int k = 0; k < PER; ++k) y[k] = 0.f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i)
#pragma unroll
      for (int k = 0; k < PER / 4; ++k) {
        const v4f a = part[(i * 4 + (lane >> 4)) * (D / 4) + j * (PER / 4) + k];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[4 * k + e] += a[e];
      }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    y[k] += __shfl_xor(y[k], 16, 64);
    y[k] += __shfl_xor(y[k], 32, 64);
  }
  const float inv = ll == 0.f ? 0.f : 1.0f / ll;
#pragma unroll
  for (int k = 0; k < PER; ++k) y[k] *= inv;
  // D / 8 lanes store 8 columns each
  if constexpr (PER == 4) {
    float z[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      z[k] = y[k];
      z[4 + k] = __shfl(y[k], lane + 1, 64);
    }
    if (lane < 16 && !(j & 1)) store_row<D>(p, row, head, j >> 1, z);
  } else {
    if (lane < 16) store_row<D>(p, row, head, j, y);
  }
  if (p.lse && lane == 0)
    p.lse[(int64_t)head * p.lse_ld + row] =
        row_lse(ll, mm);
}

// Column blocks of a workgroup: two of 16 where a sequence's (row, head)
// pairs pass one.
inline int few_blocks(int64_t max_q, int64_t G) { return max_q * G > 16 ? 2 : 1; }

// Keys per split (a multiple of 128: the four waves' steps) of sequences
// whose longest has max_used keys and which hold `keys` keys in all. A step
// of 128 keys takes a workgroup about 1 us where few run (memory latency),
// joining splits 3 us and a launch, so
//   - sequences of up to 768 keys are not split (1 of 300 keys: 6.9 us, in
//     two 9.1; 1 of 1000: 11.9 us whole, 9.5 in splits of 256);
//   - calls that one round of workgroups covers take about 256 of them (1
//     sequence of 40,000 keys: 21.3 us in 1280s, 23.9 in 640s, 26.7 in 384s;
//     16 of ~1000: 18 us, 17.3, 19.5);
//   - larger ones at least 1024 for an even end, of up to 2048 keys (16 of
//     ~9000 keys: 70.3 us in 1280s, 76.7 in 2048s; 200 of ~1900 keys: 150 us
//     in 1024s as in 2048s, 144 in 4096s; of ~350: 38.4 whole, 46 split).
int64_t split_chunk(int64_t keys, int64_t max_q, int64_t max_used, int64_t HK,
                    int64_t G) {
  const int64_t cols = 16 * few_blocks(max_q, G);
  const int64_t total = keys * HK * ((max_q * G + cols - 1) / cols);  // keys of all workgroups
  int64_t chunk = std::max(std::min<int64_t>(total / 256, 1280), std::min<int64_t>(total / 1024, 2048));
  chunk = max_used <= 768 ? max_used : std::max<int64_t>(256, std::min(chunk, max_used));
  return std::max<int64_t>(128, (chunk + 127) / 128 * 128);
}

// Heads per workgroup of the tile kernel, and its query rows.
inline int tile_heads(int64_t G) { return G % 4 == 0 ? 4 : (G % 2 == 0 ? 2 : 1); }
inline int tile_height(int64_t G) { return 32 * (4 / tile_heads(G)); }

// The few-row kernel up to two column blocks.
inline bool few_rows(int64_t max_q, int64_t G) { return max_q * G <= 32; }

template <int D>
void merge_launch(const Attn8Args& a, int64_t seqs, int64_t max_q, hipStream_t stream) {
  if (a.slots) {  // only what is split
    seqs = a.n_joins;
    if (a.tile_rows) max_q = std::min<int64_t>(max_q, a.tile_rows);
    if (seqs == 0) return;
  }
  if (a.splits > 16)
    hipLaunchKernelGGL((split_merge_kernel<D, 4>), dim3((unsigned)(max_q * a.HQ), (unsigned)seqs),
                       dim3(256), 0, stream, a);
  else if (a.splits > 1)
    hipLaunchKernelGGL((split_merge_kernel<D, 1>),
                       dim3((unsigned)((max_q * a.HQ + 3) / 4), (unsigned)seqs), dim3(256), 0,
                       stream, a);
}

// q as the call has it: normed (QN 0), or the projection's with a bf16 (1) or
// fp32 (2) cos/sin cache
template <int D, int QN>
void tile_launch(const Attn8Args& a, const QNormArgs& qn, const int* work, int64_t n_work,
                 int64_t seqs, int64_t max_q, hipStream_t stream) {
  const int G = a.HQ / a.HK, hpb = tile_heads(G), rows = tile_height(G);
  const int zgroups = a.HQ / hpb;
  const dim3 grid = work ? dim3((unsigned)(n_work * zgroups))
                         : dim3((unsigned)((max_q + rows - 1) / rows), (unsigned)seqs,
                                (unsigned)zgroups);
#define QX_TILE(H, Q)                                                                          \
  hipLaunchKernelGGL((attention8_tile_kernel<D, H, Q, QN>), grid, dim3(256), 0, stream, a,     \
                     work, zgroups, (int)seqs, qn)
  if (hpb == 4) QX_TILE(4, 1);
  else if (hpb == 2) QX_TILE(2, 2);
  else QX_TILE(1, 4);
#undef QX_TILE
  merge_launch<D>(a, seqs, max_q, stream);
}

template <int D, int QN>
void few_launch(const Attn8Args& a, const QNormArgs& qn, const int* work, int64_t n_work,
                int64_t seqs, int64_t max_q, hipStream_t stream) {
  const int G = a.HQ / a.HK, cols = 16 * few_blocks(max_q, G);
  const int64_t groups = (max_q * G + cols - 1) / cols;
  const dim3 grid(work ? (unsigned)n_work : (unsigned)a.splits, (unsigned)(a.HK * groups),
                  work ? 1u : (unsigned)seqs);
  if (cols == 16)
    hipLaunchKernelGGL((attention8_few_kernel<D, 1, QN>), grid, dim3(256), 0, stream, a, work,
                       (int)seqs, qn);
  else
    hipLaunchKernelGGL((attention8_few_kernel<D, 2, QN>), grid, dim3(256), 0, stream, a, work,
                       (int)seqs, qn);
  merge_launch<D>(a, seqs, max_q, stream);
}

template <int D, int QN>
void attention8_launch(const Attn8Args& a, const QNormArgs& qn, const int* work, int64_t n_work,
                       int64_t seqs, int64_t max_q, hipStream_t stream) {
  if (a.tile_rows) tile_launch<D, QN>(a, qn, work, n_work, seqs, max_q, stream);
  else few_launch<D, QN>(a, qn, work, n_work, seqs, max_q, stream);
}

// What a call's work items are: keys per split of the few-row kernel (> 0),
// query tiles (0), or query tiles in splits of that many keys (< 0).
int64_t list_unit(const int* cu_q, const int* used, int64_t seqs, int64_t HQ, int64_t HK,
                  int causal) {
  const int64_t G = HQ / HK;
  int64_t max_q = 0, max_used = 0, keys = 0;
  for (int64_t s = 0; s < seqs; ++s) {
    max_q = std::max<int64_t>(max_q, cu_q[s + 1] - cu_q[s]);
    max_used = std::max<int64_t>(max_used, used[s]);
    keys += std::max(used[s], 0);
  }
  if (few_rows(max_q, G)) return split_chunk(keys, max_q, max_used, HK, G);
  // 64-key steps of all workgroups, and of the longest one. A step takes about
  // 1.6 us in a workgroup alone on its CU, 2.1 beside another; joining splits a
  // launch and the traffic of their rows. Split
  //   - into 256 workgroups of equal steps, where the longest has 6 more (21
  //     rows on one document of 8000 tokens: 156 us whole, 25; on 8 of ~900:
  //     34, 21; 100 on 8 of ~8000: 228, 142);
  //   - into 512 where it has 24 more and a quarter more (12 rows on 60
  //     documents of ~4000: 203, 192); not for less (21 rows on 60 of ~1000, 33
  //     steps against 15: 56 us whole, 74; one document's 2000 rows: 60, 87).
  const int rows = tile_height(G);
  int64_t steps = 0, longest = 0;
  for (int64_t s = 0; s < seqs; ++s)
    for (int qt = 0; (int64_t)qt * rows < cu_q[s + 1] - cu_q[s]; ++qt) {
      const int64_t n = (tile_keys(used[s], cu_q[s + 1] - cu_q[s], qt, rows, causal) + kBK - 1) / kBK;
      steps += n;
      longest = std::max(longest, n);
    }
  steps *= HQ / tile_heads(G);
  const int64_t one = std::max<int64_t>(4, (steps + 255) / 256);
  if (longest > one + 6) return -kBK * one;
  const int64_t two = std::max<int64_t>(4, (steps + 511) / 512);
  if (longest > two + 24 && longest * 4 > two * 5) return -kBK * two;
  return 0;
}

// The same of a call without a list: whole query tiles where rows are many.
int64_t call_unit(int64_t keys, int64_t max_q, int64_t max_used, int64_t HK, int64_t G) {
  return few_rows(max_q, G) ? split_chunk(keys, max_q, max_used, HK, G) : 0;
}

}  // namespace
}  // namespace qx

using namespace qx;

extern "C" {

int qx_paged_attention8_unit(const int* cu_q, const int* used, int64_t seqs, int64_t HQ,
                             int64_t HK, int causal, int64_t* unit) {
  QX_CHECK(cu_q && used && unit && seqs >= 0 && HQ > 0 && HK > 0 && HQ % HK == 0,
           "attention8_unit: arguments");
  *unit = list_unit(cu_q, used, seqs, HQ, HK, causal);
  return QX_OK;
}

// Items of (sequence, part), heaviest first; rows 0: parts are splits of
// `unit` keys, else part = query tile | split << 16 (unit 0: no splits).
static int64_t work_list(const int* cu_q, const int* used, int64_t seqs, int rows, int causal,
                         int64_t unit, int* work, int64_t capacity) {
  struct Item { int64_t load; int s, part; };
  std::vector<Item> items;
  for (int64_t s = 0; s < seqs; ++s) {
    const int q_len = cu_q[s + 1] - cu_q[s];
    for (int qt = 0; rows ? qt * rows < q_len : qt < 1 && q_len > 0; ++qt) {
      const int64_t keys = rows ? tile_keys(used[s], q_len, qt, rows, causal) : used[s];
      const int64_t part = unit ? unit : std::max<int64_t>(keys, 1);
      for (int64_t i = 0, k0 = 0; i == 0 || k0 < keys; ++i, k0 += part)
        items.push_back({std::min(part, keys - k0), (int)s, rows ? (int)(qt | i << 16) : (int)i});
    }
  }
  QX_CHECK((int64_t)items.size() <= capacity, "attention8_work: %zu items, room for %lld",
           items.size(), (long long)capacity);
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& a, const Item& b) { return a.load > b.load; });
  for (size_t i = 0; i < items.size(); ++i) {
    work[2 * i] = items[i].s;
    work[2 * i + 1] = items[i].part;
  }
  return (int64_t)items.size();
}

int64_t qx_paged_attention8_work(const int* cu_q, const int* used, int64_t seqs, int64_t HQ,
                                 int64_t HK, int causal, int64_t unit, int* work,
                                 int64_t capacity) {
  QX_CHECK(cu_q && used && work && seqs >= 0 && HQ > 0 && HK > 0 && HQ % HK == 0,
           "attention8_work: arguments");
  const int rows = unit > 0 ? 0 : tile_height(HQ / HK);
  for (int64_t s = 0; s < seqs; ++s)
    QX_CHECK((cu_q[s + 1] - cu_q[s]) / 32 < 65536, "attention8_work: a sequence of %d rows",
             cu_q[s + 1] - cu_q[s]);
  try {
    return work_list(cu_q, used, seqs, rows, causal, unit < 0 ? -unit : unit, work, capacity);
  } catch (const std::bad_alloc&) {
    set_error("attention8_work: out of host memory");
    return QX_EINVAL;
  }
}

// The split tiles of a list, in the list's order of their first parts.
static int64_t join_list(const int* cu_q, const int* used, int64_t seqs, int rows, int causal,
                         int64_t unit, const int* work, int64_t n_work, int* slots, int* joins,
                         int64_t capacity, int64_t* part_rows) {
  std::unordered_map<int64_t, int64_t> first;  // (sequence, tile) -> first row of partial results
  int64_t n = 0, total = 0;
  for (int64_t i = 0; i < n_work; ++i) {
    const int s = work[2 * i];
    const int qt = rows ? work[2 * i + 1] & 0xffff : 0;
    const int split = rows ? work[2 * i + 1] >> 16 : work[2 * i + 1];
    QX_CHECK(s >= 0 && s < seqs && split >= 0, "attention8_joins: item %lld is none of this call's",
             (long long)i);
    const int q_len = cu_q[s + 1] - cu_q[s];
    const int64_t keys = rows ? tile_keys(used[s], q_len, qt, rows, causal) : used[s];
    slots[i] = -1;
    if (!unit || keys <= unit) continue;
    const int row0 = rows ? qt * rows : 0, here = rows ? std::min(rows, q_len - row0) : q_len;
    const int64_t parts = (keys + unit - 1) / unit;
    QX_CHECK(here > 0 && split < parts, "attention8_joins: item %lld is none of this call's",
             (long long)i);
    const auto at = first.emplace((int64_t)s << 32 | qt, total);
    if (at.second) {
      QX_CHECK(n < capacity, "attention8_joins: more split tiles than the %lld there is room for",
               (long long)capacity);
      QX_CHECK(total + here * parts <= INT32_MAX, "attention8_joins: too many partial rows");
      const int join[4] = {cu_q[s] + row0, here, (int)total, (int)parts};
      std::copy(join, join + 4, joins + 4 * n++);
      total += here * parts;
    }
    slots[i] = (int)at.first->second + split * here;
  }
  *part_rows = total;
  return n;
}

int64_t qx_paged_attention8_joins(const int* cu_q, const int* used, int64_t seqs, int64_t HQ,
                                  int64_t HK, int causal, int64_t unit, const int* work,
                                  int64_t n_work, int* slots, int* joins, int64_t capacity,
                                  int64_t* part_rows) {
  QX_CHECK(cu_q && used && part_rows && seqs >= 0 && HQ > 0 && HK > 0 && HQ % HK == 0 &&
               n_work >= 0 && (n_work == 0 || (work && slots)) && (capacity <= 0 || joins),
           "attention8_joins: arguments");
  try {
    return join_list(cu_q, used, seqs, unit > 0 ? 0 : tile_height(HQ / HK), causal,
                     unit < 0 ? -unit : unit, work, n_work, slots, joins, capacity, part_rows);
  } catch (const std::bad_alloc&) {
    set_error("attention8_joins: out of host memory");
    return QX_EINVAL;
  }
}

int64_t qx_paged_attention8_workspace(int64_t seqs, int64_t rows, int64_t max_q, int64_t max_used,
                                      int64_t HQ, int64_t HK, int64_t D, int has_work,
                                      int64_t unit) {
  QX_CHECK(seqs >= 0 && rows >= 0 && max_q >= 0 && max_used >= 0 && HQ > 0 && HK > 0 &&
               HQ % HK == 0 && (D == 64 || D == 128),
           "attention8_workspace: arguments");
  if (!has_work) unit = call_unit(seqs * max_used, max_q, max_used, HK, HQ / HK);
  if (unit < 0) unit = -unit;
  const int64_t splits = unit ? (max_used + unit - 1) / unit : 0;
  return splits > 1 ? splits * rows * HQ * (D + 2) * 4 : 0;
}

static int attention8(const void* q, int64_t q_ld, const int64_t* q_index, const void* k_pool,
                      const void* v_pool, const void* scales, const int* cu_q, const int* used,
                      const int* table, int64_t table_ld, int64_t seqs, int64_t rows,
                      int64_t max_q, int64_t max_used, int64_t HQ, int64_t HK, int64_t D,
                      int64_t page, float scale, int causal, void* out_bf16, void* out_fp8,
                      int64_t o_ld, float* out_scales, int64_t os_ld, float* lse, int64_t lse_ld,
                      const int* work, int64_t n_work, int64_t unit, const int* slots,
                      const int* joins, int64_t n_joins, int64_t part_rows, void* workspace,
                      int64_t workspace_bytes, const int64_t* positions, const void* cos_sin,
                      int cs_is_f32, const void* q_w, float eps, hipStream_t stream) {
  QX_CHECK(q && k_pool && v_pool && scales && cu_q && used && table, "attention8: null pointer");
  QX_CHECK((out_bf16 != nullptr) != (out_fp8 != nullptr), "attention8: one output, bf16 or e4m3");
  QX_CHECK(D == 64 || D == 128, "attention8: head_dim %lld", (long long)D);
  QX_CHECK(HQ > 0 && HK > 0 && HQ % HK == 0, "attention8: heads %lld/%lld", (long long)HQ,
           (long long)HK);
  QX_CHECK(page == kPage, "attention8: page of %lld tokens (the arena uses 16)", (long long)page);
  QX_CHECK(seqs >= 0 && rows >= 0 && max_q >= 0 && max_used >= 0 && max_used <= kMaxKeys,
           "attention8: %lld sequences, %lld rows, max_q %lld, max_used %lld (at most %d)",
           (long long)seqs, (long long)rows, (long long)max_q, (long long)max_used, kMaxKeys);
  QX_CHECK(!out_fp8 || (D == 128 && out_scales && os_ld >= rows && o_ld % 8 == 0),
           "attention8: the e4m3 output needs D = 128, its scales and o_ld %% 8 == 0");
  QX_CHECK(q_ld % 8 == 0 && o_ld % 8 == 0 && (!lse || lse_ld >= rows), "attention8: strides");
  QX_CHECK((((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out_bf16) & 15) == 0 &&
               ((uintptr_t)out_fp8 & 7) == 0 && ((uintptr_t)scales & 1) == 0,
           "attention8: alignment");
  QX_CHECK(!positions || (D == 128 && cos_sin && q_w && !q_index &&
                          (((uintptr_t)cos_sin | (uintptr_t)q_w) & 15) == 0),
           "attention8: q-norm on load takes D = 128, cos_sin and q_w, and no q_index");
  QX_CHECK(scale > 0.f && scale <= 3.402823466e38f, "attention8: scale %g", (double)scale);
  QX_CHECK(seqs < 65536, "attention8: %lld sequences exceed the grid", (long long)seqs);
  const int64_t G = HQ / HK, cols = 16 * few_blocks(max_q, G);
  const int64_t col_groups = (max_q * G + cols - 1) / cols;
  const int64_t per_item = unit > 0 ? HK * col_groups : HQ / tile_heads(G);  // 2^32 threads a launch
  QX_CHECK(!work || (n_work >= 0 && n_work < (1LL << 24) && n_work * per_item < (1LL << 24)),
           "attention8: %lld work items", (long long)n_work);
  QX_CHECK((work || !unit) && (unit <= 0 ? unit % kBK == 0 && unit >= -kMaxKeys
                                         : unit % 128 == 0 && unit <= kMaxChunk),
           "attention8: work items of %lld keys", (long long)unit);
  QX_CHECK(!slots || (work && n_joins >= 0 && n_joins < 65536 && (joins || n_joins == 0) &&
                      part_rows >= 0 && part_rows <= INT32_MAX && (part_rows > 0) == (n_joins > 0)),
           "attention8: %lld joins of %lld partial rows", (long long)n_joins, (long long)part_rows);
  if (seqs == 0 || max_q == 0 || rows == 0 || (work && n_work == 0)) return QX_OK;
  if (!work) unit = call_unit(seqs * max_used, max_q, max_used, HK, G);
  QX_CHECK(max_q * HQ < (1LL << 31) && (unit <= 0 || HK * col_groups < 65536),
           "attention8: %lld rows a sequence", (long long)max_q);
  const int64_t need =
      slots ? part_rows * HQ * (D + 2) * 4
            : qx_paged_attention8_workspace(seqs, rows, max_q, max_used, HQ, HK, D,
                                            work != nullptr, unit);
  QX_CHECK(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0),
           "attention8: workspace of %lld bytes, %lld needed", (long long)workspace_bytes,
           (long long)need);
  Attn8Args a{(const uint16_t*)q, q_ld, q_index, (const uint8_t*)k_pool, (const uint8_t*)v_pool,
              (const uint16_t*)scales, cu_q, used, table, table_ld, (int)max_used, (int)HQ, (int)HK,
              causal, scale * 1.4426950408889634f, (uint16_t*)out_bf16, (uint8_t*)out_fp8, o_ld,
              out_scales, os_ld, lse, lse_ld};
  a.chunk = (int)(unit < 0 ? -unit : unit);
  a.splits = unit ? (int)std::max<int64_t>(1, (max_used + a.chunk - 1) / a.chunk) : 1;
  a.tile_rows = unit > 0 ? 0 : tile_height(G);
  a.rows = slots ? part_rows : rows;
  a.part_o = (float*)workspace;
  a.part_ml = a.part_o + (slots ? part_rows : a.splits * rows) * HQ * D;
  a.slots = slots;
  a.joins = joins;
  a.n_joins = (int)n_joins;
  const QNormArgs qn{positions, cos_sin, (const uint16_t*)q_w, eps};
  if (D == 64) attention8_launch<64, 0>(a, qn, work, n_work, seqs, max_q, stream);
  else if (!positions) attention8_launch<128, 0>(a, qn, work, n_work, seqs, max_q, stream);
  else if (!cs_is_f32) attention8_launch<128, 1>(a, qn, work, n_work, seqs, max_q, stream);
  else attention8_launch<128, 2>(a, qn, work, n_work, seqs, max_q, stream);
  QX_LAUNCH_STATUS();
}

#define QX_ATTN8_FIRST                                                                            \
  q, q_ld, q_index, k_pool, v_pool, scales, cu_q, used, table, table_ld, seqs, rows, max_q,       \
      max_used, HQ, HK, D, page, scale, causal, out_bf16, out_fp8, o_ld, out_scales, os_ld, lse,  \
      lse_ld, work, n_work, unit
#define QX_ATTN8_LAST \
  workspace, workspace_bytes, positions, cos_sin, cs_is_f32, q_w, eps, stream

int qx_paged_attention8(const void* q, int64_t q_ld, const int64_t* q_index, const void* k_pool,
                        const void* v_pool, const void* scales, const int* cu_q, const int* used,
                        const int* table, int64_t table_ld, int64_t seqs, int64_t rows,
                        int64_t max_q, int64_t max_used, int64_t HQ, int64_t HK, int64_t D,
                        int64_t page, float scale, int causal, void* out_bf16, void* out_fp8,
                        int64_t o_ld, float* out_scales, int64_t os_ld, float* lse, int64_t lse_ld,
                        const int* work, int64_t n_work, int64_t unit, void* workspace,
                        int64_t workspace_bytes, const int64_t* positions, const void* cos_sin,
                        int cs_is_f32, const void* q_w, float eps, hipStream_t stream) {
  return attention8(QX_ATTN8_FIRST, nullptr, nullptr, 0, 0, QX_ATTN8_LAST);
}

int qx_paged_attention8_joined(
    const void* q, int64_t q_ld, const int64_t* q_index, const void* k_pool, const void* v_pool,
    const void* scales, const int* cu_q, const int* used, const int* table, int64_t table_ld,
    int64_t seqs, int64_t rows, int64_t max_q, int64_t max_used, int64_t HQ, int64_t HK, int64_t D,
    int64_t page, float scale, int causal, void* out_bf16, void* out_fp8, int64_t o_ld,
    float* out_scales, int64_t os_ld, float* lse, int64_t lse_ld, const int* work, int64_t n_work,
    int64_t unit, const int* slots, const int* joins, int64_t n_joins, int64_t part_rows,
    void* workspace, int64_t workspace_bytes, const int64_t* positions, const void* cos_sin,
    int cs_is_f32, const void* q_w, float eps, hipStream_t stream) {
  QX_CHECK(work && slots, "attention8_joined: null pointer");
  return attention8(QX_ATTN8_FIRST, slots, joins, n_joins, part_rows, QX_ATTN8_LAST);
}
#undef QX_ATTN8_FIRST
#undef QX_ATTN8_LAST

}  // extern "C"
