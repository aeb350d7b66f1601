// Attention over the 4-bit paged KV cache for up to a few dozen query rows per
// KV head: decode steps (with the step's append, RoPE and sliding windows) and
// speculative verification.
//
//   o_j = sum_t p_jt v_t / sum_t p_jt,  p_jt = 2^(x_jt - m_j),
//   x_jt = scale log2(e) q_j . k_t,  k_t, v_t = s c + b per group of 64 dims
//
// in one pass over the blocks with a running reference m, so a block's bytes go
// from HBM to registers once and nothing is dequantized:
//   x = sum_g s'_g (q . (c - 8))_g + sum_g z'_g sum_g q,   s' = s scale log2(e), z' = (b + 8 s) scale log2(e)
//   o = sum_g [ sum_t (p_t s_tg) (c_t - 8) + sum_t p_t (b_tg + 8 s_tg) ]
// Codes become matrix operands in one or two instructions per pair, from words
// loaded in the operands' order (kdev4.hpp): one wave holds 16
// rows (query positions x heads of the KV group) in the columns of
// v_mfma_f32_16x16x32_f16, K tiles of 16 tokens and V tiles of 16 dims in its
// rows; the tiles S^T = K . Q^T leave a lane four tokens of one row, which is
// where O^T += V^T . P^T wants them, so P stays in registers.
//
// Numerics: queries are scaled by a power of two and held in fp16 (exact for bf16
// and fp16 inputs down to 2^-25 of the row's largest; the power is the wave's,
// taken into s' and z', unless its rows differ by more than 2^10), sums and the
// softmax in fp32.  A weight p s enters the product as an fp16 high part and the
// fp16 rounding of the rest (2^-22 of it); bf16 outputs, whose half step is 2^-9,
// take the high part alone (2^-12).
//
// head_dim above 128: a workgroup of D/128 waves, each 128 dims of K and V (the
// registers of one wave hold no more); their parts of the scores meet in LDS, one
// barrier a block, and every wave runs the same softmax on the same sums.
//
// Work split: the flat order of the int8 kernels -- per (KV head, row group) the
// blocks of all sequences end to end, the same number to every wave -- and their
// merge of partial results.
//
// Bound, measured with the step's append, RoPE and merge (head_dim, Hq / Hkv):
//   few long contexts, 8 x 98304-131072 tokens (128, 32 / 4): the cache's reads,
//     528 MB in 101 us, 5.2 TB/s (a large copy moves 4.8);
//   32 x 512-8192 tokens (128, 40 / 8): 45.7 us for 161 MB; 38 us are this kernel,
//     of them 5 before the first block is in and 10 while the last waves end;
//   16 x 8 new rows on 1024-8192 tokens (128, 32 / 8): 41 us; conversion and
//     softmax on the VALU, each unpacked operand feeds only two products;
//   32 x 512-4096 tokens (512, 16 / 2): 45.7 us for 87 MB; the exchange of the
//     scores' parts, a barrier a block, with one wave a SIMD;
//   one sequence of 512 tokens (64, 32 / 8): 16 us, launches and the host.
// Code runs once per call over tens of blocks, and an instruction costs about
// 5.5 ns the first time it is fetched against 2 later: loops stay rolled where
// they could be unrolled.  Three waves a SIMD spill: 61 us against 46 (the second
// line above).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_common.hpp"
#include "kdev4.hpp"

namespace krill {

namespace {

// Waves per workgroup, each a slice of the dims.
template <int D>
constexpr int q4_slices() { return D > 128 ? D / 128 : 1; }

// LDS of one wave (DW dims, G groups): the block's scales [group][token] (V: zero
// where the token is not the sequence's; groups of the bias products that do not
// exist: zero), the codes and words of the step's new token.
template <int DW>
struct Q4Lds {
  static constexpr int G = DW / 64;
  __attribute__((aligned(16))) float ks[64 * G];  // s'
  __attribute__((aligned(16))) float kz[64 * 4];  // z'
  __attribute__((aligned(16))) float vs[64 * G];
  __attribute__((aligned(16))) float vz[64 * G];  // b + 8 s
  __attribute__((aligned(16))) uint8_t newk[DW], newv[DW];  // a code per byte
  uint32_t newkm[G], newvm[G];
};

__device__ __forceinline__ float4_t mfma16x16x4f32(float a, float b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// Two weights as fp16, and the fp16 rounding of what that leaves; the empty asm
// keeps the conversions packed and the rest one mixed multiply-add (`one` is 1.0
// where the compiler cannot see it).
__device__ __forceinline__ uint32_t round2(float &w0, float &w1) {
  asm("" : "+v"(w0), "+v"(w1));
  uint32_t u = h2_as_u32(half2_t{(_Float16)w0, (_Float16)w1});
  asm("" : "+v"(u));
  return u;
}
__device__ __forceinline__ uint32_t rest2(float w0, float w1, uint32_t h, float one) {
  const half2_t hh = u32_as_h2(h);
  float r0 = __builtin_fmaf(w0, one, -(float)hh[0]), r1 = __builtin_fmaf(w1, one, -(float)hh[1]);
  asm("" : "+v"(r0), "+v"(r1));
  return h2_as_u32(half2_t{(_Float16)r0, (_Float16)r1});
}

// LDS of one wave: its operations complete in order, waiting for them orders its
// lanes' writes before other lanes' reads.
__device__ __forceinline__ void wave_sync() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ uint32_t word_of(const uint4 &v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; }
__device__ __forceinline__ void set_word(uint4 &v, int w, uint32_t x) {
  (w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w) = x;
}
__device__ __forceinline__ float lo_f32(uint32_t w) { return f16_bits_to_f32((uint16_t)(w & 0xffffu)); }
__device__ __forceinline__ float hi_f32(uint32_t w) { return f16_bits_to_f32((uint16_t)(w >> 16)); }

// A raised reference lies kGap below the row's maximum, and is raised when a
// score exceeds it by kOver: p < 2^8, and p s_v is finite in fp16 for |s_v| <=
// kBig.  A block with a larger scale raises it to the maximum itself (p <= 1;
// the quantizer's scales are below 8740).
constexpr float kGap = 5.0f, kOver = 8.0f, kBig = 255.0f;

constexpr int kSeqWaves = 8, kSeqRows = 8;

// Waves per SIMD the registers are budgeted for.  Two row tiles at two waves spill
// (16 x 8 new rows: 46.6 us as two row groups of one tile at two waves a SIMD, 40.8
// as two tiles at one).
template <int D, int NRT, bool SEQ>
constexpr int q4_waves() { return NRT == 1 ? 2 : 1; }

}  // namespace

// NRT: tiles of 16 query rows per wave.  WIN: sliding window.  LOW: the weights'
// low parts too.  SEQ: instead of the flat split a workgroup of kSeqWaves waves
// per (sequence, KV head), each a share of its blocks, their partial results
// combined in LDS (at most kSeqRows query rows, head_dim up to 128).
template <int D, int NRT, bool WIN, bool LOW, bool SEQ>
__global__ __launch_bounds__(64 * (SEQ ? kSeqWaves : q4_slices<D>()), (q4_waves<D, NRT, SEQ>())) void k_attn_q4(AttnArgs a) {
  static_assert(!SEQ || (NRT == 1 && D <= 128), "one slice, one row tile");
  constexpr int DS = q4_slices<D>(), DW = D / DS;
  constexpr int GD = D / 64;    // groups of a row
  constexpr int G = DW / 64;    // of the wave's slice
  constexpr int NP = DW / 32;   // 16-byte pieces per lane of K, and of V
  constexpr int NDT = DW / 16;  // 16-dim tiles of the output
  constexpr int RR = 16 * NRT;
  constexpr int E = DW / 64;
  __shared__ Q4Lds<DW> lds_all[SEQ ? kSeqWaves : DS];
  // the slices' parts of the scores, two buffers; whether a slice has a large V scale
  __shared__ __attribute__((aligned(16))) float4_t part[DS > 1 ? 2 : 1][DS][DS > 1 ? 4 * NRT * 64 : 1];
  __shared__ int part_big[2][DS];
  // SEQ: each wave's partial, rows of o (padded by four banks), (m, l)
  __shared__ __attribute__((aligned(16))) float seq_o[SEQ ? kSeqWaves : 1][SEQ ? kSeqRows * (D + 4) : 4];
  __shared__ float2 seq_ml[SEQ ? kSeqWaves : 1][kSeqRows];

  const int lane = threadIdx.x & 63, n = lane & 15, q4 = lane >> 4;
  const int sl = DS > 1 ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) : 0;  // the wave's slice
  const int wid = SEQ ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) : 0;
  Q4Lds<DW> &lds = lds_all[SEQ ? wid : sl];
  const int hk = blockIdx.y, rg = blockIdx.z;
  // (range w of the heads goes to different XCDs)
  const int wv = (int)((blockIdx.x + (unsigned)hk) % gridDim.x);
  const int rbase = rg * RR;
  // the lane's rows: query position and head of the KV group (divided by way of
  // floats, put right by at most one: while the lengths are on their way)
  int rj[NRT], rh[NRT];
  bool rvalid[NRT];
  const int j_first = rbase / a.R, j_last = (min(a.NR, rbase + RR) - 1) / a.R;
#pragma unroll
  for (int rt = 0; rt < NRT; ++rt) {
    const int r = rbase + 16 * rt + n;
    rvalid[rt] = r < a.NR;
    int j = (int)((float)r * __builtin_amdgcn_rcpf((float)a.R)), h = r - j * a.R;
    if (h < 0) h += a.R, --j;
    if (h >= a.R) h -= a.R, ++j;
    rj[rt] = rvalid[rt] ? j : 0;
    rh[rt] = rvalid[rt] ? h : 0;
  }

  // ---- flat blocks [i0, iend) of the (head, row group) order
  int c0 = 0, lenv = 0, i0 = 0, iend = 0;
  int b = -1, s = 0;  // the sequence of block i0, the flat index of its first block
  if constexpr (SEQ) {
    // (blocks counted from the sequence's first)
    b = c0 = (int)blockIdx.x;
    lenv = seq_len_view<WIN>(a, b);
    const int nb = seq_blocks_rg(a, lenv, rg);
    i0 = (wid * nb + kSeqWaves - 1) / kSeqWaves;
    iend = ((wid + 1) * nb + kSeqWaves - 1) / kSeqWaves;
  } else {
    lenv = lane < a.B ? seq_len_view<WIN>(a, lane) : 0;
    int nbv = seq_blocks_rg(a, lenv, rg);
    int incl = wave_incl_scan(nbv);
    int T = __builtin_amdgcn_readlane(incl, 63);
    for (int cc = 64; cc < a.B; cc += 64) {
      const int bb = cc + lane;
      T += __builtin_amdgcn_readfirstlane(wave_allsum_int(bb < a.B ? seq_blocks_rg(a, seq_len_view<WIN>(a, bb), rg) : 0));
    }
    // (every wave that takes part holds a block: the merge relies on it)
    const int Wt = min(a.waves, T);
    if (wv >= Wt) return;
    i0 = __builtin_amdgcn_readfirstlane((int)(((int64_t)wv * T + Wt - 1) / Wt));
    iend = __builtin_amdgcn_readfirstlane((int)(((int64_t)(wv + 1) * T + Wt - 1) / Wt));
    {
      int carry = 0;
      for (c0 = 0; c0 < a.B; c0 += 64) {
        if (c0 > 0) {
          const int bb = c0 + lane;
          lenv = bb < a.B ? seq_len_view<WIN>(a, bb) : 0;
          nbv = seq_blocks_rg(a, lenv, rg);
          incl = wave_incl_scan(nbv) + carry;
        }
        const unsigned long long m = __ballot(c0 + lane < a.B && incl > i0);
        if (m) {
          const int l = __builtin_ctzll(m);
          b = c0 + l;
          s = __builtin_amdgcn_readlane(incl - nbv, l);
          break;
        }
        carry = __builtin_amdgcn_readlane(incl, 63);
      }
    }
    if (b < 0) return;
  }
  auto seq_len = [&](int bs) -> int { return bs - c0 < 64 ? __builtin_amdgcn_readlane(lenv, bs - c0) : seq_len_view<WIN>(a, bs); };

  // block-table entries of flat blocks tab0 .. tab0 + 63, one a lane (-1: none
  // of the pool's); reloaded every 64 blocks, walking on from sequence b
  int tab = -1, tab0 = i0;
  auto load_table = [&](int from) {
    const int f = from + lane;
    int bs = b, ss = s;
    tab = -1;
    while (bs < a.B && ss < min(iend, from + 64)) {
      const int nbs = seq_blocks_rg(a, seq_len(bs), rg);
      if (f < iend && f >= ss && f < ss + nbs) {
        const int phys = a.tables[(int64_t)bs * a.max_blocks + table_offset<WIN>(a, bs) + (f - ss)];
        tab = (unsigned)phys < (unsigned)a.lv.num_blocks ? phys : -1;
      }
      ss += nbs;
      ++bs;
    }
    tab0 = from;
  };
  load_table(i0);

  // ---- a block in registers; blocks past the range and outside the pool read as
  // zeros without touching memory
  uint4 kq[NP], vq[NP];
  uint32_t mk[G], mv[G];  // words of token `lane`
  auto rsrc_of = [&](int i) -> __amdgpu_buffer_rsrc_t {
    const int phys = __builtin_amdgcn_readlane(tab, __builtin_amdgcn_readfirstlane((i - tab0) & 63));
    const bool ok = i < iend && phys >= 0;
    return block_rsrc(head_region(a.lv, ok ? phys : 0, hk), ok ? a.lv.head_bytes : 0);
  };
  auto ld16 = [](__amdgpu_buffer_rsrc_t r, int off) {
    return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 2));
  };
  auto ld_words = [](__amdgpu_buffer_rsrc_t r, int off, uint32_t (&w)[G]) {
    if constexpr (G == 1) {
      w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 2);
    } else {
      static_assert(G == 2, "one or two groups a slice");
      const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 2);
      w[0] = v[0];
      w[1] = v[1];
    }
  };
  auto load_k = [&](__amdgpu_buffer_rsrc_t r) {
#pragma unroll
    // (a slice's pieces: one per 16-token group; head_dim 64: one per two of them)
    for (int p = 0; p < NP; ++p) kq[p] = ld16(r, (p * DS + sl) * 1024 + lane * 16);
    ld_words(r, q4_km_offset(D) + (lane * GD + sl * G) * 4, mk);
    ld_words(r, q4_vm_offset(D) + (lane * GD + sl * G) * 4, mv);
  };
  auto load_v = [&](__amdgpu_buffer_rsrc_t r) {
#pragma unroll
    for (int p = 0; p < NP; ++p) vq[p] = ld16(r, q4_v_offset(D) + (sl * NP + p) * 1024 + lane * 16);
  };

  // ---- queries: lane (n, q4) holds dims 64 g + 16 q4 + 8 h .. +7 of the slice of
  // row n in qB[..][2 g + h]
  half8_t qB[NRT][2 * G];
  float qz[NRT];       // the row's sum over group q4 (0 past the groups)
  float rd[NRT];       // what the row's scores take (1, but where exponents differ)
  float nmf[NRT];      // and its inverse, which the running reference takes
  float ksf = 1.0f;    // what s and b of K take
  bool any_rd = false;
  float qoff[LOW ? 1 : NRT][G];  // !LOW: what the codes' offsets add to a group's products
  // ---- the step's new token, where this range holds the sequence's last block:
  // quantized into LDS, patched into the registers when its block comes up,
  // stored by row group 0 at the segment's end
  uint16_t rk[E], rv[E], rk2[E];  // rk2: the dims that rk's turn with
  int patch_i = -1, patch_t = 0;
  auto owns_new = [&](int bs, int ss) -> bool {
    if (!a.k_new) return false;
    const int len = seq_len(bs), nb = seq_blocks_rg(a, len, rg);
    return nb > 0 && i0 < iend && ss + nb <= iend && ((len - 1) >> 6) == nb - 1;
  };
  const int d0 = sl * DW + lane * E;  // the lane's dims of the new rows
  auto load_new = [&](int bs) {
    const int64_t off = (int64_t)bs * a.kn_sb + (int64_t)hk * a.kn_sh;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      rk[e] = a.k_new[off + d0 + e];
      rv[e] = a.v_new[off + d0 + e];
      if (a.rope_cs) rk2[e] = a.k_new[off + (d0 ^ (D / 2)) + e];
    }
  };
  auto quantize_new = [&](int bs, int ss, auto dtype) {
    constexpr int DT = decltype(dtype)::value;
    const int len = seq_len(bs);
    float x[E];
    uint32_t code[E];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = elem_to_f32<DT>(kv ? rv[e] : rk[e]);
      if (kv == 0 && a.rope_cs) {
        const float *crow = rope_row(a, (WIN ? len_of(a, bs) : len) - 1, D) + (d0 & (D / 2 - 1));
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float c = crow[e], sn = crow[D / 2 + e], y = elem_to_f32<DT>(rk2[e]);
          x[e] = round_dt<DT>(d0 >= D / 2 ? y * sn + x[e] * c : x[e] * c - y * sn);
        }
      }
      const uint32_t meta = q4_quantize_row<DW, DT>(x, code);
#pragma unroll
      for (int e = 0; e < E; ++e) (kv ? lds.newv : lds.newk)[lane * E + e] = (uint8_t)code[e];
      if ((lane * E) % 64 == 0) (kv ? lds.newvm : lds.newkm)[lane * E / 64] = meta;
    }
    wave_sync();
    patch_i = ss + seq_blocks_rg(a, len, rg) - 1;
    patch_t = (len - 1) & 63;
  };
  auto prepare_new = [&](int bs, int ss) {
    if (a.q_dtype == DT_BF16)
      quantize_new(bs, ss, std::integral_constant<int, DT_BF16>{});
    else
      quantize_new(bs, ss, std::integral_constant<int, DT_F16>{});
  };
  // the K word of the new token's dims 8 x .. 8 x + 7 of the slice, and its V byte m
  auto new_k_word = [&](int x) -> uint32_t {
    const uint2 c = *reinterpret_cast<const uint2 *>(lds.newk + 8 * x);
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) w |= (((e < 4 ? c.x : c.y) >> (8 * (e & 3))) & 15u) << (4 * q4_nibble(e));
    return w;
  };
  auto new_v_byte = [&](int m) -> uint32_t {
    const int d = 32 * (m >> 4) + (m & 15);
    return (uint32_t)lds.newv[d] | ((uint32_t)lds.newv[d + 16] << 4);
  };
  auto patch = [&]() {
    const int t = patch_t;
    const bool mine = n == (t & 15);
#pragma unroll
    for (int tg = 0; tg < 4; ++tg)
      if ((t >> 4) == tg) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int p = DW == 64 ? tg >> 1 : tg;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w = new_k_word(8 * g + 2 * q4 + h);
            const int k = (DW == 64 ? (tg & 1) : g) * 2 + h;
            set_word(kq[p], k, mine ? w : word_of(kq[p], k));
          }
        }
      }
    const int slot = q4_v_slot(t);
    const bool mine_v = q4 == ((t >> 2) & 3);
    const uint32_t keep = ~(0xffu << (8 * (slot & 3)));
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const uint32_t nv = new_v_byte(16 * p + n) << (8 * (slot & 3));
#pragma unroll
      for (int w = 0; w < 4; ++w)
        if ((slot >> 2) == w) set_word(vq[p], w, mine_v ? (word_of(vq[p], w) & keep) | nv : word_of(vq[p], w));
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      mk[g] = lane == t ? lds.newkm[g] : mk[g];
      mv[g] = lane == t ? lds.newvm[g] : mv[g];
    }
  };
  auto store_new = [&](int phys) {
    uint8_t *reg = head_region(a.lv, phys, hk);
    if (lane < DW / 8) *reinterpret_cast<uint32_t *>(reg + q4_k_word(D, patch_t, sl * (DW / 8) + lane)) = new_k_word(lane);
    if (lane < DW / 2) reg[q4_v_byte(D, patch_t, sl * (DW / 2) + lane)] = (uint8_t)new_v_byte(lane);
    if (lane < G) {
      const int at = (patch_t * GD + sl * G + lane) * 4;
      *reinterpret_cast<uint32_t *>(reg + q4_km_offset(D) + at) = lds.newkm[lane];
      *reinterpret_cast<uint32_t *>(reg + q4_vm_offset(D) + at) = lds.newvm[lane];
    }
  };

#pragma unroll
  for (int g = G; g < 4; ++g) lds.kz[64 * g + lane] = 0.0f;
  float one = 1.0f;
  asm volatile("" : "+v"(one));
  const uint32_t magic = q4_magic();
  int i = i0;
  // ---- a segment's queries as they come, those that they turn with (another
  // slice's), its new token: ahead of the range's first block, later ahead of the
  // segment before's results
  constexpr int HALF = DW == D ? 0 : DS / 2;  // slices to the dims that turn together
  uint4 raw[NRT][2 * G], raw2[NRT][2 * G];
  const uint16_t *qp[NRT];
  bool own = false;
  auto q_piece = [&](int rt, int slice, int k) -> uint4 {
    return *reinterpret_cast<const uint4 *>(qp[rt] + slice * DW + 64 * (k >> 1) + 8 * (k & 1));
  };
  auto issue_q = [&](int bs, int ss) {
    own = owns_new(bs, ss);
    if (own) load_new(bs);
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      qp[rt] = q_row(a, bs, hk * a.R + rh[rt], rj[rt]) + 16 * q4;
#pragma unroll
      for (int k = 0; k < 2 * G; ++k) {
        raw[rt][k] = q_piece(rt, sl, k);
        raw2[rt][k] = uint4{0u, 0u, 0u, 0u};
        if (HALF && a.rope_cs) raw2[rt][k] = q_piece(rt, sl ^ HALF, k);
      }
    }
  };
  if (!SEQ || i0 < iend) {
    issue_q(b, s);
    const __amdgpu_buffer_rsrc_t r = rsrc_of(i0);
    load_k(r);
    load_v(r);
  }
  while (!SEQ || i0 < iend) {
    float mxr[NRT], mxw = 0.0f;
    // (of the largest |q| the bits: both halves of each word at once)
    auto largest = [&](const uint4 &v, ushort2_t m) -> ushort2_t {
#pragma unroll
      for (int w = 0; w < 4; ++w)
        m = __builtin_elementwise_max(m, __builtin_bit_cast(ushort2_t, word_of(v, w) & 0x7fff7fffu));
      return m;
    };
    if (own) prepare_new(b, s);
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      ushort2_t m2 = ushort2_t{0, 0};
#pragma unroll
      for (int k = 0; k < 2 * G; ++k) m2 = largest(raw[rt][k], m2);
#pragma unroll
      for (int o = 1; o < DS; ++o)
#pragma unroll
        for (int k = 0; k < 2 * G; ++k) m2 = largest(q_piece(rt, (sl + o) % DS, k), m2);
      int mb = max((int)m2[0], (int)m2[1]);
      mb = max(mb, __shfl_xor(mb, 16, 64));
      mb = max(mb, __shfl_xor(mb, 32, 64));
      const float mx = a.q_dtype == DT_BF16 ? bf16_bits_to_f32((uint16_t)mb) : f16_bits_to_f32((uint16_t)mb);
      mxr[rt] = rvalid[rt] && mx < INFINITY ? mx : 0.0f;
      mxw = fmaxf(mxw, mxr[rt]);
      if (a.rope_cs) {
        // dims d and d + D/2 turn together: in another slice's piece, this lane's
        // operand (head_dim 128) or lane ^ 32's (64)
        const int len = WIN ? len_of(a, b) : seq_len(b);  // absolute positions
        const float *crow = rope_row(a, len - a.Lq + rj[rt], D);
        uint4 old[2 * G];
#pragma unroll
        for (int k = 0; k < 2 * G; ++k) old[k] = raw[rt][k];
#pragma unroll
        for (int k = 0; k < 2 * G; ++k) {
          const int d = sl * DW + 64 * (k >> 1) + 16 * q4 + 8 * (k & 1);
          const bool up = d >= D / 2;
          const float *cp = crow + (d & (D / 2 - 1));
          uint32_t x[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t own_w = word_of(old[k], w);
            const uint32_t other = HALF        ? word_of(raw2[rt][k], w)
                                   : DW == 128 ? word_of(old[(k + G) % (2 * G)], w)
                                               : (uint32_t)__shfl_xor((int)own_w, 32, 64);
            const float2 c2 = *reinterpret_cast<const float2 *>(cp + 2 * w);
            const float2 s2 = *reinterpret_cast<const float2 *>(cp + D / 2 + 2 * w);
            uint32_t lo = up ? other : own_w, hi = up ? own_w : other;
            if (a.q_dtype == DT_BF16)
              rope_pair_words<DT_BF16>(lo, hi, c2, s2);
            else
              rope_pair_words<DT_F16>(lo, hi, c2, s2);
            x[w] = up ? hi : lo;
          }
          raw[rt][k] = uint4{x[0], x[1], x[2], x[3]};
        }
      }
    }
    // a row whose largest |q| is mx scaled by 2^e has it in [2^14, 2^15) (a turn may
    // take it a factor sqrt 2 higher: [2^13, 2^14))
    auto exponent = [&](float mx) -> int {
      const int ex = (int)(__builtin_bit_cast(uint32_t, mx) >> 23);
      return mx > 0.0f && ex < 255 ? min((a.rope_cs ? 140 : 141) - ex, 100) : 0;
    };
    // (where the wave's largest |q| passes some 2^90 its scores are taken some
    // powers of two too small, so that nothing overflows: scores that differ do so
    // by far more than the softmax resolves either way)
    const int ew = exponent(row_allmax(mxw));
    const int es = (int)((__builtin_bit_cast(uint32_t, a.scale_log2) >> 23) & 0xffu) - 127;
    const int cw = min(-ew, 100 - es);
    ksf = ldexpf(a.scale_log2, cw);
    bool differ = false;
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      int er = ew;
      rd[rt] = nmf[rt] = 1.0f;
      if (mxr[rt] > 0.0f && exponent(mxr[rt]) > ew + 10) {
        er = exponent(mxr[rt]);
        rd[rt] = ldexpf(1.0f, max(-er - cw, -126));
        nmf[rt] = 1.0f / rd[rt];
        differ = true;
      }
      float qsum[G];
      // !LOW: the codes come as 1024 + c and 1024 + 16 c, so pairs 1 and 3 are held
      // over 16, and what is too much is where the products start from
      const float f0 = rvalid[rt] ? ldexpf(1.0f, er) : 0.0f, f1 = LOW ? f0 : f0 * 0.0625f;
      auto convert = [&](auto dtype) {
        constexpr int DT = decltype(dtype)::value;
        const half2_t one2 = half2_t{(_Float16)1.0f, (_Float16)1.0f};
        const half2_t sixteen2 = half2_t{(_Float16)16.0f, (_Float16)16.0f};
        const half2_t off2 = half2_t{(_Float16)-1024.0f, (_Float16)-1024.0f};
#pragma unroll
        for (int k = 0; k < 2 * G; ++k) {
          if ((k & 1) == 0) {
            qsum[k >> 1] = 0.0f;
            if constexpr (!LOW) qoff[rt][k >> 1] = 0.0f;
          }
          uint32_t h4[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t u = word_of(raw[rt][k], w);
            const float f = (w & 1) ? f1 : f0;
            const half2_t h = half2_t{(_Float16)(elem_to_f32<DT>((uint16_t)(u & 0xffffu)) * f),
                                      (_Float16)(elem_to_f32<DT>((uint16_t)(u >> 16)) * f)};
            qsum[k >> 1] = dot2(h, !LOW && (w & 1) ? sixteen2 : one2, qsum[k >> 1]);
            if constexpr (!LOW) qoff[rt][k >> 1] = dot2(h, off2, qoff[rt][k >> 1]);
            h4[w] = h2_as_u32(h);
          }
          qB[rt][k] = __builtin_bit_cast(half8_t, uint4{h4[0], h4[1], h4[2], h4[3]});
        }
      };
      if (a.q_dtype == DT_BF16)
        convert(std::integral_constant<int, DT_BF16>{});
      else
        convert(std::integral_constant<int, DT_F16>{});
#pragma unroll
      for (int g = 0; g < G; ++g) {
        qsum[g] += shfl_xor(qsum[g], 16);
        qsum[g] += shfl_xor(qsum[g], 32);
        if constexpr (!LOW) {
          qoff[rt][g] += shfl_xor(qoff[rt][g], 16);
          qoff[rt][g] += shfl_xor(qoff[rt][g], 32);
        }
      }
      qz[rt] = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) qz[rt] = q4 == g ? qsum[g] : qz[rt];
    }
    any_rd = __any(differ);

    const int len = seq_len(b);
    const int e = s + seq_blocks_rg(a, len, rg);
    const int seg_end = __builtin_amdgcn_readfirstlane(min(e, iend));
    int lim[NRT], lo[NRT], wst = 0, lo_hi = 0;
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      lim[rt] = rvalid[rt] ? key_limit(a, len, rj[rt]) : 0;
      lo[rt] = 0;
    }
    const int lim_lo = key_limit(a, len, j_first);  // keys seen by the wave's first row
    if constexpr (WIN) {
      wst = win_view_start(a, b);
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt) lo[rt] = max(wst, len - a.Lq + rj[rt] - a.window + 1);
      lo_hi = max(wst, len - a.Lq + j_last - a.window + 1);
    }
    float m_run[NRT], nm[NRT], l_part[NRT], c_part[NRT][G];
    float4_t o[NRT][NDT];
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      m_run[rt] = -INFINITY;
      nm[rt] = 0.0f;
      l_part[rt] = 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) c_part[rt][g] = 0.0f;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[rt][dt] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int new_phys = -1;

    for (; i < seg_end; ++i) {
      const int tbase = (i - s) << 6;
      if (i == patch_i) {
        patch();
        new_phys = __builtin_amdgcn_readlane(tab, __builtin_amdgcn_readfirstlane((i - tab0) & 63));
      }
      // ---- metadata to LDS
      bool data = tbase + lane < len;
      if constexpr (WIN) data = data && tbase + lane >= wst;
      bool large = false;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float ks = lo_f32(mk[g]) * ksf;
        lds.ks[64 * g + lane] = ks;
        lds.kz[64 * g + lane] = __builtin_fmaf(hi_f32(mk[g]), ksf, LOW ? 8.0f * ks : 0.0f);
        const uint32_t w = data ? mv[g] : 0u;
        lds.vs[64 * g + lane] = lo_f32(w);
        lds.vz[64 * g + lane] = __builtin_fmaf(8.0f, lo_f32(w), hi_f32(w));
        large |= lo_f32(w) > kBig;
      }
      bool big = __any(large);
      wave_sync();

      // ---- S^T tiles of 16 tokens: lane holds tokens 16 tg + 4 q4 + x of row n,
      // relative to the running reference
      float4_t sc[4][NRT];
#pragma unroll
      for (int tg = 0; tg < 4; ++tg) {
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt) {
          const float st = DS == 1 || sl == 0 ? nm[rt] : 0.0f;
          sc[tg][rt] = mfma16x16x4f32(lds.kz[64 * q4 + 16 * tg + n], qz[rt], float4_t{st, st, st, st});
        }
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float4_t ks = *reinterpret_cast<const float4_t *>(lds.ks + 64 * g + 16 * tg + 4 * q4);
          float4_t acc[NRT];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t w = word_of(kq[DW == 64 ? tg >> 1 : tg], (DW == 64 ? (tg & 1) : g) * 2 + h);
            const half8_t A = LOW ? q4_k_operand(w, magic) : q4_k_operand_raw(w, magic);
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt)
              {
                const float st = LOW ? 0.0f : qoff[LOW ? 0 : rt][g];
                acc[rt] = mfma16x16x32(A, qB[rt][2 * g + h], h == 0 ? float4_t{st, st, st, st} : acc[rt]);
              }
          }
#pragma unroll
          for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[tg][rt][x] = __builtin_fmaf(ks[x], acc[rt][x], sc[tg][rt][x]);
        }
      }
      if constexpr (DS > 1) {
        // the slices' parts: every wave adds them in the same order
        float4_t(*const mine)[DS > 1 ? 4 * NRT * 64 : 1] = part[i & 1];
#pragma unroll
        for (int k = 0; k < 4 * NRT; ++k) mine[sl][64 * k + lane] = sc[k / NRT][k % NRT];
        if (lane == 0) part_big[i & 1][sl] = big;
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
        for (int k = 0; k < 4 * NRT; ++k) {
          float4_t v = mine[0][64 * k + lane];
#pragma unroll
          for (int o = 1; o < DS; ++o) v += mine[o][64 * k + lane];
          sc[k / NRT][k % NRT] = v;
        }
#pragma unroll
        for (int o = 0; o < DS; ++o) big = big || part_big[i & 1][o] != 0;
        big = __any(big);
      }
      if (any_rd) {
        asm volatile("; rows of other exponents");  // (a branch, not a multiplication by one)
#pragma unroll
        for (int tg = 0; tg < 4; ++tg)
#pragma unroll
          for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
            for (int x = 0; x < 4; ++x) sc[tg][rt][x] *= rd[rt];
      }
      if (i + 1 < iend && i + 1 - tab0 == 64) load_table(i + 1);
      const __amdgpu_buffer_rsrc_t rn = rsrc_of(i + 1);
      load_k(rn);

      bool edge = tbase + 64 > lim_lo;
      if constexpr (WIN) edge = edge || tbase < lo_hi;
      if (edge) {
#pragma unroll
        for (int tg = 0; tg < 4; ++tg)
#pragma unroll
          for (int rt = 0; rt < NRT; ++rt)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int tok = tbase + 16 * tg + 4 * q4 + x;
              if (tok >= lim[rt] || (WIN && tok < lo[rt])) sc[tg][rt][x] = -INFINITY;
            }
      }

      // ---- the reference moves only when some score exceeds it by more than kOver
      const float over_by = big ? 0.0f : kOver, gap = big ? 0.0f : kGap;
      float mb[NRT];
      bool over = false;
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt) {
        float v = fmaxf(sc[0][rt][0], sc[0][rt][1]);
#pragma unroll
        for (int k = 2; k < 16; k += 2) v = fmaxf(fmaxf(v, sc[k / 4][rt][k % 4]), sc[k / 4][rt][k % 4 + 1]);
        mb[rt] = v;
        over |= v > (m_run[rt] == -INFINITY ? -INFINITY : over_by);
      }
      if (__any(over)) {
#pragma unroll
        for (int rt = 0; rt < NRT; ++rt) {
          const float v = swap32_max(swap16_max(mb[rt]));  // the row's, over its four lanes
          const float mu = m_run[rt] == -INFINITY ? 0.0f : m_run[rt];
          const float mn = fmaxf(m_run[rt], v + mu - gap);
          const float al = m_run[rt] == -INFINITY ? 0.0f : fast_exp2(m_run[rt] - mn);
          const float dn = mn == -INFINITY ? 0.0f : mn - mu;
#pragma unroll
          for (int tg = 0; tg < 4; ++tg)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const float y = sc[tg][rt][x] - dn;
              sc[tg][rt][x] = y > gap ? gap : y;  // (keeps a NaN)
            }
          m_run[rt] = mn;
          nm[rt] = mn == -INFINITY ? 0.0f : -mn * nmf[rt];
          l_part[rt] *= al;
#pragma unroll
          for (int g = 0; g < G; ++g) c_part[rt][g] *= al;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) o[rt][dt] *= al;
        }
      }
#pragma unroll
      for (int rt = 0; rt < NRT; ++rt) {
        float sum = 0.0f;
#pragma unroll
        for (int tg = 0; tg < 4; ++tg)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            sc[tg][rt][x] = fast_exp2(sc[tg][rt][x]);
            sum += sc[tg][rt][x];
          }
        l_part[rt] += sum;
      }

      // ---- O^T += V^T . P^T: contraction slot 8 q4 + k is token 32 ks + 4 q4 + k
      // (k < 4) or 32 ks + 16 + 4 q4 + k - 4
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int at = 64 * g + 32 * ks + 4 * q4;
          const float4_t vs[2] = {*reinterpret_cast<const float4_t *>(lds.vs + at),
                                  *reinterpret_cast<const float4_t *>(lds.vs + at + 16)};
          const float4_t vz[2] = {*reinterpret_cast<const float4_t *>(lds.vz + at),
                                  *reinterpret_cast<const float4_t *>(lds.vz + at + 16)};
          half8_t Bh[NRT], Bl[NRT];
#pragma unroll
          for (int rt = 0; rt < NRT; ++rt) {
            uint32_t bh[4], bl[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int k = 0; k < 8; k += 2) {
              const float4_t &p = sc[2 * ks + (k >> 2)][rt];
              const int x = k & 3;
              c_part[rt][g] = __builtin_fmaf(p[x], vz[k >> 2][x], c_part[rt][g]);
              c_part[rt][g] = __builtin_fmaf(p[x + 1], vz[k >> 2][x + 1], c_part[rt][g]);
              float w0 = p[x] * vs[k >> 2][x], w1 = p[x + 1] * vs[k >> 2][x + 1];
              bh[k / 2] = round2(w0, w1);
              if constexpr (LOW) bl[k / 2] = rest2(w0, w1, bh[k / 2], one);
            }
            Bh[rt] = __builtin_bit_cast(half8_t, uint4{bh[0], bh[1], bh[2], bh[3]});
            if constexpr (LOW) Bl[rt] = __builtin_bit_cast(half8_t, uint4{bl[0], bl[1], bl[2], bl[3]});
          }
#pragma unroll
          for (int jj = 0; jj < 2; ++jj) {
            const int j = 2 * g + jj;
            half8_t Al, Ah;
            q4_v_operands(word_of(vq[j], 2 * ks), word_of(vq[j], 2 * ks + 1), magic, Al, Ah);
#pragma unroll
            for (int rt = 0; rt < NRT; ++rt) {
              o[rt][2 * j] = mfma16x16x32(Al, Bh[rt], o[rt][2 * j]);
              o[rt][2 * j + 1] = mfma16x16x32(Ah, Bh[rt], o[rt][2 * j + 1]);
              if constexpr (LOW) {
                o[rt][2 * j] = mfma16x16x32(Al, Bl[rt], o[rt][2 * j]);
                o[rt][2 * j + 1] = mfma16x16x32(Ah, Bl[rt], o[rt][2 * j + 1]);
              }
            }
          }
        }
      }
      load_v(rn);
      wave_sync();  // (the metadata is read before the next block's is written)
    }

    // the next sequence with blocks (the merge clears the others' rows)
    int bn = b + 1;
    bool more = false;
    if (!SEQ && i < iend) {
      while (bn < a.B && seq_blocks_rg(a, seq_len(bn), rg) == 0) ++bn;
      more = bn < a.B;
    }
    if (more) issue_q(bn, e);

    // ---- the segment's end: lane holds O^T[16 dt + 4 q4 + x][row n]; output or a
    // partial in slot (hk row_groups + rg) (waves + B) + range + b
    const bool whole = !a.partial_only && s >= i0 && e <= iend;
    if constexpr (SEQ) {
      float l = l_part[0];
      l += shfl_xor(l, 16);
      l += shfl_xor(l, 32);
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float c = c_part[0][g];
        c += shfl_xor(c, 16);
        c += shfl_xor(c, 32);
        if (n < kSeqRows) {
#pragma unroll
          for (int dt = 4 * g; dt < 4 * g + 4; ++dt)
            *reinterpret_cast<float4_t *>(&seq_o[wid][n * (D + 4) + 16 * dt + 4 * q4]) = o[0][dt] + c;
        }
      }
      if (q4 == 0 && n < kSeqRows) seq_ml[wid][n] = float2{m_run[0], l};
      if (new_phys >= 0) store_new(new_phys);
      break;
    }
    const int64_t slot = ((int64_t)hk * a.row_groups + rg) * (a.waves + a.B) + wv + b;
#pragma unroll
    for (int rt = 0; rt < NRT; ++rt) {
      float l = l_part[rt];
      l += shfl_xor(l, 16);
      l += shfl_xor(l, 32);
      float cg[G];
#pragma unroll
      for (int g = 0; g < G; ++g) {
        float c = c_part[rt][g];
        c += shfl_xor(c, 16);
        c += shfl_xor(c, 32);
        cg[g] = c;
      }
      if (!rvalid[rt]) continue;
      const float mul = !whole ? 1.0f : l > 0.0f ? 1.0f / l : 0.0f;
      const int64_t pi = slot * RR + 16 * rt + n;
      const int64_t ob = (whole ? (((int64_t)b * a.Hq + hk * a.R + rh[rt]) * a.Lq + rj[rt]) * D : pi * D) + sl * DW + 4 * q4;
      auto put = [&](void *out, auto dtype) {
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) {
          float run[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            run[x] = (o[rt][dt][x] + cg[dt / 4]) * mul;
          store_run<4>(out, ob + 16 * dt, run, decltype(dtype)::value);
        }
      };
      if (!whole)
        put(a.ws_o, std::integral_constant<int, DT_F32>{});
      else if (a.out_dtype == DT_F32)
        put(a.out, std::integral_constant<int, DT_F32>{});
      else if (a.out_dtype == DT_F16)
        put(a.out, std::integral_constant<int, DT_F16>{});
      else
        put(a.out, std::integral_constant<int, DT_BF16>{});
      if (!whole && sl == 0 && q4 == 0) reinterpret_cast<float2 *>(a.ws_ml)[pi] = float2{m_run[rt], l};
    }
    if (rg == 0 && new_phys >= 0) store_new(new_phys);
    if (!more) break;
    b = bn;
    s = e;
  }

  if constexpr (SEQ) {
    // a wave that had no block left nothing behind
    if (i0 >= iend && lane < kSeqRows) seq_ml[wid][lane] = float2{-INFINITY, 0.0f};
    __syncthreads();
    const int b0 = (int)blockIdx.x;
    const int nrow = min(kSeqRows, a.NR - rbase);
    for (int t = threadIdx.x; t < nrow * (D / 4); t += 64 * kSeqWaves) {
      const int r = t / (D / 4), d = 4 * (t % (D / 4));
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < kSeqWaves; ++w) M = fmaxf(M, seq_ml[w][r].x);
      float4_t acc = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kSeqWaves; ++w) {
        const float2 ml = seq_ml[w][r];
        // (a row whose scores are all NaN has m = -inf and l = NaN)
        const float f = ml.x != -INFINITY ? fast_exp2(ml.x - M) : 0.0f;
        L += f * ml.y;
        if (ml.x != -INFINITY || ml.y != 0.0f)
          acc += f * *reinterpret_cast<const float4_t *>(&seq_o[w][r * (D + 4) + d]);
      }
      const float inv = M == -INFINITY || !(L > 0.0f) ? L * 0.0f : 1.0f / L;
      const float run[4] = {acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv};
      store_run<4>(a.out, out_row_base(a, b0, hk, rbase + r, D) + d, run, a.out_dtype);
    }
  }
}

// Combines the partial results of few rows, whose sequences span dozens of ranges
// (the others take k_attn_merge_flat): four waves share a row's slots.  8 sequences
// of 115 000 tokens, 32 rows each: 6.8 us against 11.4 with a wave per row.  (Four
// rows a workgroup instead, for thousands of rows: 8.3 against 7.1, not kept.)
template <int D>
__global__ __launch_bounds__(256) void k_q4_merge(AttnArgs a) {
  constexpr int E = D / 64, K = 8, S = 4;  // K slots' rows in flight, every S-th the wave's
  __shared__ float sums[S][D];
  const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int r = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int64_t obase = out_row_base(a, b, hk, r, D);
  const int rg = r / a.rows_per_group, rr = r % a.rows_per_group;
  int s = 0, nb = 0;
  const int T = flat_total_and_start(a, b, rg, s, nb);
  int first = 0, n = 0;
  if (nb > 0) {
    const int Wt = min(a.waves, T);
    first = flat_wave_of(s, T, Wt);
    n = flat_wave_of(s + nb - 1, T, Wt) - first + 1;
    if (n == 1) return;  // (written by the attention kernel)
  }
  const int64_t slot0 = ((int64_t)hk * a.row_groups + rg) * (a.waves + a.B) + first + b;
  const float2 *ml2 = reinterpret_cast<const float2 *>(a.ws_ml);
  float M = -INFINITY, lsum = 0.0f, acc[E];
  for (int k = lane; k < n; k += 64) M = fmaxf(M, ml2[(slot0 + k) * a.rows_per_group + rr].x);
  M = uniform_f32(wave_allmax(M));
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.0f;
  for (int k0 = 0; k0 < n; k0 += 64) {
    const int cnt = min(64, n - k0);
    const float2 ml = lane < cnt ? ml2[(slot0 + k0 + lane) * a.rows_per_group + rr] : float2{-INFINITY, 0.0f};
    const float w = ml.x != -INFINITY ? fast_exp2(ml.x - M) : 0.0f;
    lsum += w * ml.y;
    // this wave's slots k, k + S, ..: past the last one its row again, weight 0
    for (int k = wid; k < cnt; k += S * K) {
      float o[K][E];
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const float *op = a.ws_o + ((slot0 + k0 + min(k + S * j, cnt - 1)) * a.rows_per_group + rr) * (int64_t)D + lane;
#pragma unroll
        for (int e = 0; e < E; ++e) o[j][e] = op[64 * e];
      }
#pragma unroll
      for (int j = 0; j < K; ++j) {
        const int kk = k + S * j;
        const float wk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), kk & 63));
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = kk < cnt ? __builtin_fmaf(wk, o[j][e], acc[e]) : acc[e];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) sums[wid][lane + 64 * e] = acc[e];
  __syncthreads();
  if (wid != 0) return;
#pragma unroll
  for (int e = 0; e < E; ++e)
    acc[e] = (sums[0][lane + 64 * e] + sums[1][lane + 64 * e]) + (sums[2][lane + 64 * e] + sums[3][lane + 64 * e]);
  const float L = uniform_f32(wave_allsum(lsum));
  const float inv = (M == -INFINITY || !(L > 0.0f)) ? L * 0.0f : 1.0f / L;  // (NaN rows: m = -inf, l = NaN)
#pragma unroll
  for (int e = 0; e < E; ++e) store_out(a.out, obase + lane + 64 * e, acc[e] * inv, a.out_dtype);
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
namespace {

template <int D, int NRT, bool SEQ>
hipError_t launch_q4(const AttnArgs &args, dim3 grid, hipStream_t st) {
  const bool low = args.out_dtype != DT_BF16;
  const dim3 block(64 * (SEQ ? kSeqWaves : q4_slices<D>()));
  if (args.window > 0) {
    if (low)
      k_attn_q4<D, NRT, true, true, SEQ><<<grid, block, 0, st>>>(args);
    else
      k_attn_q4<D, NRT, true, false, SEQ><<<grid, block, 0, st>>>(args);
  } else {
    if (low)
      k_attn_q4<D, NRT, false, true, SEQ><<<grid, block, 0, st>>>(args);
    else
      k_attn_q4<D, NRT, false, false, SEQ><<<grid, block, 0, st>>>(args);
  }
  return hipGetLastError();
}

template <int D, int NRT>
int32_t q4_occupancy() {
  static const int32_t n = [] {
    int blocks = 0;
    const auto *fn = reinterpret_cast<const void *>(&k_attn_q4<D, NRT, false, true, false>);
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, fn, 64 * q4_slices<D>(), 0) != hipSuccess || blocks < 1) {
      (void)hipGetLastError();
      blocks = 8 / q4_slices<D>();
    }
    return (int32_t)blocks;
  }();
  return n;
}

}  // namespace

// Row tiles per wave: two from 17 rows on (each unpacked operand feeds two
// products): 32 rows take 40.8 us so, 46.6 as two groups of 16 that each read the
// cache.  Up to 16 rows the second tile would be empty.
int32_t q4_row_tiles(int32_t NR) { return NR > 16 ? 2 : 1; }

int32_t q4_groups_per_cu(const PoolGeometry &g, int32_t nrt) {
  if (!g.base) return g.D <= 128 ? 8 : 8 * 128 / g.D;
  switch (g.D) {
    case 64: return nrt == 2 ? q4_occupancy<64, 2>() : q4_occupancy<64, 1>();
    case 128: return nrt == 2 ? q4_occupancy<128, 2>() : q4_occupancy<128, 1>();
    case 256: return nrt == 2 ? q4_occupancy<256, 2>() : q4_occupancy<256, 1>();
    default: return nrt == 2 ? q4_occupancy<512, 2>() : q4_occupancy<512, 1>();
  }
}

// A workgroup per (sequence, KV head), without a merge launch, while that many
// workgroups find a CU each and a wave's share is at most three blocks: one
// sequence of 512 tokens takes 16.6 us against 27.6 in the flat split (with less
// time on the host, the same for both).  Longer contexts fill the card only when
// they are split over it; a chosen split and the partials of a shared prefix need
// the flat order.
bool q4_per_sequence(const PoolGeometry &g, const AttnLaunch &a, const AttnPlan &p) {
  if (!p.q4 || g.D > 128 || p.NR > kSeqRows || p.split_blocks > 0 || a.partial_only || a.len_const >= 0 || !a.causal)
    return false;
  return (int64_t)a.B * g.Hkv <= g.num_cus && p.nb_cap <= 3 * kSeqWaves;
}

hipError_t launch_q4_merge(const PoolGeometry &g, int32_t layer, const AttnLaunch &a, const AttnPlan &p, hipStream_t st) {
  const AttnArgs args = make_attn_args(g, layer, a, p);
  const dim3 grid((unsigned)p.NR, (unsigned)g.Hkv, (unsigned)a.B), block(256);
  switch (g.D) {
    case 64: k_q4_merge<64><<<grid, block, 0, st>>>(args); break;
    case 128: k_q4_merge<128><<<grid, block, 0, st>>>(args); break;
    case 256: k_q4_merge<256><<<grid, block, 0, st>>>(args); break;
    case 512: k_q4_merge<512><<<grid, block, 0, st>>>(args); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_attn_q4(const PoolGeometry &g, int32_t layer, const AttnLaunch &a, const AttnPlan &p, hipStream_t st) {
  if (p.waves < 1 || p.group_waves != 1 || p.rows_per_group != 16 * p.nrt ||
      (int64_t)p.row_groups * p.rows_per_group < p.NR || (a.k_new && a.Lq != 1) || g.Hkv > 65535 || p.row_groups > 65535)
    return hipErrorInvalidValue;
  const AttnArgs args = make_attn_args(g, layer, a, p);
  if (q4_per_sequence(g, a, p)) {
    const dim3 seq((unsigned)a.B, (unsigned)g.Hkv);
    return g.D == 64 ? launch_q4<64, 1, true>(args, seq, st) : launch_q4<128, 1, true>(args, seq, st);
  }
  const dim3 grid((unsigned)p.waves, (unsigned)g.Hkv, (unsigned)p.row_groups);
  switch (4 * g.D + p.nrt) {
    case 4 * 64 + 1: return launch_q4<64, 1, false>(args, grid, st);
    case 4 * 64 + 2: return launch_q4<64, 2, false>(args, grid, st);
    case 4 * 128 + 1: return launch_q4<128, 1, false>(args, grid, st);
    case 4 * 128 + 2: return launch_q4<128, 2, false>(args, grid, st);
    case 4 * 256 + 1: return launch_q4<256, 1, false>(args, grid, st);
    case 4 * 256 + 2: return launch_q4<256, 2, false>(args, grid, st);
    case 4 * 512 + 1: return launch_q4<512, 1, false>(args, grid, st);
    case 4 * 512 + 2: return launch_q4<512, 2, false>(args, grid, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace krill
