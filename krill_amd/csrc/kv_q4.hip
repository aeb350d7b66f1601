// Writing and reading the 4-bit paged KV cache (layout and quantizer in
// kdev4.hpp): quantize-append with optional RoPE of K, and the read-back of
// slots or of whole sequences as fp16.
//
// Bound: memory.  A row of K and V is 4 D bytes of input and D + 8 D/64 bytes
// of cache (D = 128: 512 and 144), so an append reads 3.5 times what it
// writes and a read-back writes 3.5 times what it reads; the quantizer is some
// ten instructions per element beside them.  Measured at D = 128, Hkv = 8: 8 x 512
// rows appended 13.2 us (21 MB, 1.6 TB/s: one workgroup's rounds follow one another,
// and rolled up they take 13.2 us against 15.1 and 16.1 in twos and fours, whose
// code is fetched once per call); 64 single rows 14.7 us a call, the host's time;
// 8 sequences of 512-8192 tokens read back 63 us, 308 MB at 4.9 TB/s, the rate of
// a large copy.
#include <hip/hip_runtime.h>

#include "kdev4.hpp"
#include "launch.hpp"

namespace krill {

namespace {

LayerView view_of(const PoolGeometry &g, int32_t layer) {
  LayerView lv;
  lv.base = g.base + (int64_t)layer * g.layer_stride;
  lv.block_stride = g.block_stride;
  lv.head_bytes = g.head_bytes;
  lv.num_blocks = g.num_blocks;
  return lv;
}

// One workgroup's rows in LDS, as the head region of a block lays them out.
template <int D>
struct Q4Image {
  __attribute__((aligned(16))) uint8_t bytes[q4_region_bytes(D)];
  int slot[64];  // pool slot of row r, -1: none
  int block;     // block of all rows where row r has slot 64 block + r, else -1
};

// slot[] complete and written by wave 0: sets block.
template <int D>
__device__ __forceinline__ void find_block(Q4Image<D> &im, int slot, int lane) {
  const uint64_t have = __ballot(slot >= 0);
  int blk = -1;
  if (have) {
    blk = __builtin_amdgcn_readlane(slot, __builtin_ctzll(have)) >> 6;
    if (__ballot(slot >= 0 && slot != blk * 64 + lane)) blk = -1;
  }
  if (lane == 0) im.block = blk;
}

// Moves row `r` of the image to or from token t of head region `reg`, item by
// item: the row's K words in pairs, V bytes and metadata words.
template <int D>
constexpr int row_items() { return D / 16 + D / 2 + 2 * (D / 64); }
template <int D, bool STORE>
__device__ __forceinline__ void move_row_item(uint8_t *img, int r, uint8_t *reg, int t, int i) {
  constexpr int G = D / 64;
  auto move = [&](int im, int rg, auto word) {
    using T = decltype(word);
    if constexpr (STORE)
      *reinterpret_cast<T *>(reg + rg) = *reinterpret_cast<const T *>(img + im);
    else
      *reinterpret_cast<T *>(img + im) = *reinterpret_cast<const T *>(reg + rg);
  };
  if (i < D / 16) {
    move(q4_k_word(D, r, 2 * i), q4_k_word(D, t, 2 * i), uint2{});
  } else if (i < D / 16 + D / 2) {
    const int m = i - D / 16;
    move(q4_v_byte(D, r, m), q4_v_byte(D, t, m), uint8_t{});
  } else {
    const int k = i - D / 16 - D / 2;
    const int o = k < G ? q4_km_offset(D) : q4_vm_offset(D), g = k < G ? k : k - G;
    move(o + (r * G + g) * 4, o + (t * G + g) * 4, uint32_t{});
  }
}

}  // namespace

// ---------------------------------------------------------------------------
// Quantize + append.  A workgroup takes the rows of one (sequence, KV head)
// that fall into one aligned run of 64 tokens (the first row's slot says where
// the runs lie), quantizes them into an image of the block's head region in
// LDS -- eight lanes per group of 64 dims, 16 bytes of input each -- and writes
// the image in one contiguous run where it is a whole block, else the rows it
// has.  Slots may name any tokens; runs that are not one block's are written
// row by row.
// ---------------------------------------------------------------------------
struct Q4Rope {
  const int32_t *pos;  // [B][L] (null: none)
  const float *cs;     // [max_pos][D]: cosines of D/2 angles, then sines
  int32_t max_pos;
};

template <int D, int DT, bool ROPE>
__global__ __launch_bounds__(256) void k_q4_append(LayerView lv, const uint16_t *__restrict__ k,
                                                   const uint16_t *__restrict__ v, int64_t sb, int64_t sh, int64_t sl,
                                                   const int32_t *__restrict__ slots, int32_t L, int32_t wide,
                                                   Q4Rope rope) {
  constexpr int G = D / 64;
  constexpr int LPR = D / 8;         // lanes per row
  constexpr int RPW = 64 / LPR;      // rows of a wave at a time
  __shared__ Q4Image<D> im;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int h = blockIdx.y, b = blockIdx.z;
  const int first = slots[(int64_t)b * L];
  const int l0 = (int)blockIdx.x * 64 - (first >= 0 ? first & 63 : 0);
  const int ra = max(0, -l0), rb = min(64, L - l0);  // rows of this run: l = l0 + r
  if (ra >= rb) return;
  if (tid < 64) {
    int s = -1;
    if (lane >= ra && lane < rb) {
      s = slots[(int64_t)b * L + l0 + lane];
      if (s < 0 || (s >> 6) >= lv.num_blocks) s = -1;
      if (ROPE && (unsigned)rope.pos[(int64_t)b * L + l0 + lane] >= (unsigned)rope.max_pos) s = -1;
    }
    im.slot[lane] = s;
    find_block<D>(im, s, lane);
  }

  const int x = lane % LPR;  // dims 8 x .. 8 x + 7
  const int64_t base = (int64_t)b * sb + (int64_t)h * sh + 8 * x;
  auto load8 = [&](const uint16_t *p) -> uint4 {
    if (wide) return *reinterpret_cast<const uint4 *>(p);
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (uint32_t)p[2 * e] | ((uint32_t)p[2 * e + 1] << 16);
    return uint4{w[0], w[1], w[2], w[3]};
  };
  // Rounds of 4 RPW rows, the next round's loads ahead of this one's work; a loop,
  // because a workgroup runs through this once and what it costs is the fetch of its
  // instructions: 8 x 512 rows (D 128) take 13.2 us so, 16.1 with four rounds
  // unrolled.  (Rows without a slot are read too: no load waits for the slots.)
  struct Round {
    uint4 k, v;
    int r;
  };
  auto load_round = [&](int it) -> Round {
    const int r = (it * 4 + wid) * RPW + lane / LPR;
    Round n{uint4{0u, 0u, 0u, 0u}, uint4{0u, 0u, 0u, 0u}, r >= ra && r < rb ? r : -1};
    if (n.r >= 0) {
      const int64_t o = base + (int64_t)(l0 + r) * sl;
      n.k = load8(k + o);
      n.v = load8(v + o);
    }
    return n;
  };
  const int last = (rb + 4 * RPW - 1) / (4 * RPW);
  Round next = load_round(ra / (4 * RPW));
#pragma unroll 1
  for (int it = ra / (4 * RPW); it < last; ++it) {
    const Round cur = next;
    if (it + 1 < last) next = load_round(it + 1);
    {
      const int r = cur.r;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint4 raw = kv ? cur.v : cur.k;
        uint32_t w4[4] = {raw.x, raw.y, raw.z, raw.w};
        if (ROPE && kv == 0) {
          // element i < D/2 pairs with i + D/2, LPR/2 lanes on; each product and
          // sum rounded once, then to the element type
          int p = r >= 0 ? rope.pos[(int64_t)b * L + l0 + r] : 0;
          p = (unsigned)p < (unsigned)rope.max_pos ? p : 0;  // (outside: not written)
          const float *cs = rope.cs + (int64_t)p * D + 8 * (x % (LPR / 2));
          const bool hi = x >= LPR / 2;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t o = (uint32_t)__shfl_xor((int)w4[e], LPR / 2, 64);
            uint32_t res = 0;
#pragma unroll
            for (int f = 0; f < 2; ++f) {
              const float a = elem_to_f32<DT>((uint16_t)(w4[e] >> (16 * f)));
              const float c = elem_to_f32<DT>((uint16_t)(o >> (16 * f)));
              const float co = cs[2 * e + f], si = cs[D / 2 + 2 * e + f];
              const float y = hi ? c * si + a * co : a * co - c * si;
              res |= (uint32_t)(DT == DT_BF16 ? f32_to_bf16_bits(y) : f32_to_f16_bits(y)) << (16 * f);
            }
            w4[e] = res;
          }
        }
        uint32_t lo4, hi4;
        const uint32_t meta = q4_codes8<DT>(w4, lo4, hi4);
        if (kv == 0) {
          if (r >= 0) *reinterpret_cast<uint32_t *>(im.bytes + q4_k_word(D, r, x)) = q4_k_pack(lo4, hi4);
        } else {
          // bytes of dims (d, d + 16): the lane's and those of lane x ^ 2, four each
          const bool up = (x & 2) != 0;
          const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(up ? lo4 : hi4), 0x4E, 0xf, 0xf, false);
          const uint32_t v4 = up ? o | (hi4 << 4) : lo4 | (o << 4);
          const int m = 16 * (x >> 2) + 8 * (x & 1) + (up ? 4 : 0);
          if (r >= 0) {
#pragma unroll
            for (int e = 0; e < 4; ++e) im.bytes[q4_v_byte(D, r, m + e)] = (uint8_t)(v4 >> (8 * e));
          }
        }
        if (r >= 0 && (x & 7) == 0)
          *reinterpret_cast<uint32_t *>(im.bytes + (kv ? q4_vm_offset(D) : q4_km_offset(D)) + (r * G + (x >> 3)) * 4) = meta;
      }
    }
  }
  __syncthreads();

  const int blk = im.block;
  if (blk >= 0 && __all(lane < ra || lane >= rb || im.slot[lane] >= 0)) {
    // a run of one block's tokens
    uint8_t *reg = head_region(lv, blk, h);
    if (ra == 0 && rb == 64) {
      for (int i = tid; i < q4_region_bytes(D) / 16; i += 256)
        reinterpret_cast<uint4 *>(reg)[i] = reinterpret_cast<const uint4 *>(im.bytes)[i];
      return;
    }
    const int rows = rb - ra;
    for (int i = tid; i < rows * (D / 16); i += 256)
      move_row_item<D, true>(im.bytes, ra + i / (D / 16), reg, ra + i / (D / 16), i % (D / 16));
    for (int i = tid; i < rows * 2 * G; i += 256)
      move_row_item<D, true>(im.bytes, ra + i / (2 * G), reg, ra + i / (2 * G), D / 16 + D / 2 + i % (2 * G));
    // V words of four tokens
    for (int i = tid; i < 8 * D; i += 256) {
      const int w = i & 3, t0 = 32 * (w >> 1) + 16 * (w & 1) + 4 * ((i >> 6) & 3), at = q4_v_offset(D) + 4 * i;
      if (t0 >= ra && t0 + 4 <= rb) {
        *reinterpret_cast<uint32_t *>(reg + at) = *reinterpret_cast<const uint32_t *>(im.bytes + at);
      } else {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (t0 + x >= ra && t0 + x < rb) reg[at + (q4_v_slot(x) & 3)] = im.bytes[at + (q4_v_slot(x) & 3)];
      }
    }
    return;
  }
  for (int i = tid; i < (rb - ra) * row_items<D>(); i += 256) {
    const int r = ra + i / row_items<D>();
    const int s = im.slot[r];
    if (s >= 0) move_row_item<D, true>(im.bytes, r, head_region(lv, s >> 6, h), s & 63, i % row_items<D>());
  }
}

// The same for a few rows (a decode step's tokens, drafts): a wave per row of K or
// of V, no image and no barrier.
template <int D, int DT, bool ROPE>
__global__ __launch_bounds__(256) void k_q4_append_rows(LayerView lv, const uint16_t *__restrict__ k,
                                                        const uint16_t *__restrict__ v, int64_t sb, int64_t sh,
                                                        int64_t sl, const int32_t *__restrict__ slots, int32_t B,
                                                        int32_t L, int32_t H, Q4Rope rope) {
  constexpr int G = D / 64, E = D / 64;
  const int lane = threadIdx.x & 63;
  const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (wave >= 2 * (int64_t)B * H * L) return;
  const int kv = (int)(wave & 1);
  const int64_t row = wave >> 1;  // [B][L][H]: neighbours share their slot
  const int h = (int)(row % H), l = (int)(row / H % L), b = (int)(row / H / L);
  const int64_t at = (int64_t)b * L + l;
  const int slot = slots[at];
  const int p = ROPE ? rope.pos[at] : 0;
  const uint16_t *src = (kv ? v : k) + (int64_t)b * sb + (int64_t)h * sh + (int64_t)l * sl;
  const int d0 = lane * E;
  float x[E];
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = elem_to_f32<DT>(src[d0 + e]);
  if (slot < 0 || (slot >> 6) >= lv.num_blocks) return;
  if constexpr (ROPE) {
    if ((unsigned)p >= (unsigned)rope.max_pos) return;
    if (kv == 0) {
      const float *cs = rope.cs + (int64_t)p * D + (d0 & (D / 2 - 1));
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float y = __shfl_xor(x[e], 32, 64), c = cs[e], sn = cs[D / 2 + e];
        x[e] = round_dt<DT>(lane >= 32 ? y * sn + x[e] * c : x[e] * c - y * sn);
      }
    }
  }
  uint32_t code[E];
  const uint32_t meta = q4_quantize_row<D, DT>(x, code);
  const int t = slot & 63;
  uint8_t *reg = head_region(lv, slot >> 6, h);
  if (kv == 0) {
    // 8/E lanes hold a word
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) w |= code[e] << (4 * q4_nibble((d0 + e) & 7));
    if constexpr (E < 8) w |= (uint32_t)__shfl_xor((int)w, 1, 64);
    if constexpr (E < 4) w |= (uint32_t)__shfl_xor((int)w, 2, 64);
    if constexpr (E < 2) w |= (uint32_t)__shfl_xor((int)w, 4, 64);
    if ((d0 & 7) == 0) *reinterpret_cast<uint32_t *>(reg + q4_k_word(D, t, d0 / 8)) = w;
  } else {
    // dims d and d + 16 share a byte
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t up = (uint32_t)__shfl_xor((int)code[e], 16 / E, 64);
      if ((d0 & 16) == 0) reg[q4_v_byte(D, t, 16 * (d0 >> 5) + ((d0 + e) & 15))] = (uint8_t)(code[e] | (up << 4));
    }
  }
  if ((d0 & 63) == 0)
    *reinterpret_cast<uint32_t *>(reg + (kv ? q4_vm_offset(D) : q4_km_offset(D)) + (t * G + d0 / 64) * 4) = meta;
}

// ---------------------------------------------------------------------------
// Read-back as fp16.  A workgroup stages up to 64 rows of one (sequence, KV
// head) in LDS -- the whole head region where they are one block's -- and
// writes eight dims per lane.
//  SLOTS: out rows [B][H][L][D], row l from slots[b][l] (zeros where it names
//  no slot);  else: out rows [B][H][S_out][D], token ti of sequence b at row
//  ti (left_pad: S_out - len + ti), zeros elsewhere.
// ---------------------------------------------------------------------------
struct Q4Read {
  const int32_t *slots;               // SLOTS: [B][L]
  const int32_t *tables, *lens;       // else
  int32_t rows, max_blocks, left_pad; // rows: L or S_out
  int32_t nbx;                        // else: workgroups of data; the others clear rows without a token
};

template <int D, bool SLOTS>
__global__ __launch_bounds__(256) void k_q4_read(LayerView lv, Q4Read a, uint16_t *__restrict__ k_out,
                                                 uint16_t *__restrict__ v_out) {
  constexpr int G = D / 64, LPR = D / 8;
  __shared__ Q4Image<D> im;
  const int tid = threadIdx.x, lane = tid & 63;
  const int h = blockIdx.y, b = blockIdx.z;
  const int64_t row0 = ((int64_t)b * gridDim.y + h) * a.rows;
  int ra, rb, o0;  // rows r in [ra, rb) go to output row o0 + r
  if constexpr (SLOTS) {
    const int first = a.slots[(int64_t)b * a.rows];
    o0 = (int)blockIdx.x * 64 - (first >= 0 ? first & 63 : 0);
    ra = max(0, -o0);
    rb = min(64, a.rows - o0);
    if (ra >= rb) return;
    if (tid < 64) {
      int s = lane >= ra && lane < rb ? a.slots[(int64_t)b * a.rows + o0 + lane] : -1;
      if (s < 0 || (s >> 6) >= lv.num_blocks) s = -1;
      im.slot[lane] = s;
      find_block<D>(im, s, lane);
    }
  } else {
    const int len = a.lens[b];
    const int off = a.left_pad ? a.rows - len : 0;
    const int t_lo = max(0, -off), t_hi = min(len, a.rows - off);  // tokens that have a row
    if ((int)blockIdx.x >= a.nbx) {
      const int s0 = ((int)blockIdx.x - a.nbx) * 64;
      for (int p = tid; p < 64 * LPR; p += 256) {
        const int s = s0 + p / LPR, ti = s - off;
        if (s < a.rows && (ti < t_lo || ti >= t_hi)) {
          const int64_t o = (row0 + s) * D + 8 * (p % LPR);
          *reinterpret_cast<uint4 *>(k_out + o) = *reinterpret_cast<uint4 *>(v_out + o) = uint4{0u, 0u, 0u, 0u};
        }
      }
      return;
    }
    if (t_hi <= t_lo) return;
    const int j = (t_lo >> 6) + (int)blockIdx.x;
    ra = max(t_lo - 64 * j, 0);
    rb = min(t_hi - 64 * j, 64);
    if (ra >= rb) return;
    o0 = 64 * j + off;
    const int blk = j < a.max_blocks ? a.tables[(int64_t)b * a.max_blocks + j] : -1;
    const bool ok = (unsigned)blk < (unsigned)lv.num_blocks;
    if (tid < 64) {
      im.slot[lane] = ok && lane >= ra && lane < rb ? blk * 64 + lane : -1;
      if (lane == 0) im.block = ok ? blk : -1;
    }
  }
  __syncthreads();
  const int blk = im.block;
  if (blk >= 0 && rb - ra >= 16) {
    const uint8_t *reg = head_region(lv, blk, h);
    for (int i = tid; i < q4_region_bytes(D) / 16; i += 256)
      reinterpret_cast<uint4 *>(im.bytes)[i] = reinterpret_cast<const uint4 *>(reg)[i];
  } else {
    for (int i = tid; i < (rb - ra) * row_items<D>(); i += 256) {
      const int r = ra + i / row_items<D>();
      const int s = im.slot[r];
      if (s >= 0) move_row_item<D, false>(im.bytes, r, head_region(lv, s >> 6, h), s & 63, i % row_items<D>());
    }
  }
  __syncthreads();
  for (int i = tid; i < (rb - ra) * LPR; i += 256) {
    const int r = ra + i / LPR, x = i % LPR, g = x >> 3;
    const bool have = im.slot[r] >= 0;
    uint4 res[2] = {uint4{0u, 0u, 0u, 0u}, uint4{0u, 0u, 0u, 0u}};
    // V: four bytes of dims (d, d + 16) here, four in lane x ^ 2 (all lanes of
    // a group take part: LPR is a multiple of 8 and so is the loop's end)
    const bool up = (x & 2) != 0;
    const int m = 16 * (x >> 2) + 8 * (x & 1) + (up ? 4 : 0);
    uint32_t a4 = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) a4 |= (uint32_t)im.bytes[q4_v_byte(D, r, m + e)] << (8 * e);
    const uint32_t o4 = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a4, 0x4E, 0xf, 0xf, false);
    if (have) {
      const uint32_t kw = *reinterpret_cast<const uint32_t *>(im.bytes + q4_k_word(D, r, x));
      const uint32_t v0 = (up ? o4 : a4) >> (up ? 4 : 0), v1 = (up ? a4 : o4) >> (up ? 4 : 0);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t meta = *reinterpret_cast<const uint32_t *>(
            im.bytes + (kv ? q4_vm_offset(D) : q4_km_offset(D)) + (r * G + g) * 4);
        const float s = f16_bits_to_f32((uint16_t)(meta & 0xffffu)), bias = f16_bits_to_f32((uint16_t)(meta >> 16));
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const uint32_t c0 = kv ? ((e < 4 ? v0 : v1) >> (8 * (e & 3))) & 15u : (kw >> (4 * q4_nibble(e))) & 15u;
          const uint32_t c1 = kv ? ((e < 4 ? v0 : v1) >> (8 * ((e + 1) & 3))) & 15u : (kw >> (4 * q4_nibble(e + 1))) & 15u;
          w[e / 2] = q4_value_bits(c0, s, bias) | (q4_value_bits(c1, s, bias) << 16);
        }
        res[kv] = uint4{w[0], w[1], w[2], w[3]};
      }
    }
    const int64_t o = (row0 + o0 + r) * D + 8 * x;
    *reinterpret_cast<uint4 *>(k_out + o) = res[0];
    *reinterpret_cast<uint4 *>(v_out + o) = res[1];
  }
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
#define KRILL_Q4_DISPATCH(D_, ...)                      \
  switch (D_) {                                         \
    case 64: { constexpr int D = 64; __VA_ARGS__; } break;   \
    case 128: { constexpr int D = 128; __VA_ARGS__; } break; \
    case 256: { constexpr int D = 256; __VA_ARGS__; } break; \
    case 512: { constexpr int D = 512; __VA_ARGS__; } break; \
    default: return hipErrorInvalidValue;               \
  }

hipError_t launch_q4_append(const PoolGeometry &g, int32_t layer, const void *k, const void *v, int64_t sb, int64_t sh,
                            int64_t sl, const int32_t *slots, int32_t B, int32_t L, hipStream_t st,
                            const int32_t *rope_pos, const float *rope_cs, int32_t rope_max_pos) {
  if ((int64_t)B * L * g.Hkv == 0) return hipSuccess;
  const auto *kk = static_cast<const uint16_t *>(k), *vv = static_cast<const uint16_t *>(v);
  // 16-byte loads where every row starts on 16 bytes
  const int32_t wide = ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                         (uintptr_t)(2 * (sb | sh | sl))) & 15) == 0;
  const dim3 grid((unsigned)(((int64_t)L + 126) / 64), (unsigned)g.Hkv, (unsigned)B), block(256);
  const LayerView lv = view_of(g, layer);
  const Q4Rope rope{rope_pos, rope_cs, rope_max_pos};
  // A wave per row up to 16 rows a sequence (64 x 1 row, Hkv 8: 14.9 us a call against
  // 22.8 in windows, whose workgroups would be nearly empty), windows of 64 rows
  // above, which store whole words of several tokens.
  if (L <= 16 || B > 65535 || g.Hkv > 65535) {
    const int64_t waves = 2 * (int64_t)B * g.Hkv * L;
    if (waves > 4 * (int64_t)0xffffff) return hipErrorInvalidValue;  // (2^32 threads a launch)
    const dim3 rows((unsigned)((waves + 3) / 4));
    KRILL_Q4_DISPATCH(g.D, {
      if (g.in_dtype == DT_BF16) {
        if (rope_pos)
          k_q4_append_rows<D, DT_BF16, true><<<rows, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, B, L, g.Hkv, rope);
        else
          k_q4_append_rows<D, DT_BF16, false><<<rows, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, B, L, g.Hkv, rope);
      } else {
        if (rope_pos)
          k_q4_append_rows<D, DT_F16, true><<<rows, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, B, L, g.Hkv, rope);
        else
          k_q4_append_rows<D, DT_F16, false><<<rows, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, B, L, g.Hkv, rope);
      }
    });
    return hipGetLastError();
  }
  KRILL_Q4_DISPATCH(g.D, {
    if (g.in_dtype == DT_BF16) {
      if (rope_pos)
        k_q4_append<D, DT_BF16, true><<<grid, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, L, wide, rope);
      else
        k_q4_append<D, DT_BF16, false><<<grid, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, L, wide, rope);
    } else {
      if (rope_pos)
        k_q4_append<D, DT_F16, true><<<grid, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, L, wide, rope);
      else
        k_q4_append<D, DT_F16, false><<<grid, block, 0, st>>>(lv, kk, vv, sb, sh, sl, slots, L, wide, rope);
    }
  });
  return hipGetLastError();
}

hipError_t launch_q4_gather_dequant(const PoolGeometry &g, int32_t layer, const int32_t *tables, const int32_t *lens,
                                    int32_t B, int32_t max_blocks, int32_t S_out, int32_t left_pad, void *k_out,
                                    void *v_out, hipStream_t st) {
  if ((int64_t)B * g.Hkv * S_out == 0) return hipSuccess;
  if (B > 65535 || g.Hkv > 65535) return hipErrorInvalidValue;
  // the tokens that have a row span at most ceil(S_out / 64) + 1 blocks; then a
  // workgroup per 64 rows for those without
  const int32_t tiles = (int32_t)(((int64_t)S_out + 63) / 64), nbx = tiles + 1;
  const dim3 grid((unsigned)nbx + (unsigned)tiles, (unsigned)g.Hkv, (unsigned)B), block(256);
  const LayerView lv = view_of(g, layer);
  const Q4Read a{nullptr, tables, lens, S_out, max_blocks, left_pad, nbx};
  auto *ko = static_cast<uint16_t *>(k_out), *vo = static_cast<uint16_t *>(v_out);
  KRILL_Q4_DISPATCH(g.D, { k_q4_read<D, false><<<grid, block, 0, st>>>(lv, a, ko, vo); });
  return hipGetLastError();
}

hipError_t launch_q4_read_slots(const PoolGeometry &g, int32_t layer, const int32_t *slots, int32_t B, int32_t L,
                                void *k_out, void *v_out, hipStream_t st) {
  if ((int64_t)B * g.Hkv * L == 0) return hipSuccess;
  if (B > 65535 || g.Hkv > 65535) return hipErrorInvalidValue;
  const dim3 grid((unsigned)(((int64_t)L + 126) / 64), (unsigned)g.Hkv, (unsigned)B), block(256);
  const LayerView lv = view_of(g, layer);
  const Q4Read a{slots, nullptr, nullptr, L, 0, 0, 0};
  auto *ko = static_cast<uint16_t *>(k_out), *vo = static_cast<uint16_t *>(v_out);
  KRILL_Q4_DISPATCH(g.D, { k_q4_read<D, true><<<grid, block, 0, st>>>(lv, a, ko, vo); });
  return hipGetLastError();
}

}  // namespace krill
