// Attention over the 4-bit K/V cache (gfx950); the cache's layout is in fdl_kv4.h.
//
//  * fdl_kv4_attention: for query row r and head h of a tile, with G query heads to a K/V head,
//        O[r, h] = softmax over keys n in [k_begin, k_end) of (scale Q[r, h] . K[n, h / G]) V[n, h / G]
//    and the raw-logit importance sum_{r < n_imp} Q[r, h] . K[n, h / G] per key.
//  * fdl_kv4_verify_attention: the same over gathered cache keys and the block's own rows (bf16)
//    under the Flash-Verify mask.
//
// Per 64-key block and operand of 16 query rows
//    S^T = K Q^T   v_mfma_f32_16x16x32_bf16, K converted in registers (exact in bf16: two significant bits
//                  times a power of two), so a logit is a 32-bit sum of exact products. The scaled MFMA
//                  takes K as stored and Q as two 8-bit parts at the same matrix rate, but aligns the
//                  products of a 32-channel group to the largest and drops what lies 2^-13 below it: with
//                  one channel of a query far above the others, outputs were 8 times as far off as
//                  the rounding of P allows. The conversions cost up to 3.4% (8 x 1024 rows and keys,
//                  whose issue slots are full: 153 -> 158 us; one token over 2011 keys 9.4 -> 9.0, since
//                  Q needs no parts).
//    O^T = V^T P^T v_mfma_f32_16x16x32_bf16, V converted alike, P rounded to bf16 as the bf16
//                  cache's attention does; the rows' sums of P are one more row of V^T, all ones, so
//                  they are of the rounded P and cost no vector instructions.
// Keys sit so that nothing moves between lanes. Of a block's 64 keys, MFMA row mm of the t-th K operand
// is key 4 mm + t, so lane (c = lane % 16, g = lane / 16) ends up with the logits of query c and the 16
// keys of the block's g-th cell, in the order in which P V takes them.
//
// Two kernels. kv4_wave_kernel (up to 32 rows, i.e. rows x query heads to a K/V head: single tokens, small
// blocks) lets every wavefront take blocks of its own, straight from memory into registers with the
// next one in flight, and merges at the end: no barrier in the key loop, and V is converted once as no
// two wavefronts read the same keys. kv4_tile_kernel (more rows, and Flash-Verify) splits the rows over
// the wavefronts of a workgroup, which convert a block's V once into LDS and share it.
#include "fdl_host.h"
#include "fdl_kv4.h"

#include <type_traits>

namespace fdl {
namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kHeadDim = kKv4HeadDim;
constexpr int kBlockKeys = 64;
// A row's partial result: O (relative to the maximum), the maximum (log2 units), the sum, padding.
constexpr int kPartFloats = FDL_KV4_PART_FLOATS;
// Digits of a summed query (base 16, -8..8): 2^-28 of its largest element. Digits, not 8-bit floats: the
// scaled MFMA aligns the products of a 32-channel group to the largest and drops what lies 2^-13 below
// it; products of digits and codes span 2^8, so their sums are exact.
constexpr int kImpDigits = 7;
constexpr int kImpMaxGroup = 16;  // query heads to a K/V head with importance

struct Kv4Args {
  const uint16_t* q;
  const uint8_t* cache;
  uint16_t* out;
  const int32_t* page_table;
  const int32_t* work;
  const int32_t* row_idx;
  float* imp_part;
  float* part;  // [n_parts][n_items][tile_rows][heads][kPartFloats]
  int64_t n_q_rows, n_slots, n_row_idx, max_pages;
  int n_seq, page_log2;
  int heads, kv_heads, group;
  int tile_rows, n_items;  // verify: block_rows, verify blocks
  int n_parts, part_blocks;
  int n_ranges;  // workgroups to an item's rows
  float scale_log2;
  // verify
  const uint16_t* kblk;
  const uint16_t* vblk;
  const int64_t* key_slots;
  const int32_t* vblocks;
  const uint8_t* mask;
  const int32_t* vmeta;
  int64_t n_keys;
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void* lds_ptr;

// IEEE maximum (a NaN wins): one instruction where fmaxf takes three to quiet its operands.
__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), bf16x2));
}
// Maximum over the four lane groups (lane ^ 16, lane ^ 32) on the VALU.
__device__ __forceinline__ float xmax(float v) {
  const auto a =
      __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  const float m = vmax(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b =
      __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
  return vmax(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Exponent (biased by 127) of the 8-bit scale that brings magnitudes up to `top` below 256, kept
// inside [30, 249] so that the scales of its parts exist.
__device__ __forceinline__ int q_scale(float top) {
  const int e = static_cast<int>(__float_as_uint(top) >> 23) - 7;
  return min(max(e, 30), 249);
}
__device__ __forceinline__ float exp2i(int biased) { return __uint_as_float(uint32_t(biased) << 23); }

// The 128 channels of a query as four B operands: lane group g's share of operand x is channels 32 g + 8 x ..,
// word x of the 32 channels that the lane holds of a key. A query with a NaN or an infinity is NaN as a
// whole: its logits, which may all be the same infinity, are then never taken for keys left out.
struct QFrag {
  u32x4 x[4];
};

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ QFrag load_q(const uint16_t* row, int g, bool valid) {
  QFrag f;
  u16x2 top = {0, 0};
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    f.x[x] = valid ? ld16(row + 32 * g + 8 * x) : u32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, f.x[x][j] & 0x7fff7fffu));
  }
  if (top[0] >= 0x7f80 || top[1] >= 0x7f80) f.x[0][0] = ~0u;
  return f;
}

// A 64-key block of one K/V head as lane (c, g) holds it: K operand t (key 4 c + t, channels 32 g ..),
// its scales (byte t), four keys' words of channels 8 c .. in each v[i] (keys 16 g + 4 i ..), and the
// scale bytes of the cell's 16 keys for those channels.
struct Block {
  u32x4 k[4];
  uint32_t ks;
  u32x4 v[4];
  u32x4 vs;
};

// The state of R x 16 query rows: lane (c, g) holds query c's reference maximum (log2 units), the sum of
// its probabilities (in every element of l), and O^T: element e of o[.][i] is O^T row 4 g + e of the
// i-th V^T operand.
template <int R>
struct Rows {
  float m[R], limit[R];  // limit: logits above it raise the reference
  f32x4 l[R];
  f32x4 o[R][8];
  bool far;  // the same in every lane: a reference lies past kFar
  __device__ __forceinline__ void clear() {
    far = false;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      m[r] = limit[r] = -INFINITY;
      l[r] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; ++i) o[r][i] = l[r];
    }
  }
};

// The reference maximum may lag the true one by this much (log2 units): P stays below 2^kSlack, with
// the same relative rounding, and O is rescaled a few times per row instead of at every new maximum.
constexpr float kSlack = 8.f;
// Past this a reference, rounded to 32 bits, may be off the product that it stands for by more than the
// exponential takes: the other logits' products are then rounded too.
constexpr float kFar = 0x1p24f;

// Brings operand r's reference maxima up to a block's logits (s[t][e]: key 16 g + 4 e + t). Returns the factor
// that the logits still lack.
template <int R>
__device__ __forceinline__ float raise_maxima(Rows<R>& st, int r, f32x4 (&s)[4], float scale) {
  float top = vmax(vmax(s[0][0], s[0][1]), vmax(s[0][2], s[0][3]));
#pragma unroll
  for (int t = 1; t < 4; ++t) {
    top = vmax(vmax(top, s[t][0]), s[t][1]);
    top = vmax(vmax(top, s[t][2]), s[t][3]);
  }
  const float m = xmax(top) * scale;
  if (__any(m > st.limit[r]) || st.far) {
    const float to = vmax(st.m[r], m);
    st.far = st.far || __any(fabsf(to) > kFar && to != -INFINITY);  // (-infinity: no keys yet)
    // a NaN or an infinity as the maximum makes the row NaN all the same
    const float keep = st.m[r] == to ? 1.f : fast_exp2(st.m[r] - to);
    st.l[r] *= keep;
#pragma unroll
    for (int i = 0; i < 8; ++i) st.o[r][i] *= keep;
    st.m[r] = to;
    st.limit[r] = to == -INFINITY ? to : to + kSlack;
    if (st.far) {
#pragma unroll
      for (int t = 0; t < 4; ++t) s[t] *= scale;
      return 1.f;
    }
  }
  return scale;
}

// Logits -> probabilities as the operands of P V: element j of the u-th is key 16 g + 8 u + j.
__device__ __forceinline__ void probabilities(const f32x4 (&s)[4], float scale, float m,
                                              u32x4 (&p)[2]) {
  const float base = m == -INFINITY ? 0.f : m;
  float x[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[t][e] = fast_exp2(__builtin_fmaf(s[t][e], scale, -base));
#pragma unroll
  for (int u = 0; u < 2; ++u)
    p[u] = u32x4{pack2(x[0][2 * u], x[1][2 * u]), pack2(x[2][2 * u], x[3][2 * u]),
                 pack2(x[0][2 * u + 1], x[1][2 * u + 1]), pack2(x[2][2 * u + 1], x[3][2 * u + 1])};
}

// Adds the sums of P: an operand of ones.
__device__ __forceinline__ f32x4 add_sums(f32x4 l, u32x4 p) {
  const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  return mfma16(as_bf16x8(ones), as_bf16x8(p), l);
}

// Logits of a cache block's K operands (byte t of ks: operand t's scales), converted a word at a time for all
// R operands of queries: four sums side by side to each, of exact products in 32 bits.
template <int R>
__device__ __forceinline__ void logits(const u32x4 (&k)[4], uint32_t ks, const QFrag (&q)[R],
                                       f32x4 (&s)[R][4]) {
  float scale[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    scale[t] = __uint_as_float((ks >> (8 * t) & 255u) << 23);
#pragma unroll
    for (int r = 0; r < R; ++r) s[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int x = 0; x < 4; ++x)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const uint32_t w = k[t][x];
      const u32x4 a = {kv4_bf16x2<0>(w, scale[t]), kv4_bf16x2<1>(w, scale[t]),
                       kv4_bf16x2<2>(w, scale[t]), kv4_bf16x2<3>(w, scale[t])};
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][t] = mfma16(as_bf16x8(a), as_bf16x8(q[r].x[x]), s[r][t]);
    }
}

// Keys that do not count (bit 4 e + t of ok clear) leave the softmax.
__device__ __forceinline__ void hide(f32x4 (&s)[4], uint32_t ok) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (!(ok >> (4 * e + t) & 1)) s[t][e] = -INFINITY;
}

// Operands i = 2 b and 2 b + 1 of V^T for keys 16 g + 8 u ..: two channels of two keys per conversion
// pair, regrouped to two keys of a channel.
template <int b>
__device__ __forceinline__ void v_operands(const u32x4& w0, const u32x4& w1, const float (&sc)[8],
                                           u32x4& even, u32x4& odd) {
  uint32_t x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = kv4_bf16x2<b>(j < 4 ? w0[j] : w1[j - 4], sc[j]);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    even[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x05040100u);
    odd[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], 0x07060302u);
  }
}

// P V of a block in registers.
template <int R>
__device__ __forceinline__ void pv_step(Rows<R>& st, const Block& blk, const u32x4 (&p)[R][2],
                                        uint32_t ok) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int r = 0; r < R; ++r) st.l[r] = add_sums(st.l[r], p[r][u]);
    float sc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      sc[j] = __uint_as_float(((blk.vs[2 * u + j / 4] >> (8 * (j % 4))) & 255u) << 23);
    if (__any(ok != 0xffffu)) {
      // a key that does not count has probability 0, but its scale byte may be anything
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!(ok >> (8 * u + j) & 1)) sc[j] = 1.f;
    }
    auto pair = [&](auto b) {
      constexpr int kB = decltype(b)::value;
      u32x4 even, odd;
      v_operands<kB>(blk.v[2 * u], blk.v[2 * u + 1], sc, even, odd);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        st.o[r][2 * kB] = mfma16(as_bf16x8(even), as_bf16x8(p[r][u]), st.o[r][2 * kB]);
        st.o[r][2 * kB + 1] = mfma16(as_bf16x8(odd), as_bf16x8(p[r][u]), st.o[r][2 * kB + 1]);
      }
    };
    pair(std::integral_constant<int, 0>{});
    pair(std::integral_constant<int, 1>{});
    pair(std::integral_constant<int, 2>{});
    pair(std::integral_constant<int, 3>{});
  }
}

// One K operand (byte t of ks: its scales) times the digits of summed queries, whose row 8 hh + p is digit p
// of head hh: lane (c, g) gets digits 4 g .. 4 g + 3 of key 4 c + t, summed.
template <int t>
__device__ __forceinline__ float digits_k(i32x8 digits, int scale, u32x4 k, uint32_t ks) {
  const i32x8 b = {static_cast<int>(k.x), static_cast<int>(k.y), static_cast<int>(k.z),
                   static_cast<int>(k.w), 0, 0, 0, 0};
  const f32x4 s = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      digits, b, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 4, 0, scale, t, static_cast<int>(ks));
  return (s[3] + s[2]) + (s[1] + s[0]);
}

// x + y of lane ^ 16: of x in the even lane groups, of y in the odd ones.
__device__ __forceinline__ float fold16(float x, float y) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The raw importance of a block's keys for the two heads of one operand: lane (c, g) writes keys 4 c +
// 2 (g % 2) and the next of head g / 2, at dst (bits 0, 1 of ok: they count).
__device__ __forceinline__ void importance_step(const u32x4 (&k)[4], uint32_t ks, i32x8 digits,
                                                int scale, uint32_t ok, float* dst) {
  const float s0 = digits_k<0>(digits, scale, k[0], ks), s1 = digits_k<1>(digits, scale, k[1], ks);
  const float s2 = digits_k<2>(digits, scale, k[2], ks), s3 = digits_k<3>(digits, scale, k[3], ks);
  const f32x2 two = {fold16(s0, s2), fold16(s1, s3)};
  if (ok == 3) {
    *reinterpret_cast<f32x2*>(dst) = two;
  } else {
    if (ok & 1) dst[0] = two[0];
    if (ok & 2) dst[1] = two[1];
  }
}

// Tables read at workgroup-uniform places go through the scalar cache: their waits are not queued behind
// the blocks' loads, which return in order.
__device__ __forceinline__ int scalar_at(const int32_t* p, int64_t i) {
  typedef const __attribute__((address_space(4))) int32_t* cptr;
  return reinterpret_cast<cptr>(reinterpret_cast<uintptr_t>(p))[i];
}

// What a workgroup does: part x item x range of rows x K/V head. Workgroup i runs on XCD i % 8, and an XCD's
// workgroups go round its compute units.
//  * The parts come slowest, so that every XCD gets the same mix of parts (24 sequences of 1000-32768 keys
//    in 8 parts: 115 us with the parts fastest, where an XCD had one part of all of them and the last
//    parts are mostly empty; 88 so).
//  * Verify blocks of uneven length: the row ranges of a block side by side, so that a long one's spread
//    over the compute units (six blocks of 537-2395 keys in 8 ranges: 96 us with the ranges slowest,
//    where some units have two of the longest; 84 so).
//  * Tiles: the ranges slowest, since a mixed launch's tiles of few rows leave theirs empty (32 sequences
//    of up to 1516 keys, six of them whole: 204 us, with the ranges side by side 208).
template <bool kVerify>
struct Unit {
  int z, kvh, y;
  int64_t item;
  __device__ __forceinline__ explicit Unit(const Kv4Args& a) {
    uint32_t i = blockIdx.x;
    kvh = i % a.kv_heads;
    i /= a.kv_heads;
    if constexpr (kVerify) {
      y = i % a.n_ranges;
      i /= a.n_ranges;
    }
    item = i % a.n_items;
    i /= a.n_items;
    z = kVerify ? i : i % a.n_parts;
    if constexpr (!kVerify) y = i / a.n_parts;
  }
};

// A work item (or verify block) as a workgroup sees it: its query rows and key range, checked against
// the tables; rows == 0: nothing to do.
struct Tile {
  int batch, rows, n_imp;
  int64_t roff;
  int k_begin, k_end;  // positions are 32-bit, as in the work items
  int b_first, n_blk;  // 64-key blocks
  int parts;
};
__device__ __forceinline__ Tile read_tile(const Kv4Args& a, int64_t item) {
  const int32_t* it = a.work + 8 * item;
  Tile t;
  t.batch = scalar_at(it, 0);
  t.k_begin = max(scalar_at(it, 1), 0);
  t.k_end = static_cast<int>(min(int64_t(scalar_at(it, 2)), a.max_pages << a.page_log2));
  t.roff = scalar_at(it, 3);
  t.rows = min(scalar_at(it, 4), a.tile_rows);
  t.n_imp = min(scalar_at(it, 5), t.rows);
  if (t.batch < 0 || t.batch >= a.n_seq || t.roff < 0 || t.rows < 0 || t.roff + t.rows > a.n_row_idx)
    t.rows = 0;
  t.b_first = t.k_begin / kBlockKeys;
  t.n_blk = t.k_end > t.k_begin ? (t.k_end - 1) / kBlockKeys + 1 - t.b_first : 0;
  t.parts = min(a.n_parts, (t.n_blk - 1) / a.part_blocks + 1);  // 1 without keys
  return t;
}

// A verify block: roff its first query row, k_begin its first key in the list, k_end the number of its cache
// keys, n_blk the 64-key blocks of its own rows and of its cache keys, in this order.
__device__ __forceinline__ Tile read_vblock(const Kv4Args& a, int64_t item) {
  const int32_t* it = a.vblocks + 4 * item;
  const int k0 = scalar_at(it, 0), k1 = scalar_at(it, 1), q0 = scalar_at(it, 2), q1 = scalar_at(it, 3);
  Tile t = {};
  if (q0 < 0 || q1 <= q0 || q1 > a.n_q_rows || k0 < 0 || k1 > a.n_keys) return t;
  t.rows = min(q1 - q0, a.tile_rows);
  t.roff = q0;
  t.k_begin = k0;
  t.k_end = max(k1 - k0, 0);
  t.n_blk = (t.rows + kBlockKeys - 1) / kBlockKeys + (t.k_end + kBlockKeys - 1) / kBlockKeys;
  t.parts = min(a.n_parts, (t.n_blk - 1) / a.part_blocks + 1);
  return t;
}

// Partial result of row `row` of an item for head `head` in part z.
__device__ __forceinline__ float* part_record(const Kv4Args& a, int z, int64_t item, int row, int head) {
  return a.part + (((int64_t(z) * a.n_items + item) * a.tile_rows + row) * a.heads + head) * kPartFloats;
}

// Logical 16-key cells of a tile -> physical cells. Cells past the tile's keys read its own ends (a tile
// without keys the first page), so every table and cache access is in range; a page outside the cache
// gives -1.
struct Pages {
  const int32_t* table;
  int c_first, c_last;
  int64_t n_cells;
  int cell_log2;  // cells per page
  __device__ __forceinline__ Pages(const Kv4Args& a, const Tile& t)
      : table(a.page_table + int64_t(t.batch) * a.max_pages),
        c_first(t.n_blk ? t.k_begin / kCellSlots : 0),
        c_last(t.n_blk ? (t.k_end - 1) / kCellSlots : 0),
        n_cells(a.n_slots / kCellSlots),
        cell_log2(a.page_log2 - 4) {}
  // physical cell of a workgroup-uniform logical cell
  __device__ __forceinline__ int phys(int cell) const {
    cell = min(max(cell, c_first), c_last);
    const int page = scalar_at(table, cell >> cell_log2);
    const int64_t p = (int64_t(page) << cell_log2) | (cell & ((1 << cell_log2) - 1));
    return page < 0 || p >= n_cells ? -1 : static_cast<int>(p);
  }
};

// Bits of the keys of logical cell `cell` inside [k_begin, k_end).
__device__ __forceinline__ uint32_t keys_of(const Tile& t, int cell) {
  const int key0 = kCellSlots * cell;  // at most 47 past k_end, which the last block's end is not
  const int lo = min(max(t.k_begin - key0, 0), kCellSlots);
  const int hi = min(max(t.k_end - key0, 0), kCellSlots);
  return ((1u << hi) - 1) & ~((1u << lo) - 1);
}

constexpr int kFragInts = 12;  // a lane's digits (8), their scale, padding to 16 bytes
__host__ __device__ constexpr int imp_frag_bytes(int group) { return (group + 1) / 2 * 64 * kFragInts * 4; }

// Leaves the operands of the tile's importance in `frags`: the digits of each head's queries summed over
// the first n_imp rows in 32 bits. `tmp`: 32 * threads bytes. Every thread of the workgroup comes here.
template <int kThreads>
__device__ __forceinline__ void importance_operands(const Kv4Args& a, const Tile& t, int kvh,
                                                    float* tmp, int* frags) {
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int G = a.group;
  // 16 threads for a head's channels, the rows over the rest
  const int splits = kThreads / 16 / G, at = tid / 16 % G, sp = tid / 16 / G, ch = 8 * (tid % 16);
  if (sp < splits) {
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    constexpr int kRows = 4;  // asked for at once
    for (int r = sp; r < t.n_imp; r += kRows * splits) {
      int64_t row[kRows];
      u32x4 w[kRows];
#pragma unroll
      for (int x = 0; x < kRows; ++x) row[x] = a.row_idx[t.roff + min(r + x * splits, t.n_imp - 1)];
#pragma unroll
      for (int x = 0; x < kRows; ++x) {
        if (r + x * splits >= t.n_imp || row[x] >= a.n_q_rows) row[x] = -1;
        w[x] = ld16(a.q + (max(row[x], int64_t(0)) * a.heads + kvh * G + at) * kHeadDim + ch);
      }
#pragma unroll
      for (int x = 0; x < kRows; ++x) {
        if (row[x] < 0) w[x] = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[2 * j] += __uint_as_float(w[x][j] << 16);
          sum[2 * j + 1] += __uint_as_float(w[x][j] & 0xffff0000u);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) tmp[(sp * G + at) * kHeadDim + ch + j] = sum[j];
  }
  __syncthreads();
  for (int i = tid; i < G * kHeadDim; i += kThreads) {  // only this thread reads and writes element i
    float sum = tmp[i];
    for (int s = 1; s < splits; ++s) sum += tmp[s * G * kHeadDim + i];
    tmp[i] = sum;
  }
  __syncthreads();
  for (int pr = tid / 64; pr < (G + 1) / 2; pr += kThreads / 64) {
    const int head = 2 * pr + c / 8, digit = c % 8;
    float x[32];
#pragma unroll
    for (int j = 0; j < 32; ++j)
      x[j] = head < G ? tmp[head * kHeadDim + 16 * g + j % 16 + 64 * (j / 16)] : 0.f;
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < 32; ++j) top = fmaxf(top, fabsf(x[j]));
    const int e = q_scale(xmax(top));
    // below 8, then in units of 16^-6: integers below 2^27, whose digits are those of the number with 8
    // added at every place, less 8 (the first keeps what is above it)
    const float to_int = exp2i(249 - e) * 0x1p24f;
    int* f = frags + (pr * 64 + lane) * kFragInts;
    const int at = 4 * max(kImpDigits - 1 - digit, 0);
    uint32_t odd = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float y = x[4 * j + i];
        odd |= !__builtin_isfinite(y);
        const uint32_t n = static_cast<uint32_t>(__float2int_rn(y * to_int)) + 0x8888888u;
        const int v = static_cast<int>(digit == 0 ? n >> 4 * (kImpDigits - 1) : n >> at & 15u) - 8;
        d[i] = digit < kImpDigits ? static_cast<float>(v) : 0.f;
      }
      const int w = __builtin_amdgcn_cvt_pk_fp8_f32(d[0], d[1], 0, false);
      f[j] = __builtin_amdgcn_cvt_pk_fp8_f32(d[2], d[3], w, true);
    }
    f[8] = odd ? 255 : max(e + 5 - 4 * digit, 0);  // 255: NaN, whatever the digits
  }
  __syncthreads();
}

// A wavefront's importance of one block: ok and cell (-1: no page) of the cell of the lane's keys, c / 4.
__device__ __forceinline__ void importance_block(const Kv4Args& a, const u32x4 (&k)[4], uint32_t ks,
                                                 const int* frags, int kvh, int lane, uint32_t ok,
                                                 int cell) {
  const int c = lane & 15, g = lane >> 4, G = a.group;
  const int key = 4 * (c & 3) + 2 * (g & 1);
  for (int pr = 0; pr < (G + 1) / 2; ++pr) {
    const int* f = frags + (pr * 64 + lane) * kFragInts;
    i32x8 digits;
#pragma unroll
    for (int x = 0; x < 8; ++x) digits[x] = f[x];
    const int head = 2 * pr + (g >> 1);
    float* dst = a.imp_part + (int64_t(kvh) * G + min(head, G - 1)) * a.n_slots +
                 int64_t(max(cell, 0)) * kCellSlots + key;
    importance_step(k, ks, digits, f[8], head < G ? ok >> key & 3 : 0u, dst);
  }
}

// The same for one K operand t (byte 0 of ks: its scales), key 4 c + t of the block to a lane: the share of a
// wavefront where four hold the block.
__device__ __forceinline__ void importance_share(const Kv4Args& a, u32x4 k, uint32_t ks, int t,
                                                 const int* frags, int kvh, int lane, uint32_t ok,
                                                 int cell) {
  const int c = lane & 15, g = lane >> 4, G = a.group;
  const int key = 4 * (c & 3) + t;
  for (int pr = 0; pr < (G + 1) / 2; ++pr) {
    const int* f = frags + (pr * 64 + lane) * kFragInts;
    i32x8 digits;
#pragma unroll
    for (int x = 0; x < 8; ++x) digits[x] = f[x];
    const float s = digits_k<0>(digits, f[8], k, ks);
    const float sum = fold16(s, s);
    const int head = 2 * pr + (g >> 1);
    if (!(g & 1) && head < G && (ok >> key & 1))
      a.imp_part[(int64_t(kvh) * G + head) * a.n_slots + int64_t(max(cell, 0)) * kCellSlots + key] = sum;
  }
}

// 1 / the sum of a row's probabilities; 0 without any key, so that such rows are zeros.
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// ---- up to 32 rows: every wavefront takes blocks of its own

constexpr int kWaves = 4;

// Bound by memory where there are many keys: 24 tokens of 32 heads over 368403 keys of 8 heads in 85 us (401
// MB, 4.7 TB/s; 0.22 of the wavefronts' cycles issue vector work), 32 rows of 32 heads over 65501 keys in 63
// (4.6 TB/s), 67-71 with the importance, whose 4 MFMAs and 20 additions a block no longer hide; by the chain
// of loads at its start and by the merge for few (2011 keys: 6.4 us + 3 of merging).
//
// R x 16 rows per workgroup. Lane (c, g) ends with channels 32 g + 8 e + i of query c in o[.][i][e]: the
// i-th V^T operand's row m is channel 8 m + i, i.e. word m of a key's codes.
template <int R, bool kImp>
__global__ __launch_bounds__(64 * kWaves, R == 1 ? 3 : 2) void kv4_wave_kernel(Kv4Args a) {
  constexpr int kRowBytes = kWaves * R * 64 * 8 * 16;  // the merge's O, then its (m, l)
  constexpr int kMerge = kRowBytes + kWaves * R * 64 * 8;
  extern __shared__ __align__(16) uint8_t smem[];  // kMerge, then the importance operands
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c = lane & 15, g = lane >> 4;

  const Unit<false> u(a);
  const int z = u.z, kvh = u.kvh;
  const Tile t = read_tile(a, u.item);
  const int G = a.group;
  const int m0 = u.y * 16 * R;
  if (m0 >= t.rows * G || (z > 0 && z >= t.parts)) return;
  const int b_lo = t.b_first + z * a.part_blocks;
  const int b_hi = z + 1 >= t.parts ? t.b_first + t.n_blk : b_lo + a.part_blocks;

  const Pages pages(a, t);
  // physical cells of the lane: of K (keys 4 c ..) and of V (keys 16 g ..)
  auto pick = [](int i, int x0, int x1, int x2, int x3) {
    const int lo = i & 1 ? x1 : x0, hi = i & 1 ? x3 : x2;
    return i & 2 ? hi : lo;
  };
  auto cells_of = [&](int i, int& kcell, int& vcell) __attribute__((always_inline)) {
    const int x0 = pages.phys(4 * i), x1 = pages.phys(4 * i + 1), x2 = pages.phys(4 * i + 2),
              x3 = pages.phys(4 * i + 3);
    kcell = pick(c >> 2, x0, x1, x2, x3);
    vcell = pick(g, x0, x1, x2, x3);
  };
  auto load_k = [&](Block& blk, int cell) __attribute__((always_inline)) {
    const uint8_t* p = a.cache + (int64_t(max(cell, 0)) * a.kv_heads + kvh) * kCellBytes;
    const int s = 4 * (c & 3);
#pragma unroll
    for (int y = 0; y < 4; ++y) blk.k[y] = ld16(p + 64 * (s + y) + 16 * g);
    blk.ks = *reinterpret_cast<const uint32_t*>(p + kCellKs + 16 * g + s);
  };
  auto load_v = [&](Block& blk, int cell) __attribute__((always_inline)) {
    const uint8_t* p = a.cache + (int64_t(max(cell, 0)) * a.kv_heads + kvh) * kCellBytes;
#pragma unroll
    for (int y = 0; y < 4; ++y) blk.v[y] = ld16(p + kCellV + 256 * y + 16 * c);
    blk.vs = ld16(p + kCellVs + 16 * (c >> 2));
  };
  // The first block's loads go out before the queries'. A block's registers are loaded anew as soon as
  // its K, then its V is used: one block per wavefront on its way, and registers for more wavefronts.
  // Loads are never skipped, only repeated past the end: a wait behind a load that may not have been
  // issued would wait for everything.
  int i = b_lo + wave;
  Block blk;
  int kcell, vcell, knext, vnext;
  cells_of(i, kcell, vcell);
  load_k(blk, kcell);
  load_v(blk, vcell);
  cells_of(i + kWaves, knext, vnext);

  int64_t orow[R];  // row * heads + head, or -1
  QFrag q[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int m = m0 + r * 16 + c;
    orow[r] = -1;
    if (m < t.rows * G) {
      const int64_t row = a.row_idx[t.roff + m / G];
      if (row >= 0 && row < a.n_q_rows) orow[r] = row * a.heads + kvh * G + m % G;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    q[r] = load_q(a.q + max(orow[r], int64_t(0)) * kHeadDim, g, orow[r] >= 0);

  const bool imp = kImp && t.n_imp > 0 && m0 == 0;
  int* const frags = reinterpret_cast<int*>(smem + kMerge);
  if constexpr (kImp)
    if (imp) importance_operands<64 * kWaves>(a, t, kvh, reinterpret_cast<float*>(smem), frags);

  Rows<R> st;
  st.clear();
  for (; i < b_hi; i += kWaves) {
    const uint32_t ok = vcell < 0 ? 0u : keys_of(t, 4 * i + g);
    const bool edge = __any(ok != 0xffffu);
    float scale[R];
    f32x4 s[R][4];
    u32x4 p[R][2];
    logits<R>(blk.k, blk.ks, q, s);
    if constexpr (kImp)
      if (imp)
        importance_block(a, blk.k, blk.ks, frags, kvh, lane,
                         !edge ? 0xffffu : kcell < 0 ? 0u : keys_of(t, 4 * i + (c >> 2)), kcell);
    load_k(blk, knext);
    if (edge)
#pragma unroll
      for (int r = 0; r < R; ++r) hide(s[r], ok);
#pragma unroll
    for (int r = 0; r < R; ++r) scale[r] = raise_maxima<R>(st, r, s[r], a.scale_log2);
#pragma unroll
    for (int r = 0; r < R; ++r) probabilities(s[r], scale[r], st.m[r], p[r]);
    pv_step<R>(st, blk, p, ok);
    load_v(blk, vnext);
    kcell = knext;
    vcell = vnext;
    cells_of(i + 2 * kWaves, knext, vnext);
  }

  // merge the wavefronts: each leaves (m, l) and O in LDS, then finishes e = wave
  static_assert(kWaves == 4, "one e to a wavefront");
  f32x2* const ml = reinterpret_cast<f32x2*>(smem + kRowBytes);
  f32x4* const os = reinterpret_cast<f32x4*>(smem);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    ml[(wave * R + r) * 64 + lane] = f32x2{st.m[r], st.l[r][0]};
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        os[(((wave * R + r) * 4 + e) * 2 + h) * 64 + lane] =
            f32x4{st.o[r][4 * h][e], st.o[r][4 * h + 1][e], st.o[r][4 * h + 2][e],
                  st.o[r][4 * h + 3][e]};
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (orow[r] < 0) continue;
    float m = -INFINITY, l = 0.f, w[kWaves];
#pragma unroll
    for (int x = 0; x < kWaves; ++x) m = fmaxf(m, ml[(x * R + r) * 64 + lane][0]);
    const float base = m == -INFINITY ? 0.f : m;
    float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      const f32x2 v = ml[(x * R + r) * 64 + lane];
      w[x] = fast_exp2(v[0] - base);
      l = __builtin_fmaf(w[x], v[1], l);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 y = os[(((x * R + r) * 4 + wave) * 2 + h) * 64 + lane];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[4 * h + k] = __builtin_fmaf(w[x], y[k], o[4 * h + k]);
      }
    }
    const int ch = 32 * g + 8 * wave;
    if (t.parts > 1) {
      const int mi = m0 + r * 16 + c;
      float* rec = part_record(a, z, u.item, mi / G, kvh * G + mi % G);
      *reinterpret_cast<f32x4*>(rec + ch) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(rec + ch + 4) = f32x4{o[4], o[5], o[6], o[7]};
      if (ch == 0) *reinterpret_cast<f32x2*>(rec + kHeadDim) = f32x2{m, l};
    } else {
      const float inv = inverse(l);
      st16(a.out + orow[r] * kHeadDim + ch,
           u32x4{pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv),
                 pack2(o[4] * inv, o[5] * inv), pack2(o[6] * inv, o[7] * inv)});
    }
  }
}

// ---- more rows, and verify: the wavefronts of a workgroup share each block

// LDS of kv4_tile_kernel: kBufs blocks' V as bf16 [64 keys][128 channels], their K codes, K scales and the
// keys that count, then the importance operands.
//   V  16-byte chunk w (channels 8 w ..) of key n at chunk pair (w / 2) ^ v_swizzle(n): a transposing
//      read takes one chunk pair of the keys 16 g + n0 .. n0 + 3, g = 0..3: 16 rows over 8 pair places.
//   K  16-byte part g of key 4 c + t at ((t * 16 + c) * 4 + g) * 16: operand t is 1 KB in lane order.
constexpr int kBufs = 2;  // being multiplied, being filled
constexpr int kVBuf = kBlockKeys * kHeadDim * 2, kKBuf = kBlockKeys * 64;
constexpr int kLdsK = kBufs * kVBuf, kLdsKs = kLdsK + kBufs * kKBuf, kLdsOk = kLdsKs + kBufs * 256;
constexpr int kLdsCell = kLdsOk + kBufs * 16, kLdsFrags = kLdsCell + kBufs * 16;
constexpr int kSlotKeys = 2048;  // verify: keys whose slots are in LDS (in the place of the operands)
__device__ __forceinline__ int v_swizzle(int n) { return (n & 3) | ((n >> 4 & 1) << 2); }
__device__ __forceinline__ int v_chunk(int n, int w) {
  return (16 * n + (((w >> 1) ^ v_swizzle(n)) << 1 | (w & 1))) * 16;
}

// P V from a V buffer: operand i's row m is channel 16 i + m. In each 16-lane group, source lane s of a
// transposing read brings 4 channels of key n0 + s / 4 and lane m receives the 4 keys of channel m. All
// operands for one half of the keys, then for the other: an MFMA that adds to the result of the last
// but one waits for it (30 cycles instead of 20).
template <int R>
__device__ __forceinline__ void pv_lds(Rows<R>& st, const uint8_t* vbuf, const u32x4 (&p)[R][2], int c,
                                       int g) {
  const int n0 = 16 * g + (c >> 2);
  const uint8_t* row = vbuf + 256 * n0 + 8 * (c & 3);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int r = 0; r < R; ++r) st.l[r] = add_sums(st.l[r], p[r][u]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint8_t* at = row + 32 * (i ^ v_swizzle(n0)) + 2048 * u;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(lds_ptr)(at));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) s16x4*)(lds_ptr)(at + 1024));
      const bf16x8 v = as_bf16x8(__builtin_bit_cast(u32x2, lo), __builtin_bit_cast(u32x2, hi));
#pragma unroll
      for (int r = 0; r < R; ++r) st.o[r][i] = mfma16(v, as_bf16x8(p[r][u]), st.o[r][i]);
    }
  }
}

// Bits 0..15 of the keys at .. at + 15 that lie below `end`.
__device__ __forceinline__ uint32_t below(int end, int at) {
  return (1u << min(max(end - at, 0), 16)) - 1u;
}

// Bit j: key `at` + j (j = 0..15) of a verify block of n_in rows is seen by row r: a row of the mask, or the
// closed form with T fill, S draft and S mask rows, where a row sees all but a run of S keys (fill
// rows: the drafts; draft i: drafts past i and masks up to i; mask i: drafts from i and masks before i).
__device__ __forceinline__ uint32_t seen_keys(const Kv4Args& a, int64_t vb, int T, int S, int r, int n_in,
                                              int at) {
  if (a.vmeta) {
    const int lo = r < T ? T : r < T + S ? r + 1 : min(r - S, T + S);
    const int hi = r < T ? T + S : r < T + S ? r + S + 1 : r;
    return below(n_in, at) & (below(lo, at) | (below(hi, at) ^ 0xffffu));
  }
  const uint8_t* row = a.mask + (vb * a.tile_rows + r) * a.tile_rows + at;
  uint32_t bits = 0;
  if (at + 16 <= a.tile_rows) {
    uint32_t w[4];
    __builtin_memcpy(w, row, 16);  // of any alignment
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      // bit 8 t where byte t is not 0, then bit t
      const uint32_t x = (((w[e] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[e]) >> 7 & 0x01010101u;
      bits |= (x * 0x01020408u >> 24 & 15u) << (4 * e);
    }
  } else {
    for (int j = 0; j < 16 && at + j < a.tile_rows; ++j) bits |= uint32_t(row[j] != 0) << j;
  }
  return bits & below(n_in, at);
}

// The verify block's own 64 keys from ib * 64 on: K (bf16) in kbuf, channels 32 g + 8 x .. of key 4 c + t at
// ((t * 16 + 4 x + g) * 16 + c) * 16, V in vbuf as above with its NaNs and infinities left out (`odd`: there
// are some): 0 times them would reach rows that do not see the key.
template <int R>
__device__ __forceinline__ void own_keys(const Kv4Args& a, Rows<R>& st, const QFrag (&q)[R],
                                         const int (&qi)[R], int64_t q0, int n_in, int64_t vb,
                                         int kvh, int T, int S, int ib, bool odd,
                                         const uint8_t* kbuf, const uint8_t* vbuf, int c, int g) {
  const int j0 = kBlockKeys * ib;
  f32x4 s[R][4];
  u32x4 p[R][2];
  uint32_t seen[R];  // bit 4 e + t: the lane's query sees key j0 + 16 g + 4 e + t
#pragma unroll
  for (int r = 0; r < R; ++r) {
    seen[r] = seen_keys(a, vb, T, S, qi[r], n_in, j0 + 16 * g);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      s[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < 4; ++x)
        s[r][t] = mfma16(as_bf16x8(ld16(kbuf + ((t * 16 + 4 * x + g) * 16 + c) * 16)),
                         as_bf16x8(q[r].x[x]), s[r][t]);
    }
    hide(s[r], seen[r]);
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float scale = raise_maxima<R>(st, r, s[r], a.scale_log2);
    probabilities(s[r], scale, st.m[r], p[r]);
  }
  pv_lds<R>(st, vbuf, p, c, g);
  if (!odd) return;
  // P times the values left out, for the rows that see the key
#pragma unroll
  for (int j = 0; j < 16; ++j)
    for (int gg = 0; gg < 4; ++gg) {
      const int key = j0 + 16 * gg + j;
      if (key >= n_in) continue;  // the same in every lane
      const uint16_t* vp = a.vblk + ((q0 + key) * a.kv_heads + kvh) * kHeadDim + 4 * g;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const uint32_t w = p[r][j / 8][j % 8 / 2];
        const float pj = bf2f(static_cast<uint16_t>(__shfl(w, 16 * gg + c) >> (16 * (j % 2))));
        const bool vis = __shfl(seen[r], 16 * gg + c) >> j & 1;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const u32x2 x = ld8(vp + 16 * i);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = __uint_as_float(e % 2 ? x[e / 2] & 0xffff0000u : x[e / 2] << 16);
            if (vis && !__builtin_isfinite(v)) st.o[r][i][e] += pj * v;
          }
        }
      }
    }
}

// Bound by issue and power: 8 x 1024 rows and keys of 32 heads in 158 us (0.87 PFLOP/s; MFMAs busy 0.35 of
// the cycles, LDS 0.20, vector instructions 0.3 of the wavefronts'). Verify over 16 x 64 rows and 946-978
// gathered keys of 32 heads: 45.5 us, of which 11 for the own keys and the start. Tried with K on the scaled
// MFMA, where the first took 150-165 us in one run or another: no maximum per block 168, wavefront
// priorities 159-166; 32 rows to a wavefront with the blocks halved between two pairs of wavefronts 45 for
// 47 us of the second, and 15.8 for 14.9 with one sequence of 264 keys.
//
// 16 R rows to a wavefront. A wavefront brings its cell of each block; kAhead blocks are in registers, on
// their way, and two are in LDS. Four wavefronts of up to 32 rows, so that workgroups of different phases
// share a compute unit: eight in one workgroup took 163 us on 8 x 1024 rows and keys of 32 heads where
// four took 156 (K on the scaled MFMA), also with half of them a phase behind the others (172).
template <int R, int kAhead, bool kImp, bool kVerify>
__global__ __launch_bounds__(64 * kWaves, 2) void kv4_tile_kernel(Kv4Args a) {
  static_assert(kAhead == 2 || kAhead == 4, "the buffers alternate, the ring is a power of two");
  extern __shared__ __align__(16) uint8_t smem[];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int c = lane & 15, g = lane >> 4;

  const Unit<kVerify> unit(a);
  const int z = unit.z, kvh = unit.kvh;
  const int64_t item = unit.item;
  const int G = a.group;
  const Tile t = kVerify ? read_vblock(a, item) : read_tile(a, item);
  const int m0 = unit.y * 16 * R * kWaves;
  if (m0 >= t.rows * G || (z > 0 && z >= t.parts)) return;
  int b_lo = t.b_first + z * a.part_blocks;
  int b_hi = z + 1 >= t.parts ? t.b_first + t.n_blk : b_lo + a.part_blocks;
  // verify: own keys from own_lo to own_hi, then cache blocks
  const int64_t q0 = t.roff, k0 = t.k_begin;
  const int n_list = t.k_end;
  int own_lo = 0, own_hi = 0;
  if constexpr (kVerify) {
    const int n_own = (t.rows + kBlockKeys - 1) / kBlockKeys;
    own_lo = min(b_lo, n_own);
    own_hi = min(b_hi, n_own);
    b_lo = max(b_lo - n_own, 0);
    b_hi = max(b_hi - n_own, 0);
  }

  // ---- a thread's share of a block: of cell `own` 16 bytes of the K of slot kslot, and of V the words vw
  // of quad vq as they are stored (verify, where every key has a cell of its own: words 4 kpart .. of kslot)
  const int own = wave, kslot = lane >> 2, kpart = lane & 3;
  const int kc = 4 * own + (kslot >> 2), kt = kslot & 3;  // key 4 kc + kt of the block
  const int vw = lane & 15, vq = lane >> 4;
  const Pages pages(a, t);
  int* const slots = reinterpret_cast<int*>(smem + kLdsFrags);  // verify: of keys from s_first on
  int s_first = 0;
  struct Share {
    u32x4 k, v;
    uint32_t ks, vs, ok;  // ok: bit j: key j of the quad counts (verify: bit j: of the cell)
    int cell;             // physical, -1 for none
  };
  const uint8_t* const head0 = a.cache + kvh * kCellBytes;
  const uint32_t cell_bytes = a.kv_heads * kCellBytes;
  auto cell_at = [&](int cell) {
    return head0 + uint64_t(uint32_t(max(cell, 0))) * cell_bytes;
  };
  // verify: the slot of this thread's key of block i
  auto slot_of = [&](int i) { return slots[kBlockKeys * i - s_first + 16 * own + kslot]; };
  // Requests are never skipped, only repeated past the end: a wait behind a load that may not have been
  // issued would wait for everything.
  auto request = [&](Share& s, int i, int cell) __attribute__((always_inline)) {
    if constexpr (kVerify) {
      const int x = max(cell, 0);  // (a slot)
      const uint8_t* p = cell_at(x >> 4);
      s.k = ld16(p + 64 * (x & 15) + 16 * kpart);
      const uint8_t* v = p + kCellV + 64 * (x & 12) + 4 * (x & 3) + 64 * kpart;
#pragma unroll
      for (int j = 0; j < 4; ++j) s.v[j] = *reinterpret_cast<const uint32_t*>(v + 16 * j);
      const uint8_t* sc = p + kCellKs + 16 * kpart + (x & 15);
      s.ks = sc[0];
      s.vs = sc[kCellVs - kCellKs];
      s.ok = cell >= 0;
    } else {
      const uint8_t* p = cell_at(cell);
      s.k = ld16(p + 16 * lane);
      s.ks = *reinterpret_cast<const uint32_t*>(p + kCellKs + 16 * kpart + (kslot & 12));
      s.v = ld16(p + kCellV + 16 * lane);
      s.vs = *reinterpret_cast<const uint32_t*>(p + kCellVs + 16 * (vw >> 2) + 4 * vq);
      s.ok = cell < 0 ? 0u : keys_of(t, 4 * i + own) >> (4 * vq) & 15u;
      s.cell = cell;
    }
  };
  // into buffer b: K as stored, V as bf16 (zeros for keys that do not count); lanes of the same place
  // write the same value
  auto put = [&](const Share& s, int b) __attribute__((always_inline)) {
    st16(smem + kLdsK + kKBuf * b + ((kt * 16 + kc) * 4 + kpart) * 16, s.k);
    if constexpr (kVerify)
      smem[kLdsKs + 256 * b + (kc * 4 + kpart) * 4 + kt] = static_cast<uint8_t>(s.ks);
    else
      *reinterpret_cast<uint32_t*>(smem + kLdsKs + 256 * b + (kc * 4 + kpart) * 4) = s.ks;
    u32x4 w = s.v;
    uint32_t vs = s.vs;
    if constexpr (kVerify) {
      uint64_t bits = __ballot(s.ok);
      if (bits != ~uint64_t(0)) {
        if (!s.ok) {
          w = u32x4{0, 0, 0, 0};
          vs = 0;
        }
        // bit 4 n, of key n, to bit n
        bits &= 0x1111111111111111u;
        bits = (bits | bits >> 3) & 0x0303030303030303u;
        bits = (bits | bits >> 6) & 0x000f000f000f000fu;
        bits = (bits | bits >> 12) & 0x000000ff000000ffu;
        bits |= bits >> 24;
      }
      *reinterpret_cast<uint32_t*>(smem + kLdsOk + 16 * b + 4 * own) = bits & 0xffffu;
    } else {
      if (__any(s.ok != 15u)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (!(s.ok >> j & 1)) {
            w[j] = 0;
            vs &= ~(255u << (8 * j));
          }
      }
      smem[kLdsOk + 16 * b + 4 * own + vq] = static_cast<uint8_t>(s.ok);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float sc = __uint_as_float(kVerify ? vs << 23 : (vs >> (8 * j) & 255u) << 23);
      st16(smem + kVBuf * b + (kVerify ? v_chunk(16 * own + kslot, 4 * kpart + j)
                                       : v_chunk(16 * own + 4 * vq + j, vw)),
           u32x4{kv4_bf16x2<0>(w[j], sc), kv4_bf16x2<1>(w[j], sc), kv4_bf16x2<2>(w[j], sc),
                 kv4_bf16x2<3>(w[j], sc)});
    }
    if constexpr (kImp) *reinterpret_cast<int*>(smem + kLdsCell + 16 * b + 4 * own) = s.cell;
  };

  // kAhead blocks are on their way in registers; verify starts when it has the slots
  Share share[kAhead];
  auto start = [&](int lo, int hi) {
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
      request(share[x], min(lo + x, hi - 1),
              kVerify ? slot_of(min(lo + x, hi - 1)) : pages.phys(4 * (lo + x) + own));
  };
  // verify: the slots of blocks lo .. hi - 1 into LDS, then their requests
  auto stage = [&](int lo, int hi) {
    s_first = kBlockKeys * lo;
    for (int x = tid; x < kBlockKeys * (hi - lo); x += 64 * kWaves) {
      int64_t sl = -1;
      if (s_first + x < n_list) sl = a.key_slots[k0 + s_first + x];
      slots[x] = sl < 0 || sl >= a.n_slots ? -1 : static_cast<int>(sl);
    }
    __syncthreads();
    start(lo, hi);
  };
  // verify: a thread's share of 64 of the block's own keys
  u32x4 own_k[4], own_v[4];
  const int64_t own_ld = int64_t(a.kv_heads) * kHeadDim;
  auto own_load = [&](int ib) __attribute__((always_inline)) {
    const int64_t base = q0 * own_ld + int64_t(kvh) * kHeadDim;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int kk = 64 * kWaves * x + tid;
      const int n = 4 * (kk >> 2 & 15) + (kk >> 8), cc = (kk & 3) + 4 * (kk >> 6 & 3);
      own_k[x] = ld16(a.kblk + base + min(kBlockKeys * ib + n, t.rows - 1) * own_ld + 8 * cc);
      own_v[x] = ld16(a.vblk + base + min(kBlockKeys * ib + (kk >> 4), t.rows - 1) * own_ld +
                      8 * (kk & 15));
    }
  };
  // verify: with one operand to a wavefront there are registers to ask for the own keys a step ahead, and
  // for the cache's first blocks to be on their way meanwhile (two: 103 us on six blocks of 256 rows of 4
  // query heads where waiting takes 95)
  constexpr bool kOwnAhead = R == 1;
  if constexpr (!kVerify) start(b_lo, b_hi);
  if constexpr (kVerify && kOwnAhead) own_load(own_lo);

  int64_t orow[R];
  int qi[R];  // row within the tile
  QFrag q[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int m = m0 + (wave * R + r) * 16 + c;
    orow[r] = -1;
    qi[r] = min(m / G, t.rows - 1);
    if (m < t.rows * G) {
      const int64_t row = kVerify ? q0 + qi[r] : int64_t(a.row_idx[t.roff + qi[r]]);
      if (row >= 0 && row < a.n_q_rows) orow[r] = row * a.heads + kvh * G + m % G;
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    q[r] = load_q(a.q + max(orow[r], int64_t(0)) * kHeadDim, g, orow[r] >= 0);
  const bool idle = m0 + wave * R * 16 >= t.rows * G;  // no rows: the wavefront only moves blocks

  const bool imp = kImp && t.n_imp > 0 && m0 == 0;
  int* const frags = reinterpret_cast<int*>(smem + kLdsFrags);
  if constexpr (kImp)
    if (imp) importance_operands<64 * kWaves>(a, t, kvh, reinterpret_cast<float*>(smem), frags);

  Rows<R> st;
  st.clear();
  constexpr int kChunk = kSlotKeys / kBlockKeys;
  if constexpr (kVerify) {
    // the block's own keys
    if (kOwnAhead && b_lo < b_hi) stage(b_lo, min(b_lo + kChunk, b_hi));
    const int T = a.vmeta ? a.vmeta[2 * item] : 0, S = a.vmeta ? a.vmeta[2 * item + 1] : 0;
    for (int ib = own_lo; ib < own_hi; ++ib) {
      bool odd = false;
      if constexpr (!kOwnAhead) own_load(ib);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int kk = 64 * kWaves * x + tid;
        const int n = 4 * (kk >> 2 & 15) + (kk >> 8), cc = (kk & 3) + 4 * (kk >> 6 & 3);
        st16(smem + kVBuf + ((n & 3) * 256 + (4 * (cc & 3) + (cc >> 2)) * 16 + (n >> 2)) * 16, own_k[x]);
        const int vn = kk >> 4, w = kk & 15;
        u32x4 v = own_v[x];
        if (kBlockKeys * ib + vn >= t.rows) v = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool lo = (v[j] & 0x7f80u) == 0x7f80u, hi = (v[j] & 0x7f800000u) == 0x7f800000u;
          odd = odd || lo || hi;
          v[j] &= (lo ? 0xffff0000u : ~0u) & (hi ? 0xffffu : ~0u);
        }
        st16(smem + v_chunk(vn, w), v);
      }
      odd = __syncthreads_or(odd);
      if (kOwnAhead && ib + 1 < own_hi) own_load(ib + 1);
      if (!idle)
        own_keys<R>(a, st, q, qi, q0, t.rows, item, kvh, T, S, ib, odd, smem + kVBuf, smem, c, g);
      __syncthreads();
    }
  }
  for (int lo = b_lo; lo < b_hi; lo += kVerify ? kChunk : b_hi - b_lo) {
    const int hi = kVerify ? min(lo + kChunk, b_hi) : b_hi;
    if constexpr (kVerify)
      if (!kOwnAhead || lo != b_lo) stage(lo, hi);
    // cell or slot of the next request
    auto place = [&](int i) {
      return kVerify ? slot_of(min(i, hi - 1)) : pages.phys(4 * min(i, hi - 1) + own);
    };
    int cell = place(lo + kAhead);
    auto fill = [&](Share& sh, int i, int b) __attribute__((always_inline)) {
      put(sh, b);
      request(sh, min(i + kAhead, hi - 1), cell);
      cell = place(i + kAhead + 1);
    };
    auto keys_ok = [&](int b, int cell) {
      const uint32_t x = *reinterpret_cast<const uint32_t*>(smem + kLdsOk + 16 * b + 4 * cell);
      if constexpr (kVerify) return x;
      return (x & 15u) | (x >> 4 & 0xf0u) | (x >> 8 & 0xf00u) | (x >> 12 & 0xf000u);
    };
    auto read_k = [&](u32x4 (&k)[4], uint32_t& ks, int b) __attribute__((always_inline)) {
#pragma unroll
      for (int y = 0; y < 4; ++y)
        k[y] = ld16(smem + kLdsK + kKBuf * b + ((y * 16 + c) * 4 + g) * 16);
      ks = *reinterpret_cast<const uint32_t*>(smem + kLdsKs + 256 * b + (c * 4 + g) * 4);
    };
    // a wavefront's share of a block's importance: K operand `wave`
    auto importance = [&](int b) {
      const u32x4 k = ld16(smem + kLdsK + kKBuf * b + ((wave * 16 + c) * 4 + g) * 16);
      const uint32_t ks = smem[kLdsKs + 256 * b + (c * 4 + g) * 4 + wave];
      importance_share(a, k, ks, wave, frags, kvh, lane, keys_ok(b, c >> 2),
                       *reinterpret_cast<const int*>(smem + kLdsCell + 16 * b + 4 * (c >> 2)));
    };
    fill(share[0], lo, 0);
    __syncthreads();
    for (int base = lo; base < hi; base += kAhead) {
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int i = base + x;
        if (i >= hi) break;
        const int b = x & 1;
        fill(share[(x + 1) & (kAhead - 1)], i + 1, b ^ 1);
        if (!idle) {
          u32x4 k[4], p[R][2];
          uint32_t ks;
          f32x4 s[R][4];
          read_k(k, ks, b);
          const uint32_t ok = keys_ok(b, g);
          const bool edge = __any(ok != 0xffffu);
          logits<R>(k, ks, q, s);
          if (edge)
#pragma unroll
            for (int r = 0; r < R; ++r) hide(s[r], ok);
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const float scale = raise_maxima<R>(st, r, s[r], a.scale_log2);
            probabilities(s[r], scale, st.m[r], p[r]);
          }
          pv_lds<R>(st, smem + kVBuf * b, p, c, g);
        }
        if constexpr (kImp)
          if (imp) importance(b);
        __syncthreads();
      }
    }
  }
  // lane (c, g): channels 16 i + 4 g .. + 3 of query c
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (orow[r] < 0) continue;
    if (t.parts > 1) {
      const int mi = m0 + (wave * R + r) * 16 + c;
      float* rec = part_record(a, z, item, mi / G, kvh * G + mi % G);
#pragma unroll
      for (int i = 0; i < 8; ++i) *reinterpret_cast<f32x4*>(rec + 16 * i + 4 * g) = st.o[r][i];
      if (g == 0) *reinterpret_cast<f32x2*>(rec + kHeadDim) = f32x2{st.m[r], st.l[r][0]};
    } else {
      const float inv = inverse(st.l[r][0]);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        st8(a.out + orow[r] * kHeadDim + 16 * i + 4 * g,
            u32x2{pack2(st.o[r][i][0] * inv, st.o[r][i][1] * inv),
                  pack2(st.o[r][i][2] * inv, st.o[r][i][3] * inv)});
    }
  }
}

// Merges the parts of a row and head: kGroups groups of 32 lanes (4 channels each) take the parts in turn,
// then one another's results. Eight groups to a row for many parts (one row of 32 heads in 59 parts: 12
// us less than one group); for few parts a row per group (400 rows of 32 heads in 4 parts: 8 us less).
constexpr int kCombineThreads = 256;
template <int kGroups, bool kVerify>
__global__ __launch_bounds__(kCombineThreads) void kv4_combine_kernel(Kv4Args a) {
  constexpr int kRows = kCombineThreads / 32 / kGroups;
  __shared__ __align__(16) f32x4 os[kGroups][32];
  __shared__ f32x2 ml[kGroups];
  const int per_item = (a.tile_rows * a.heads + kRows - 1) / kRows;
  const int item = blockIdx.x / per_item;
  const Tile t = kVerify ? read_vblock(a, item) : read_tile(a, item);
  const int grp = kGroups == 1 ? 0 : threadIdx.x >> 5, ch = threadIdx.x & 31;
  const int i = blockIdx.x % per_item * kRows + (kGroups == 1 ? threadIdx.x >> 5 : 0);
  if (t.parts <= 1 || i >= t.rows * a.heads) return;  // (one part: written by the attention itself)
  const int64_t row = kVerify ? t.roff + i / a.heads : int64_t(a.row_idx[t.roff + i / a.heads]);
  if (row < 0 || row >= a.n_q_rows) return;
  const float* rec = part_record(a, 0, item, 0, i);
  const int64_t stride = int64_t(a.n_items) * a.tile_rows * a.heads * kPartFloats;
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = grp; p < t.parts; p += kGroups) {
    const f32x2 v = *reinterpret_cast<const f32x2*>(rec + p * stride + kHeadDim);
    const f32x4 x = *reinterpret_cast<const f32x4*>(rec + p * stride + 4 * ch);
    const float to = fmaxf(m, v[0]), base = to == -INFINITY ? 0.f : to;
    const float w0 = fast_exp2(m - base), w1 = fast_exp2(v[0] - base);
    l = w0 * l + w1 * v[1];
    o = w0 * o + w1 * x;
    m = to;
  }
  if constexpr (kGroups > 1) {
    os[grp][ch] = o;
    if (ch == 0) ml[grp] = f32x2{m, l};
    __syncthreads();
    if (grp != 0) return;
    m = -INFINITY;
#pragma unroll
    for (int x = 0; x < kGroups; ++x) m = fmaxf(m, ml[x][0]);
    const float base = m == -INFINITY ? 0.f : m;
    l = 0.f;
    o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < kGroups; ++x) {
      const float w = fast_exp2(ml[x][0] - base);
      l += w * ml[x][1];
      o += w * os[x][ch];
    }
  }
  const float inv = inverse(l);
  st8(a.out + (row * a.heads + i % a.heads) * kHeadDim + 4 * ch,
      u32x2{pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv)});
}

int check_common(const char* fn, const void* q, const void* cache, const void* out,
                 int64_t n_q_rows, int64_t n_slots, int64_t n_heads, int64_t n_kv_heads,
                 int64_t head_dim, float softmax_scale) {
  FDL_REQUIRE(head_dim == kHeadDim, FDL_ERR_UNSUPPORTED,
              "%s: head_dim = %lld (only 128 is implemented)", fn, (long long)head_dim);
  FDL_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024 && n_heads >= n_kv_heads && n_heads <= 4096 &&
                  n_heads % n_kv_heads == 0,
              FDL_ERR_SHAPE, "%s: n_heads = %lld is not a multiple of n_kv_heads = %lld", fn,
              (long long)n_heads, (long long)n_kv_heads);
  FDL_REQUIRE(n_slots >= kCellSlots && n_slots % kCellSlots == 0 && n_slots < (int64_t(1) << 31),
              FDL_ERR_SHAPE, "%s: n_slots = %lld is not a multiple of 16 from 16 below 2^31", fn,
              (long long)n_slots);
  FDL_REQUIRE(n_q_rows >= 1 && n_q_rows < (int64_t(1) << 31), FDL_ERR_SHAPE,
              "%s: n_q_rows = %lld out of range", fn, (long long)n_q_rows);
  FDL_REQUIRE(softmax_scale > 0.f && softmax_scale <= 2.3e38f, FDL_ERR_SHAPE,
              "%s: softmax_scale must be positive and at most 2.3e38 (log2(e) times it is finite)", fn);
  const void* const ptrs[] = {q, cache, out};
  const char* const names[] = {"q", "cache", "out"};
  for (int i = 0; i < 3; ++i) {
    FDL_REQUIRE(ptrs[i] != nullptr, FDL_ERR_NULL, "%s: %s is NULL", fn, names[i]);
    FDL_REQUIRE(reinterpret_cast<uintptr_t>(ptrs[i]) % 16 == 0, FDL_ERR_SHAPE,
                "%s: %s is not 16-byte aligned", fn, names[i]);
  }
  return FDL_OK;
}

template <int R>
hipError_t launch_wave(const Kv4Args& a, unsigned grid, bool imp, hipStream_t s) {
  constexpr int kMerge = kWaves * R * 64 * (8 * 16 + 8);
  if (imp)
    hipLaunchKernelGGL((kv4_wave_kernel<R, true>), dim3(grid), dim3(64 * kWaves),
                       kMerge + imp_frag_bytes(a.group), s, a);
  else
    hipLaunchKernelGGL((kv4_wave_kernel<R, false>), dim3(grid), dim3(64 * kWaves), kMerge, s, a);
  return hipGetLastError();
}

template <int R, int kAhead>
hipError_t launch_tile(const Kv4Args& a, unsigned grid, bool imp, hipStream_t s) {
  if (a.vblocks)
    hipLaunchKernelGGL((kv4_tile_kernel<R, kAhead, false, true>), dim3(grid), dim3(64 * kWaves),
                       kLdsFrags + 4 * kSlotKeys, s, a);
  else if (imp)
    hipLaunchKernelGGL((kv4_tile_kernel<R, kAhead, true, false>), dim3(grid), dim3(64 * kWaves),
                       kLdsFrags + imp_frag_bytes(a.group), s, a);
  else
    hipLaunchKernelGGL((kv4_tile_kernel<R, kAhead, false, false>), dim3(grid), dim3(64 * kWaves),
                       kLdsFrags, s, a);
  return hipGetLastError();
}

// Rows of a workgroup: the kernel that `m` rows x query heads to a K/V head get (verify: a tile kernel).
int workgroup_rows(int m, bool verify) {
  if (m <= 32 && !verify) return m <= 16 ? 16 : 32;
  return m <= 64 ? 64 : 128;
}

hipError_t launch_attention(const Kv4Args& a, bool imp, hipStream_t s) {
  const int rows = workgroup_rows(a.tile_rows * a.group, a.vblocks != nullptr);
  const unsigned grid = static_cast<unsigned>(int64_t(a.n_items) * a.kv_heads * a.n_parts * a.n_ranges);
  switch (rows) {
    case 16: return launch_wave<1>(a, grid, imp, s);
    case 32: return launch_wave<2>(a, grid, imp, s);
    case 64: return launch_tile<1, 4>(a, grid, imp, s);
    default: return launch_tile<2, 2>(a, grid, imp, s);
  }
}

template <bool kVerify>
hipError_t launch_combine(const Kv4Args& a, hipStream_t s) {
  const int64_t rows = int64_t(a.tile_rows) * a.heads;
  if (a.n_parts > 8)
    hipLaunchKernelGGL((kv4_combine_kernel<8, kVerify>), dim3(static_cast<unsigned>(a.n_items * rows)),
                       dim3(kCombineThreads), 0, s, a);
  else
    hipLaunchKernelGGL((kv4_combine_kernel<1, kVerify>),
                       dim3(static_cast<unsigned>(a.n_items * ((rows + 7) / 8))), dim3(kCombineThreads),
                       0, s, a);
  return hipGetLastError();
}

// Key split of a call: parts, their workspace, and the number of workgroups of both launches (a launch has
// fewer than 2^32 threads).
int check_parts(const char* fn, int64_t n_items, int64_t n_heads, int64_t n_kv_heads, int32_t tile_rows,
                int32_t n_parts, int32_t part_blocks, const float* workspace,
                int64_t workspace_floats, bool verify, int* n_ranges) {
  FDL_REQUIRE(n_parts >= 1 && n_parts <= FDL_KV4_MAX_PARTS && part_blocks >= 1, FDL_ERR_SHAPE,
              "%s: n_parts = %d outside [1, %d] or part_blocks = %d < 1", fn, n_parts,
              FDL_KV4_MAX_PARTS, part_blocks);
  if (n_parts > 1) {
    FDL_REQUIRE_PTR(workspace);
    FDL_REQUIRE_ALIGNED(workspace, 16);
    FDL_REQUIRE(workspace_floats / (n_items * tile_rows * n_heads * kPartFloats) >= n_parts,
                FDL_ERR_SHAPE, "%s: workspace of %lld floats for %d parts of %lld tiles of %d rows", fn,
                (long long)workspace_floats, n_parts, (long long)n_items, tile_rows);
  }
  const int m = tile_rows * static_cast<int>(n_heads / n_kv_heads), wg = workgroup_rows(m, verify);
  *n_ranges = (m + wg - 1) / wg;
  FDL_REQUIRE(n_items * n_kv_heads * n_parts * *n_ranges < (int64_t(1) << 24), FDL_ERR_UNSUPPORTED,
              "%s: %lld tiles of %d rows and %lld heads in %d parts are too many for one call", fn,
              (long long)n_items, tile_rows, (long long)n_heads, n_parts);
  FDL_REQUIRE(n_parts == 1 || n_items * tile_rows * n_heads < (int64_t(1) << 24),
              FDL_ERR_UNSUPPORTED, "%s: %lld tiles of %d rows and %lld heads are too many for parts",
              fn, (long long)n_items, tile_rows, (long long)n_heads);
  return FDL_OK;
}

}  // namespace
}  // namespace fdl

extern "C" int fdl_kv4_attention(const void* q, const void* cache, int64_t n_q_rows,
                                 int64_t n_slots, int64_t n_heads, int64_t n_kv_heads,
                                 int64_t head_dim, const int32_t* page_table, int64_t n_seq,
                                 int64_t max_pages, int32_t page_log2, const int32_t* work,
                                 int64_t n_work, const int32_t* row_idx, int64_t n_row_idx,
                                 int32_t tile_rows, float softmax_scale, void* out,
                                 int32_t imp_mode, float* imp_part, int32_t n_parts,
                                 int32_t part_blocks, float* workspace, int64_t workspace_floats,
                                 void* stream) {
  using namespace fdl;
  const char* fn = "fdl_kv4_attention";
  FDL_REQUIRE(n_work >= 0 && n_work < 65536, FDL_ERR_SHAPE, "%s: n_work = %lld out of range", fn,
              (long long)n_work);
  if (n_work == 0) return ok();
  int rc = check_common(fn, q, cache, out, n_q_rows, n_slots, n_heads, n_kv_heads, head_dim,
                        softmax_scale);
  if (rc != FDL_OK) return rc;
  FDL_REQUIRE(n_row_idx >= 0 && n_row_idx < (int64_t(1) << 31), FDL_ERR_SHAPE,
              "%s: n_row_idx out of range", fn);
  FDL_REQUIRE(page_log2 >= 4 && page_log2 <= 12 && n_seq >= 1 && n_seq < (int64_t(1) << 31) &&
                  max_pages >= 1 && max_pages < (int64_t(1) << 31),
              FDL_ERR_SHAPE, "%s: page table [%lld][%lld] of 2^%d-slot pages", fn,
              (long long)n_seq, (long long)max_pages, page_log2);
  FDL_REQUIRE(tile_rows >= 1 && tile_rows <= 256, FDL_ERR_UNSUPPORTED,
              "%s: tile_rows = %d outside [1, 256]", fn, tile_rows);
  FDL_REQUIRE(imp_mode == FDL_IMP_NONE || imp_mode == FDL_IMP_RAW_LOGIT, FDL_ERR_UNSUPPORTED,
              "%s: imp_mode = %d (none or raw logits)", fn, imp_mode);
  FDL_REQUIRE(imp_mode == FDL_IMP_NONE || n_heads / n_kv_heads <= kImpMaxGroup,
              FDL_ERR_UNSUPPORTED, "%s: importance with %lld query heads to a K/V head (at most %d)",
              fn, (long long)(n_heads / n_kv_heads), kImpMaxGroup);
  FDL_REQUIRE_PTR(page_table);
  FDL_REQUIRE_PTR(work);
  FDL_REQUIRE_PTR(row_idx);
  FDL_REQUIRE(imp_mode == FDL_IMP_NONE || imp_part != nullptr, FDL_ERR_NULL, "%s: imp_part is NULL",
              fn);
  FDL_REQUIRE_ALIGNED(imp_part, 16);
  Kv4Args a = {};
  rc = check_parts(fn, n_work, n_heads, n_kv_heads, tile_rows, n_parts, part_blocks, workspace,
                   workspace_floats, false, &a.n_ranges);
  if (rc != FDL_OK) return rc;
  a.q = static_cast<const uint16_t*>(q);
  a.cache = static_cast<const uint8_t*>(cache);
  a.out = static_cast<uint16_t*>(out);
  a.page_table = page_table;
  a.work = work;
  a.row_idx = row_idx;
  a.imp_part = imp_mode == FDL_IMP_NONE ? nullptr : imp_part;
  a.part = n_parts > 1 ? workspace : nullptr;
  a.n_q_rows = n_q_rows;
  a.n_slots = n_slots;
  a.n_row_idx = n_row_idx;
  a.max_pages = max_pages;
  a.n_seq = static_cast<int>(n_seq);
  a.page_log2 = page_log2;
  a.heads = static_cast<int>(n_heads);
  a.kv_heads = static_cast<int>(n_kv_heads);
  a.group = static_cast<int>(n_heads / n_kv_heads);
  a.tile_rows = tile_rows;
  a.n_items = static_cast<int>(n_work);
  a.n_parts = n_parts;
  a.part_blocks = part_blocks;
  a.scale_log2 = softmax_scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  FDL_HIP_CHECK(launch_attention(a, imp_mode != FDL_IMP_NONE, s));
  if (n_parts > 1) FDL_HIP_CHECK(launch_combine<false>(a, s));
  return ok();
}

extern "C" int fdl_kv4_verify_attention(const void* q, const void* k_blk, const void* v_blk,
                                        const void* cache, int64_t n_q_rows, int64_t n_slots,
                                        int64_t n_heads, int64_t n_kv_heads, int64_t head_dim,
                                        const int64_t* key_slots, int64_t n_keys,
                                        const int32_t* vblocks, int64_t n_vblocks,
                                        const uint8_t* mask, const int32_t* vmeta,
                                        int32_t block_rows, float softmax_scale, void* out,
                                        int32_t n_parts, int32_t part_blocks, float* workspace,
                                        int64_t workspace_floats, void* stream) {
  using namespace fdl;
  const char* fn = "fdl_kv4_verify_attention";
  FDL_REQUIRE(n_vblocks >= 0 && n_vblocks < 65536, FDL_ERR_SHAPE,
              "%s: n_vblocks = %lld out of range", fn, (long long)n_vblocks);
  if (n_vblocks == 0) return ok();
  int rc = check_common(fn, q, cache, out, n_q_rows, n_slots, n_heads, n_kv_heads, head_dim,
                        softmax_scale);
  if (rc != FDL_OK) return rc;
  FDL_REQUIRE_PTR(k_blk);
  FDL_REQUIRE_PTR(v_blk);
  FDL_REQUIRE_PTR(vblocks);
  FDL_REQUIRE_ALIGNED(k_blk, 16);
  FDL_REQUIRE_ALIGNED(v_blk, 16);
  FDL_REQUIRE((mask != nullptr) != (vmeta != nullptr), FDL_ERR_NULL,
              "%s: exactly one of mask and vmeta must be given", fn);
  FDL_REQUIRE(block_rows >= 1 && block_rows <= 256, FDL_ERR_UNSUPPORTED,
              "%s: block_rows = %d outside [1, 256]", fn, block_rows);
  FDL_REQUIRE(n_keys >= 0 && n_keys < (int64_t(1) << 31), FDL_ERR_SHAPE, "%s: n_keys out of range",
              fn);
  FDL_REQUIRE(n_keys == 0 || key_slots != nullptr, FDL_ERR_NULL, "%s: key_slots is NULL", fn);
  Kv4Args a = {};
  rc = check_parts(fn, n_vblocks, n_heads, n_kv_heads, block_rows, n_parts, part_blocks,
                   workspace, workspace_floats, true, &a.n_ranges);
  if (rc != FDL_OK) return rc;
  a.q = static_cast<const uint16_t*>(q);
  a.kblk = static_cast<const uint16_t*>(k_blk);
  a.vblk = static_cast<const uint16_t*>(v_blk);
  a.cache = static_cast<const uint8_t*>(cache);
  a.out = static_cast<uint16_t*>(out);
  a.key_slots = key_slots;
  a.vblocks = vblocks;
  a.mask = mask;
  a.vmeta = vmeta;
  a.n_q_rows = n_q_rows;
  a.n_slots = n_slots;
  a.n_keys = n_keys;
  a.heads = static_cast<int>(n_heads);
  a.kv_heads = static_cast<int>(n_kv_heads);
  a.group = static_cast<int>(n_heads / n_kv_heads);
  a.tile_rows = block_rows;
  a.n_items = static_cast<int>(n_vblocks);
  a.n_parts = n_parts;
  a.part_blocks = part_blocks;
  a.part = n_parts > 1 ? workspace : nullptr;
  a.page_log2 = 4;
  a.scale_log2 = softmax_scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  FDL_HIP_CHECK(launch_attention(a, false, s));
  if (n_parts > 1) FDL_HIP_CHECK(launch_combine<true>(a, s));
  return ok();
}
