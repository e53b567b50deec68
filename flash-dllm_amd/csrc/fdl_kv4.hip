// Rows into and out of the 4-bit K/V cache (gfx950); its layout is in fdl_kv4.h.
//
//  * fdl_kv4_append: for each row with a slot, K rotated by the row's position (when sin/cos tables are
//    given), K and V quantised and written to the slot; Q rotated alike in the same launch.
//        k'[c]      = k[c] cos[c] - k[c + 64] sin[c]
//        k'[c + 64] = k[c + 64] cos[c + 64] + k[c] sin[c + 64]
//  * fdl_kv4_read: the rows of slots as bf16, exactly what the codes stand for.
//
// The rotation runs in 64 bits and is rounded once, K to 32 bits, Q to bf16: a bf16 times a float is exact in
// 64 bits, so the rotated value is correctly rounded and the codes do not depend on how a compiler orders
// or fuses the arithmetic (a value next to the border of two codes would otherwise flip a whole step).
#include "fdl_host.h"
#include "fdl_kv4.h"

namespace fdl {
namespace {

constexpr int kThreads = 256;
constexpr int kUnitLanes = 8;  // lanes of one head's row: lane i has channels 8 i .. + 7 and 64 + 8 i ..

struct AppendArgs {
  const uint16_t* k;
  const uint16_t* v;
  const uint16_t* q;
  int64_t ld_k, ld_v, ld_q;  // elements between rows
  const float* sin;
  const float* cos;
  int64_t n_rope_rows;
  const int64_t* slot;
  const int64_t* rope_row;  // NULL: the slot
  int64_t n_rows, n_slots;
  int kv_heads, heads;  // heads: 0 without Q
  uint8_t* cache;
  uint16_t* q_out;  // [n_rows][heads * 128]
};

__device__ __forceinline__ void unpack8(const uint16_t* p, float (&x)[8]) {
  const u32x4 v = ld16(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float(v[j] << 16);
    x[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
  }
}

__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[j] = a[j];
    x[4 + j] = b[j];
  }
}

// Largest magnitude over the four lanes of a group of 32 channels (a DPP quad); a NaN counts as
// infinite, so that either marks the group.
__device__ __forceinline__ float group_top(const float (&x)[8]) {
  float top = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j] != x[j] ? INFINITY : fabsf(x[j]));
  top = fmaxf(top, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(top), 0xB1, 0xF, 0xF, false)));
  return fmaxf(top, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(top), 0x4E, 0xF, 0xF, false)));
}

// A float half way between two bf16 values: rounded from a double it says no more on which side the double was.
__device__ __forceinline__ bool half_way(float f) { return __float_as_uint(f) << 16 == 0x80000000u; }

// Such a float, moved by a bit to the double's side, so that its rounding to bf16 is the double's.
__device__ __forceinline__ float to_side(float f, double d) {
  const double to = fabs(d), at = fabs(static_cast<double>(f));
  const uint32_t b = __float_as_uint(f);
  return !half_way(f) || to == at ? f : __uint_as_float(to > at ? b + 1 : b - 1);
}

// One unit of 8 lanes per (row, head of K, V or Q), the heads of a row side by side: whole 64-byte runs of
// every input row, and a lane's two words of codes need no other lane. Bound by memory: 7919 rows with Q of
// 32 heads and K and V of 8, rotated, in 35.5 us (179 MB, 5.0 TB/s); by
// the launch for few rows (8: 3.4 us).
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(AppendArgs a) {
  const int64_t unit = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / kUnitLanes;
  const int lane = threadIdx.x % kUnitLanes;
  const int per_row = 2 * a.kv_heads + a.heads;
  const int64_t row = unit / per_row;
  if (row >= a.n_rows) return;  // whole units: the quads below stay together
  int head = static_cast<int>(unit - row * per_row);
  const int64_t slot = a.slot[row];
  if (slot < 0 || slot >= a.n_slots) return;
  int64_t rr = 0;
  if (a.sin) {
    rr = a.rope_row ? a.rope_row[row] : slot;
    if (rr < 0 || rr >= a.n_rope_rows) return;
  }
  enum { kK, kV, kQ } what = kK;
  const uint16_t* src = a.k + row * a.ld_k;
  if (head >= 2 * a.kv_heads) {
    what = kQ;
    head -= 2 * a.kv_heads;
    src = a.q + row * a.ld_q;
  } else if (head >= a.kv_heads) {
    what = kV;
    head -= a.kv_heads;
    src = a.v + row * a.ld_v;
  }
  src += head * kKv4HeadDim + 8 * lane;
  float lo[8], hi[8];
  unpack8(src, lo);
  unpack8(src + 64, hi);
  if (a.sin && what != kV) {
    float s0[8], s1[8], c0[8], c1[8];
    const float* sp = a.sin + rr * kKv4HeadDim + 8 * lane;
    const float* cp = a.cos + rr * kKv4HeadDim + 8 * lane;
    load8(sp, s0);
    load8(sp + 64, s1);
    load8(cp, c0);
    load8(cp + 64, c1);
    bool again = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const double x = lo[j], y = hi[j];
      lo[j] = static_cast<float>(x * c0[j] - y * s0[j]);
      hi[j] = static_cast<float>(y * c1[j] + x * s1[j]);
      again = again || half_way(lo[j]) || half_way(hi[j]);
    }
    if (what == kQ && again) {  // one lane in 4000: a second look (for every value: 2 of 48 us of 7919 rows)
      float x[8], y[8];
      unpack8(src, x);
      unpack8(src + 64, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        lo[j] = to_side(lo[j], double(x[j]) * c0[j] - double(y[j]) * s0[j]);
        hi[j] = to_side(hi[j], double(y[j]) * c1[j] + double(x[j]) * s1[j]);
      }
    }
  }
  if (what == kQ) {
    uint16_t* dst = a.q_out + row * a.heads * kKv4HeadDim + head * kKv4HeadDim + 8 * lane;
    u32x4 w0, w1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w0[j] = pack_bf16x2(lo[2 * j], lo[2 * j + 1]);
      w1[j] = pack_bf16x2(hi[2 * j], hi[2 * j + 1]);
    }
    st16(dst, w0);
    st16(dst + 64, w1);
    return;
  }
  const uint32_t b0 = kv4_scale_byte(group_top(lo)), b1 = kv4_scale_byte(group_top(hi));
  const uint32_t w0 = kv4_codes(lo, b0), w1 = kv4_codes(hi, b1);
  const int s = static_cast<int>(slot % kCellSlots);
  uint8_t* cell = a.cache + (slot / kCellSlots * a.kv_heads + head) * kCellBytes;
  const int at = what == kK ? 64 * s + 4 * lane : kCellV + 256 * (s / 4) + 4 * (s % 4) + 16 * lane;
  *reinterpret_cast<uint32_t*>(cell + at) = w0;
  *reinterpret_cast<uint32_t*>(cell + at + (what == kK ? 32 : 128)) = w1;
  if (lane % 4 == 0) {
    uint8_t* sc = cell + (what == kK ? kCellKs : kCellVs) + 16 * (lane / 4) + s;
    sc[0] = static_cast<uint8_t>(b0);
    sc[32] = static_cast<uint8_t>(b1);
  }
}

// As above: 8 lanes per (row, head of K or V). A row without a slot in the cache reads as zeros. 8192 rows
// of 8 heads: 9 us.
__global__ __launch_bounds__(kThreads) void kv4_read_kernel(
    const uint8_t* __restrict__ cache, int64_t n_slots, int kv_heads,
    const int64_t* __restrict__ slot_of, int64_t n_rows, uint16_t* __restrict__ k_out,
    uint16_t* __restrict__ v_out) {
  const int64_t unit = (int64_t(blockIdx.x) * kThreads + threadIdx.x) / kUnitLanes;
  const int lane = threadIdx.x % kUnitLanes;
  const int64_t row = unit / (2 * kv_heads);
  if (row >= n_rows) return;
  int head = static_cast<int>(unit - row * 2 * kv_heads);
  const bool is_v = head >= kv_heads;
  if (is_v) head -= kv_heads;
  uint16_t* dst = (is_v ? v_out : k_out) + (row * kv_heads + head) * kKv4HeadDim + 8 * lane;
  const int64_t slot = slot_of[row];
  if (slot < 0 || slot >= n_slots) {
    st16(dst, u32x4{0, 0, 0, 0});
    st16(dst + 64, u32x4{0, 0, 0, 0});
    return;
  }
  const int s = static_cast<int>(slot % kCellSlots);
  const uint8_t* cell = cache + (slot / kCellSlots * kv_heads + head) * kCellBytes;
  const int at = is_v ? kCellV + 256 * (s / 4) + 4 * (s % 4) + 16 * lane : 64 * s + 4 * lane;
  const uint8_t* sc = cell + (is_v ? kCellVs : kCellKs) + 16 * (lane / 4) + s;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(cell + at + half * (is_v ? 128 : 32));
    const float scale = __uint_as_float(uint32_t(sc[32 * half]) << 23);
    st16(dst + 64 * half, u32x4{kv4_bf16x2<0>(w, scale), kv4_bf16x2<1>(w, scale),
                                kv4_bf16x2<2>(w, scale), kv4_bf16x2<3>(w, scale)});
  }
}

int check_cache(const char* fn, const void* cache, int64_t n_slots, int64_t n_kv_heads,
                int64_t head_dim) {
  FDL_REQUIRE(head_dim == kKv4HeadDim, FDL_ERR_UNSUPPORTED,
              "%s: head_dim = %lld (only 128 is implemented)", fn, (long long)head_dim);
  FDL_REQUIRE(n_kv_heads >= 1 && n_kv_heads <= 1024, FDL_ERR_SHAPE,
              "%s: n_kv_heads = %lld outside [1, 1024]", fn, (long long)n_kv_heads);
  FDL_REQUIRE(n_slots >= kCellSlots && n_slots % kCellSlots == 0 && n_slots < (int64_t(1) << 31),
              FDL_ERR_SHAPE, "%s: n_slots = %lld is not a multiple of 16 from 16 below 2^31", fn,
              (long long)n_slots);
  FDL_REQUIRE(cache != nullptr, FDL_ERR_NULL, "%s: cache is NULL", fn);
  FDL_REQUIRE(reinterpret_cast<uintptr_t>(cache) % 16 == 0, FDL_ERR_SHAPE,
              "%s: cache is not 16-byte aligned", fn);
  return FDL_OK;
}

}  // namespace
}  // namespace fdl

extern "C" int fdl_kv4_append(const void* k, int64_t ld_k, const void* v, int64_t ld_v,
                              const void* q, int64_t ld_q, const float* rope_sin,
                              const float* rope_cos, int64_t n_rope_rows, const int64_t* slot,
                              const int64_t* rope_row, int64_t n_rows, int64_t n_heads,
                              int64_t n_kv_heads, int64_t head_dim, void* cache, int64_t n_slots,
                              void* q_out, void* stream) {
  using namespace fdl;
  FDL_REQUIRE(n_rows >= 0 && n_rows < (int64_t(1) << 31), FDL_ERR_SHAPE,
              "fdl_kv4_append: n_rows = %lld out of range", (long long)n_rows);
  if (n_rows == 0) return ok();
  int rc = check_cache("fdl_kv4_append", cache, n_slots, n_kv_heads, head_dim);
  if (rc != FDL_OK) return rc;
  FDL_REQUIRE_PTR(k);
  FDL_REQUIRE_PTR(v);
  FDL_REQUIRE_PTR(slot);
  FDL_REQUIRE((q == nullptr) == (q_out == nullptr), FDL_ERR_NULL,
              "fdl_kv4_append: q and q_out go together");
  FDL_REQUIRE(q == nullptr || (n_heads >= 1 && n_heads <= 4096), FDL_ERR_SHAPE,
              "fdl_kv4_append: n_heads = %lld outside [1, 4096]", (long long)n_heads);
  FDL_REQUIRE((rope_sin == nullptr) == (rope_cos == nullptr), FDL_ERR_NULL,
              "fdl_kv4_append: rope_sin and rope_cos go together");
  FDL_REQUIRE(rope_sin == nullptr || n_rope_rows >= 1, FDL_ERR_SHAPE,
              "fdl_kv4_append: empty rope tables");
  FDL_REQUIRE(ld_k >= n_kv_heads * head_dim && ld_v >= n_kv_heads * head_dim && ld_k % 8 == 0 &&
                  ld_v % 8 == 0 && (q == nullptr || (ld_q >= n_heads * head_dim && ld_q % 8 == 0)),
              FDL_ERR_SHAPE,
              "fdl_kv4_append: row strides must be multiples of 8 and hold a row's heads");
  FDL_REQUIRE_ALIGNED(k, 16);
  FDL_REQUIRE_ALIGNED(v, 16);
  FDL_REQUIRE_ALIGNED(q, 16);
  FDL_REQUIRE_ALIGNED(q_out, 16);
  FDL_REQUIRE_ALIGNED(rope_sin, 16);
  FDL_REQUIRE_ALIGNED(rope_cos, 16);
  AppendArgs a;
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q = static_cast<const uint16_t*>(q);
  a.ld_k = ld_k;
  a.ld_v = ld_v;
  a.ld_q = ld_q;
  a.sin = rope_sin;
  a.cos = rope_cos;
  a.n_rope_rows = n_rope_rows;
  a.slot = slot;
  a.rope_row = rope_row;
  a.n_rows = n_rows;
  a.n_slots = n_slots;
  a.kv_heads = static_cast<int>(n_kv_heads);
  a.heads = q ? static_cast<int>(n_heads) : 0;
  a.cache = static_cast<uint8_t*>(cache);
  a.q_out = static_cast<uint16_t*>(q_out);
  const int64_t units = n_rows * (2 * a.kv_heads + a.heads);
  const int64_t blocks = (units * kUnitLanes + kThreads - 1) / kThreads;
  FDL_REQUIRE(blocks < (int64_t(1) << 24), FDL_ERR_UNSUPPORTED,
              "fdl_kv4_append: %lld rows of %d heads are too many for one call", (long long)n_rows,
              2 * a.kv_heads + a.heads);
  hipLaunchKernelGGL(kv4_append_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), a);
  FDL_HIP_CHECK(hipGetLastError());
  return ok();
}

extern "C" int fdl_kv4_read(const void* cache, int64_t n_slots, int64_t n_kv_heads,
                            int64_t head_dim, const int64_t* slot, int64_t n_rows, void* k_out,
                            void* v_out, void* stream) {
  using namespace fdl;
  FDL_REQUIRE(n_rows >= 0 && n_rows < (int64_t(1) << 31), FDL_ERR_SHAPE,
              "fdl_kv4_read: n_rows = %lld out of range", (long long)n_rows);
  if (n_rows == 0) return ok();
  int rc = check_cache("fdl_kv4_read", cache, n_slots, n_kv_heads, head_dim);
  if (rc != FDL_OK) return rc;
  FDL_REQUIRE_PTR(slot);
  FDL_REQUIRE_PTR(k_out);
  FDL_REQUIRE_PTR(v_out);
  FDL_REQUIRE_ALIGNED(k_out, 16);
  FDL_REQUIRE_ALIGNED(v_out, 16);
  const int64_t blocks = (n_rows * 2 * n_kv_heads * kUnitLanes + kThreads - 1) / kThreads;
  FDL_REQUIRE(blocks < (int64_t(1) << 24), FDL_ERR_UNSUPPORTED,
              "fdl_kv4_read: %lld rows of %lld heads are too many for one call", (long long)n_rows,
              (long long)n_kv_heads);
  hipLaunchKernelGGL(kv4_read_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0,
                     static_cast<hipStream_t>(stream), static_cast<const uint8_t*>(cache), n_slots,
                     static_cast<int>(n_kv_heads), slot, n_rows, static_cast<uint16_t*>(k_out),
                     static_cast<uint16_t*>(v_out));
  FDL_HIP_CHECK(hipGetLastError());
  return ok();
}
