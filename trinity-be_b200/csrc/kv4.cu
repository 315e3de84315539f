// A paged key/value cache held in 4 bits: writing it, reading it back, and the attention of one new
// token per sequence over it.
//
// Cache format.  A key or value row (one position, one cached head) of D channels is cut into
// groups of 32, 64 or 128 channels.  A group keeps zero = min (exact in BF16), scale =
// bf16((max - min) / 15) and for each channel code = rint((x - zero) / scale) in 0..15; a code
// stands for zero + scale * code.  A group whose values are all equal has scale 0 and codes 0; one
// that holds an infinity or a NaN has scale NaN and reads back as NaN.
//   codes  [pages, kv_heads, page, D / 2]         two channels a byte, the even one in the low bits
//   scales [pages, kv_heads, page, D / group, 2]  BF16 (scale, zero)
#include <cuda_fp16.h>

#include "host_common.h"
#include "sm100_ptx.cuh"

namespace trinity_sm100 {
namespace {

// Device status sites of invalid device-side data (no access is made with it).
constexpr uint32_t kSiteKv4AppendSlot = 0x901;
constexpr uint32_t kSiteKv4ReadSlot = 0x902;
constexpr uint32_t kSiteKv4Page = 0x903;

// ---------------------------------------------------------------- append and read
//
// Bound by memory: 2 D bytes read and D / 2 + 4 D / group written per row (append).  A lane owns
// sixteen channels (one 32-byte access, two 32-bit words of codes) or eight, with keys and values in
// one launch; a group's extrema meet by shuffles within its 2 to 16 lanes.  32771 tokens x 8 heads x
// 128 channels in groups of 32, written and read back: 63 us for 352.6 MB (append 32.7, read 29.0: 0.82 and
// 0.93 of the measured copy rate; read in FP32 48.7 us for 311 MB; with eight channels a lane and single
// FP32 arithmetic instruction issue took 84).  One token of 64 sequences: 3.1 us for both.
struct Kv4Rows {
  const __nv_bfloat16* in[2];      // append: keys, values
  void* out[2];                    // read: keys, values
  uint8_t* codes[2];
  __nv_bfloat162* scales[2];
  const long long* slots;
  long long tokens, positions;     // positions = pages * page
  long long token_stride[2], head_stride[2];
  int kv_heads, page, out_f32;
  int group_shift;                 // logarithm of the group
  int heads_shift, page_shift;     // logarithms of kv_heads and page, -1 where they are no powers of two
};

// Row of the cache that holds head `head` of position `slot` (the cache has fewer than 2^31 rows).
__device__ __forceinline__ uint32_t kv4_row(const Kv4Rows& p, uint32_t slot, uint32_t head) {
  const uint32_t page = p.page_shift >= 0 ? slot >> p.page_shift : slot / uint32_t(p.page);
  return (page * p.kv_heads + head) * p.page + (slot - page * p.page);
}
// Index of the (scale, zero) of a row's channel.
template <int kD>
__device__ __forceinline__ uint64_t kv4_pair(const Kv4Rows& p, uint32_t row, int channel) {
  return static_cast<uint64_t>(row) * uint32_t(kD >> p.group_shift) + (channel >> p.group_shift);
}
// The kBatch rows (token, head) of a group of kLanes lanes, a block's rows apart; the launcher keeps
// all lanes of a launch below 2^31.  All loads of a step are issued before the first use.
template <int kLanes, int kBatch>
struct Kv4Batch {
  uint32_t token[kBatch], head[kBatch];
  long long slot[kBatch];     // -1: nothing to do
  bool live[kBatch];
  __device__ __forceinline__ Kv4Batch(const Kv4Rows& p) {
    constexpr uint32_t kRows = 256 / kLanes;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const uint32_t index = (blockIdx.x * kBatch + i) * kRows + threadIdx.x / kLanes;
      token[i] = p.heads_shift >= 0 ? index >> p.heads_shift : index / uint32_t(p.kv_heads);
      head[i] = index - token[i] * p.kv_heads;
      live[i] = token[i] < uint32_t(p.tokens);
      slot[i] = live[i] ? p.slots[token[i]] : -1;
    }
  }
  __device__ __forceinline__ long long offset(const Kv4Rows& p, int which, int i) const {
    return static_cast<long long>(token[i]) * p.token_stride[which] + static_cast<long long>(head[i]) * p.head_stride[which];
  }
};

// Larger, or smaller, of each pair of BF16 values; NaN if either is.
__device__ __forceinline__ uint32_t nan_max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t nan_min2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float reciprocal_approx(float x) {   // 2^-23 relative
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The divisions that hardly any group needs, out of line.
__device__ __noinline__ uint32_t divided_code(float x, float scale) {
  return static_cast<uint32_t>(fminf(rintf(x / scale), 15.0f));
}
__device__ __noinline__ float divided_spread(float spread) { return spread / 15.0f; }

// Two FP32 numbers an instruction (each rounded as the single ones are).
__device__ __forceinline__ uint64_t pair_f32(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves_f32(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// 16 or 32 bytes that are not read or written again soon.
template <int kCount>
__device__ __forceinline__ void load_once(const void* p, uint32_t (&w)[kCount]) {
  static_assert(kCount == 4 || kCount == 8, "");
  if constexpr (kCount == 4)
    asm volatile("ld.global.cs.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
  else
    asm volatile("ld.global.cs.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}
template <int kCount>
__device__ __forceinline__ void store_once(void* p, const uint32_t (&w)[kCount]) {
  static_assert(kCount == 4 || kCount == 8, "");
  if constexpr (kCount == 4)
    asm volatile("st.global.cs.v4.b32 [%4], {%0, %1, %2, %3};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "l"(p) : "memory");
  else
    asm volatile("st.global.cs.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(p)
                 : "memory");
}

// Five blocks of sixteen channels a lane an SM: 32.1 to 32.7 us at the size above; four 35.4, six (spilling) 32.4.
template <int kD, int kWords, bool kVector, int kBatch>
__global__ void __launch_bounds__(256, kWords == 2 ? 5 : 1) kv4_append_kernel(const Kv4Rows p) {
  constexpr int kChannels = 8 * kWords, kLanes = kD / kChannels;
  grid_dependents_may_launch();
  grid_dependency_wait();
  const int which = blockIdx.y, lane = threadIdx.x % kLanes;
  const Kv4Batch<kLanes, kBatch> rows(p);
  uint32_t raw[kBatch][4 * kWords];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const __nv_bfloat16* src = p.in[which] + rows.offset(p, which, i) + lane * kChannels;
#pragma unroll
    for (int e = 0; e < 4 * kWords; ++e) raw[i][e] = 0;
    if (!rows.live[i]) continue;
    if constexpr (kVector) {
      load_once(src, raw[i]);
    } else {
      const uint16_t* one = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
      for (int e = 0; e < 4 * kWords; ++e) raw[i][e] = one[2 * e] | uint32_t(one[2 * e + 1]) << 16;
    }
  }
  const int group_lanes = 1 << p.group_shift >> (kWords == 2 ? 4 : 3);
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {      // (the shuffles need every lane of the warp, rows or not)
    const uint32_t(&w)[4 * kWords] = raw[i];
    // (max, -min) of the group as a BF16 pair; a NaN goes through, an infinity stays one
    uint32_t extrema = w[0], smallest = w[0];
#pragma unroll
    for (int e = 1; e < 4 * kWords; ++e) {
      extrema = nan_max2(extrema, w[e]);
      smallest = nan_min2(smallest, w[e]);
    }
    const uint32_t negated = smallest ^ 0x80008000u;
    extrema = nan_max2(__byte_perm(extrema, negated, 0x5410), __byte_perm(extrema, negated, 0x7632));
    for (int step = 1; step < group_lanes; step *= 2)     // the lanes of a group are neighbours
      extrema = nan_max2(extrema, __shfl_xor_sync(0xffffffffu, extrema, step));
    const float high = bf16_lo(extrema), low = -bf16_hi(extrema), spread = high - low;
    // spread / 15, correctly rounded: a product with 1 / 15 and one Newton step (the remainder is exact
    // unless it is subnormal)
    float fifteenth = spread * (1.0f / 15.0f);
    fifteenth = fmaf(fmaf(-15.0f, fifteenth, spread), 1.0f / 15.0f, fifteenth);
    if (!(spread > 0x1p-90f)) fifteenth = divided_spread(spread);
    const __nv_bfloat16 scale16 = __float2bfloat16(spread < INFINITY ? fifteenth : NAN);
    const float scale = __bfloat162float(scale16);
    uint64_t v[4 * kWords];                        // pairs of x - zero
    const uint64_t minus_low = pair_f32(-low, -low);
#pragma unroll
    for (int e = 0; e < 4 * kWords; ++e) v[e] = add_f32x2(pair_f32(bf16_lo(w[e]), bf16_hi(w[e])), minus_low);
    // code = rint((x - zero) / scale), at most 15.06 before rounding as the scale is rounded by 2^-8 at
    // most.  BF16 values and scales are so coarse that half of all warps meet a quotient of exactly k + 1/2,
    // so the quotient must be the correctly rounded one: the product with the correctly rounded
    // reciprocal, corrected once by its exact remainder (Markstein's division; an 8-bit divisor is
    // none of its exceptions).
    uint32_t codes[kWords];
#pragma unroll
    for (int c = 0; c < kWords; ++c) codes[c] = 0;
    if (scale > 0x1p-100f) {
      constexpr float kInteger = 12582912.0f;      // 1.5 * 2^23: adding it rounds to an integer, half to even
      float inverse = reciprocal_approx(scale);
      inverse = fmaf(inverse, fmaf(-scale, inverse, 1.0f), inverse);
      const uint64_t inverses = pair_f32(inverse, inverse), minus_scale = pair_f32(-scale, -scale);
      const uint64_t integers = pair_f32(kInteger, kInteger);
#pragma unroll
      for (int e = 4 * kWords - 1; e >= 0; --e) {
        uint64_t quotient = mul_f32x2(v[e], inverses);
        quotient = fma_f32x2(fma_f32x2(quotient, minus_scale, v[e]), inverses, quotient);
        const float2 sums = halves_f32(add_f32x2(quotient, integers));   // the codes in the last four bits
        codes[e / 4] = codes[e / 4] * 16u + __float_as_uint(sums.y);
        codes[e / 4] = codes[e / 4] * 16u + __float_as_uint(sums.x);
      }
#pragma unroll
      for (int c = 0; c < kWords; ++c) codes[c] -= 0x3f400000u;   // what the exponents of the eight sums have added up to
    } else if (scale > 0.0f) {
#pragma unroll
      for (int e = 0; e < 4 * kWords; ++e) {
        const float2 x = halves_f32(v[e]);
        codes[e / 4] |= (divided_code(x.x, scale) | divided_code(x.y, scale) << 4) << (8 * (e % 4));
      }
    }
    if (rows.slot[i] < 0) continue;
    if (rows.slot[i] >= p.positions) {
      report_timeout(kSiteKv4AppendSlot);
      continue;
    }
    const uint32_t row = kv4_row(p, uint32_t(rows.slot[i]), rows.head[i]);
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.codes[which]) + static_cast<uint64_t>(row) * (kD / 8) + lane * kWords;
    if constexpr (kWords == 2)
      *reinterpret_cast<uint2*>(dst) = make_uint2(codes[0], codes[1]);
    else
      *dst = codes[0];
    if ((lane & (group_lanes - 1)) == 0) {
      __nv_bfloat162 pair;
      pair.x = scale16;
      pair.y = __float2bfloat16(low);
      p.scales[which][kv4_pair<kD>(p, row, lane * kChannels)] = pair;
    }
  }
}

// The values that the codes at `slots` stand for, rounded to the output type: BF16 in one fused
// multiplication and addition, FP32 likewise (there the product is exact too).  A negative slot reads
// as zeros.
template <int kD, int kWords, int kBatch>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4Rows p) {
  constexpr int kChannels = 8 * kWords, kLanes = kD / kChannels;
  grid_dependents_may_launch();
  grid_dependency_wait();
  const int which = blockIdx.y, lane = threadIdx.x % kLanes;
  const Kv4Batch<kLanes, kBatch> rows(p);
  uint32_t codes[kBatch][kWords];
  uint32_t pair[kBatch];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
#pragma unroll
    for (int c = 0; c < kWords; ++c) codes[i][c] = 0;
    pair[i] = 0;
    if (rows.slot[i] >= 0 && rows.slot[i] < p.positions) {
      const uint32_t row = kv4_row(p, uint32_t(rows.slot[i]), rows.head[i]);
      const uint32_t* src = reinterpret_cast<const uint32_t*>(p.codes[which]) + static_cast<uint64_t>(row) * (kD / 8) + lane * kWords;
      if constexpr (kWords == 2) {
        const uint2 both = *reinterpret_cast<const uint2*>(src);
        codes[i][0] = both.x;
        codes[i][1] = both.y;
      } else {
        codes[i][0] = *src;
      }
      pair[i] = reinterpret_cast<const uint32_t*>(p.scales[which])[kv4_pair<kD>(p, row, lane * kChannels)];
    } else if (rows.slot[i] >= 0) {
      report_timeout(kSiteKv4ReadSlot);
    }
  }
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    if (!rows.live[i]) continue;
    const long long at = rows.offset(p, which, i) + lane * kChannels;
    if (p.out_f32) {
      const float scale = bf16_lo(pair[i]), zero = bf16_hi(pair[i]);
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // the code in the last mantissa bits of 2^23 (five of them reach without a shift); the scale
          // times a power of two is exact, even at its smallest
          constexpr float kInteger = 8388608.0f;
          const int shift = 4 * (e < 4 ? e : e - 4);
          const uint32_t bits = ((e < 4 ? codes[i][c] : codes[i][c] >> 16) & (15u << shift)) | __float_as_uint(kInteger);
          v[e] = __float_as_uint(fmaf(__uint_as_float(bits) - kInteger, scale * (1.0f / (1 << shift)), zero));
        }
        float* dst = static_cast<float*>(p.out[which]) + at + 8 * c;
        if constexpr (kWords == 2) {
          store_once(dst, v);
        } else {
          store_once(dst, {v[0], v[1], v[2], v[3]});
          store_once(dst + 4, {v[4], v[5], v[6], v[7]});
        }
      }
    } else {
      const uint32_t scales = __byte_perm(pair[i], 0, 0x1010), zeros = __byte_perm(pair[i], 0, 0x3232);
      uint32_t out[4 * kWords];
#pragma unroll
      for (int c = 0; c < kWords; ++c) {
        uint32_t v[4];                             // channels (j, j + 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t large = ((codes[i][c] >> (4 * j)) & 0x000f000fu) | 0x43004300u;   // 128 + code
          v[j] = fma_bf16x2(add_bf16x2(large, 0xc300c300u), scales, zeros);
        }
        out[4 * c] = __byte_perm(v[0], v[1], 0x5410);
        out[4 * c + 1] = __byte_perm(v[2], v[3], 0x5410);
        out[4 * c + 2] = __byte_perm(v[0], v[1], 0x7632);
        out[4 * c + 3] = __byte_perm(v[2], v[3], 0x7632);
      }
      store_once(static_cast<__nv_bfloat16*>(p.out[which]) + at, out);
    }
  }
}

// ---------------------------------------------------------------- attention
//
//   s[t] = scale * q . k[t],   out = sum_t exp(s[t] - max s) v[t] / sum_t exp(s[t] - max s)
//
// for one query row per sequence and head, heads / kv_heads query heads to a cached head.  Bound by
// memory (D + 8 D / group bytes a position and cached head) as long as the arithmetic on the codes
// keeps up, so:
//
// * The positions of all (sequence, cached head) rows are cut into tiles of 128 and the tiles, in
//   order, into equal runs, one for each thread block of a grid that fills the GPU once (a row
//   counts two tiles more than it has: what its start and end cost): whatever the lengths are (they
//   are read on the device), every SM has the same share.  A row that one
//   block holds whole is written at once; the parts of a row that is cut go to the workspace and a
//   second kernel joins them in block order, so results do not depend on timing.
// * Tiles are fetched into a ring of stages: codes by tiled TMA as rows of 128 bytes (two or four
//   positions) with the 128-byte swizzle, so that the code rows that ldmatrix reads lie in distinct
//   banks; scales by bulk copies.
// * Four warps take twice 16 positions of a tile each (two independent chains of products), with
//   their own running maximum, sum and accumulator; they meet only at the end of a run's row.  The
//   warps refill the ring in turn: a warp of its own for that would cost registers that the others
//   need.
// * Scores are computed transposed, S^T[16 positions x 8 heads] = K Q^T with mma.sync (m16n8k16):
//   decoded codes are the A operand straight from registers (tcgen05 would want them written to
//   shared or tensor memory first, four times the cache bytes), and eight query heads fill a
//   tile's columns.  The exponentials, transposed in registers, are the B operand of
//   O^T[channels x 8 heads] += V^T P^T, whose A operand ldmatrix.trans delivers as pairs of
//   positions with four channels each.
//
// Codes are never converted: `word & 0x000f000f` read as two FP16 numbers is code * 2^-24 exactly
// (subnormal; the tensor cores take those at full rate), `& 0x00f000f0` is 16 times that, and a
// shift by 8 gives the other two pairs: five integer instructions for eight codes.  Scales and
// zeros are applied outside the products:
// * keys: s = scale_k * (q . codes) + zero_k * (sum of q), per group, in FP32.  The query enters as
//   FP16 times a power of two per head, exactly down to 2^-22 of its largest element.
// * values: out = sum_t (p_t scale_v[t]) (codes[t] - 8) + sum_t p_t (zero_v[t] + 8 scale_v[t]), per group;
//   the second sum is FP32.  (Without the 8 both sums would be some 3 where the values average to 0: over
//   262144 positions that cancellation cost 2.5 times the output's own rounding.  One product of the
//   weights with a constant operand gives what the 8 takes off every channel; it is added to the
//   accumulators every fourth tile.)  p_t scale_v[t] enters as FP16 (2^-11, an eighth of the
//   output's rounding).  What must fit FP16 is the product, so the reference point of a head's exponentials follows
//   the largest product of weight and value magnitude, not the largest weight: a loud value that
//   hardly weighs anything takes no bits from the others, and values may have any size that
//   FP32 sums of the weights allow.
//
// Measured: 64 sequences x 4096 positions x 8 cached heads (287 MB) 72 us, 2 x 262144 with sixteen query
// heads to a cached one (604 MB) 189 us, 200 sequences of 0 to 8191 positions 25 us, one of 1023 9.5 us.
// When the first took 77, it took 60 without the arithmetic and 64 without the copies: what bounds it is
// the latency of a warp's chain of products, exponentials and products at the twelve (eight) warps that
// the registers allow.  Tiles of 64 positions (85 to 90 us) and four blocks an SM with two stages (84)
// were slower then.
constexpr int kKv4Tile = 128;          // positions in a stage
constexpr int kKv4Warps = 4;
constexpr int kKv4Sub = kKv4Tile / (16 * kKv4Warps);   // groups of 16 positions a warp takes of each tile
constexpr int kKv4RowUnits = 2;
// Resident blocks an SM: three (twelve warps of up to 168 registers), or two with sixteen heads, whose accumulators
// take 212 to 255 registers and which hold twice the queries.
__host__ __device__ constexpr int kv4_per_sm(int head_tiles) { return head_tiles > 1 ? 2 : 3; }
constexpr uint32_t kKv4Lag = 2;
// The largest exponential times value magnitude is 2^kKv4Top when the reference point is set, and 2^kKv4Room
// times that at most before it is set again; times kKv4Unit it is an FP16 number (below 2^15).  The
// factor keeps the exponentials themselves inside FP32's range where values are large: those of values of 2^100
// are some 2^-73, and what is below 2^-126 is lost.  Magnitudes below kKv4Smallest count as that
// (sums of the weights of values that are all zero must not overflow).
constexpr float kKv4Top = 27.0f, kKv4Room = 8.0f, kKv4Unit = 0x1p-20f, kKv4Smallest = 0x1p-60f;
constexpr float kKv4NoScore = -3e38f;     // reference point before the first score: below any but -infinity
// Reference points from here on are too coarse for sums with them: such heads take the exact way at every tile.
constexpr float kKv4Coarse = 0x1p22f;
constexpr int kKv4Threads = kKv4Warps * 32;

struct Kv4Attend {
  const __nv_bfloat16* q;
  const __nv_bfloat162* k_scales;
  const __nv_bfloat162* v_scales;
  const int* table;
  const int* lengths;
  __nv_bfloat16* out;
  float* lse;
  // Workspace: of each block two parts (sums, then maximum and total), and the row it leaves unfinished.
  float* parts;          // [blocks][2][8 kNT heads][D], behind them [blocks][2][8 kNT heads][2]
  // Rows whose parts are to be joined: {sequence, row in it, last block that holds a part, 1 + first block}, or
  // {.., 0}: of every row while there are at most as many rows as blocks, else of the last row that
  // each block begins.
  int4* cuts;
  int cuts_by_row;
  long long q_batch, q_head, table_stride;
  int batch, heads, kv_heads, group_heads, head_blocks, pages, page, max_pages, box, box_shift, page_shift;
  float scale_log2;
};

// Where the run of one block starts, and the size of all.
struct Kv4Start {
  long long total, base;        // units of all rows; units before sequence `sequence`
  int sequence, runs;           // runs: blocks that have one
};

__device__ __forceinline__ int kv4_length(const Kv4Attend& p, int b) {
  const long long most = static_cast<long long>(p.max_pages) * p.page;
  const int n = p.lengths[b];
  return n < 0 ? 0 : n > most ? int(most) : n;
}
__device__ __forceinline__ int kv4_page_of(const Kv4Attend& p, int position) {
  return p.page_shift >= 0 ? position >> p.page_shift : position / p.page;
}
// Units of work of a row: its tiles, and what starting and ending a row costs beside them (none for an
// empty sequence).  The runs are equal in units.
__device__ __forceinline__ int kv4_units(int length) {
  return length ? (length + kKv4Tile - 1) / kKv4Tile + kKv4RowUnits : 0;
}
// First unit of a block's run; `runs` is at most the number of units, so that no run is empty.
__device__ __forceinline__ long long kv4_first_unit(long long total, int runs, int block) {
  if (total < (1 << 20)) return uint32_t(total) * uint32_t(block) / uint32_t(runs);   // (runs are below 2^11)
  return total * block / runs;
}
// Block whose run holds unit t: the largest i with total * i / runs <= t.
__device__ __forceinline__ int kv4_block_of(long long total, int runs, long long t) {
  return int(((t + 1) * runs - 1) / total);
}

// All threads of the block; finds the sequence in which its run begins.
template <int kThreads>
__device__ __forceinline__ Kv4Start kv4_locate(const Kv4Attend& p, int blocks, int block, long long* scratch) {
  constexpr int kWarps = kThreads / 32;
  const int rows = p.kv_heads * p.head_blocks;
  const int per = (p.batch + kThreads - 1) / kThreads;
  const int begin = min(p.batch, int(threadIdx.x) * per), end = min(p.batch, begin + per);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long sum = 0;
  for (int b = begin; b < end; ++b) sum += static_cast<long long>(kv4_units(kv4_length(p, b))) * rows;
  long long inclusive = sum;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const long long below = __shfl_up_sync(0xffffffffu, inclusive, o);
    if (lane >= o) inclusive += below;
  }
  if (lane == 31) scratch[warp] = inclusive;
  __syncthreads();
  long long base = inclusive - sum, total = 0;
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += scratch[w];
    total += scratch[w];
  }
  const int runs = total < blocks ? int(total) : blocks;
  const long long first = block < runs ? kv4_first_unit(total, runs, block) : -1;
  if (first >= base && first < base + sum) {   // exactly one thread, if there is any tile
    int b = begin;
    for (;; ++b) {
      const long long n = static_cast<long long>(kv4_units(kv4_length(p, b))) * rows;
      if (first < base + n) break;
      base += n;
    }
    scratch[kWarps] = base;
    scratch[kWarps + 1] = b;
  }
  __syncthreads();
  Kv4Start s;
  s.total = total;
  s.base = scratch[kWarps];
  s.sequence = int(scratch[kWarps + 1]);
  s.runs = runs;
  return s;
}

// Walks the rows (sequence, cached head, head block) that a run of tiles covers.
struct Kv4Walk {
  long long next, end;       // units of the run not yet visited
  long long base;            // first unit of sequence b
  int b, length, units, tiles;
  // the current piece
  int row, first, count;     // row within the sequence, first tile of the piece, its tiles (0: the run is over)
  int kv, hb;                // cached head and head block of the row
  int tile;                  // for next_tile
  Kv4Walk() = default;
  __device__ __forceinline__ Kv4Walk(const Kv4Attend& p, const Kv4Start& s, int block) {
    next = end = 0;
    if (block < s.runs) {
      next = kv4_first_unit(s.total, s.runs, block);
      end = kv4_first_unit(s.total, s.runs, block + 1);
    }
    base = s.base;
    b = s.sequence;
    length = next < end ? kv4_length(p, b) : 0;
    units = kv4_units(length);
  }
  __device__ __forceinline__ bool step(const Kv4Attend& p) {
    if (next >= end) {
      count = 0;
      return false;
    }
    const int rows = p.kv_heads * p.head_blocks;
    for (;;) {
      while (next >= base + static_cast<long long>(units) * rows) {   // the run ends inside a sequence with tiles
        base += static_cast<long long>(units) * rows;
        ++b;
        length = kv4_length(p, b);
        units = kv4_units(length);
      }
      const int local = int(next - base);
      row = local / units;
      const int from = local - row * units;
      const long long left = end - next;
      const int to = int(left < units - from ? from + left : units);
      next += to - from;
      tiles = units - kKv4RowUnits;
      first = max(0, from - kKv4RowUnits);
      count = to - kKv4RowUnits - first;
      if (count > 0) break;
      if (next >= end) {
        count = 0;
        return false;
      }
    }
    tile = first;
    kv = p.head_blocks == 1 ? row : row / p.head_blocks;
    hb = row - kv * p.head_blocks;
    return true;
  }
  __device__ __forceinline__ bool next_tile(const Kv4Attend& p) { return ++tile < first + count || step(p); }
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float exp2_approx(float x) {   // 2^-22 relative; results below 2^-126 are 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_or_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <bool kTrans>
__device__ __forceinline__ void load_matrices(uint32_t a, uint32_t (&r)[4]) {
  if (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
// The (scale, zero) pairs of one position.
template <int kNG>
__device__ __forceinline__ void load_pairs(uint32_t a, uint32_t (&r)[kNG]) {
  if (kNG == 1)
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r[0]) : "r"(a));
  else if (kNG == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1 % kNG]) : "r"(a));
  else
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1 % kNG]), "=r"(r[2 % kNG]), "=r"(r[3 % kNG]) : "r"(a));
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
template <int kD, int kNG>
__host__ __device__ constexpr int kv4_stage_bytes() {
  return 2 * kKv4Tile * (kD / 2) + 2 * kKv4Tile * kNG * 4;
}
template <int kD>
__host__ __device__ constexpr int kv4_join_bytes() {   // four heads' accumulators per warp, rows padded by four floats, and (maximum, sum)
  return kKv4Warps * 4 * ((kD + 4) * 4 + 8);
}
template <int kD, int kNT>
__host__ __device__ constexpr int kv4_query_bytes() {
  return 2 * kNT * (kD / 32) * 32 * 16;
}
template <int kD, int kNG, int kNT>
__host__ __device__ constexpr int kv4_stages() {
  // what a block's share of an SM's 228 KB leaves beside the system's 1 KB a block, static variables and alignment
  return (228 * 1024 / kv4_per_sm(kNT) - 3 * 1024 - kv4_join_bytes<kD>() - kv4_query_bytes<kD, kNT>()) / kv4_stage_bytes<kD, kNG>();
}
template <int kD, int kNG, int kNT>
__host__ __device__ constexpr int kv4_smem_bytes() {
  return 1024 + kv4_stages<kD, kNG, kNT>() * kv4_stage_bytes<kD, kNG>() + kv4_query_bytes<kD, kNT>() +
         kv4_join_bytes<kD>() + 256;
}

template <int kD, int kNG, int kNT>
__global__ void __launch_bounds__(kKv4Threads, kv4_per_sm(kNT))
kv4_attend_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                  const Kv4Attend p) {
  constexpr int kRow = kD / 2;                         // bytes of codes a position
  constexpr int kCodes = kKv4Tile * kRow;
  constexpr int kScales = kKv4Tile * kNG * 4;
  constexpr int kStages = kv4_stages<kD, kNG, kNT>();
  constexpr int kStage = kv4_stage_bytes<kD, kNG>();
  constexpr int kChunks = kD / 32;                     // 16-byte chunks of a code row
  constexpr int kMT = kD / 16;                         // channel tiles of the accumulator
  constexpr int kHeads = 8 * kNT;
  constexpr int kPitch = kD + 4;
  static_assert(kStages >= 2, "the ring needs two stages");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem = smem_raw + (base - smem_u32(smem_raw));
  uint4 (*query)[kChunks][32] = reinterpret_cast<uint4 (*)[kChunks][32]>(smem + kStages * kStage);   // [tile of heads][chunk][lane]
  uint4 (*raw_query)[kChunks][32] = query + kNT;                                                      // the same, as it came
  float* join = reinterpret_cast<float*>(smem + kStages * kStage + kv4_query_bytes<kD, kNT>());       // [warp][head][kPitch]
  float* join_ml = join + kKv4Warps * 4 * kPitch;                                                     // [warp][head][2]
  const uint32_t bars = base + kStages * kStage + kv4_query_bytes<kD, kNT>() + kv4_join_bytes<kD>();
  __shared__ float factors[kHeads][1 + kNG];     // of a head's scores: scale, and zero per group
  auto full = [&](int s) { return bars + 8u * s; };
  auto empty = [&](int s) { return bars + 8u * (kStages + s); };
  __shared__ long long locate_scratch[kKv4Threads / 32 + 2];
  __shared__ uint32_t fetched[kStages];                    // tiles fetched into a stage so far
  static_assert(kStages > int(kKv4Lag), "a tile must be on its way before it is waited for");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), kKv4Warps);
      fetched[s] = 0;
    }
    mbar_fence_init();
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  grid_dependency_wait();
  grid_dependents_may_launch();
  const int blocks = gridDim.x, block = blockIdx.x;
  const Kv4Start start = kv4_locate<kKv4Threads>(p, blocks, block, locate_scratch);   // also orders the barriers
  Kv4Walk walk(p, start, block);

  // ---------------------------------------------------------- refilling the ring
  // At tile i one warp, number i modulo the warps, fetches tile i - kKv4Lag + kStages once all warps are
  // through with tile i - kKv4Lag.  Every warp walks its own every-fourth tile ahead and has loaded its
  // page numbers (each lane that of its copy) since its last turn.
  auto load_page = [&](const Kv4Walk& at) {       // page of this lane's piece of the tile, if it has one
    const int piece = lane >> 2;
    const int live = (min(kKv4Tile, at.length - at.tile * kKv4Tile) + p.box - 1) >> p.box_shift;
    return piece < live ? p.table[at.b * p.table_stride + kv4_page_of(p, at.tile * kKv4Tile + (piece << p.box_shift))] : 0;
  };
  auto issue = [&](const Kv4Walk& at, int s, int page) {             // one warp: a tile's copies into stage s
    const int live = (min(kKv4Tile, at.length - at.tile * kKv4Tile) + p.box - 1) >> p.box_shift;
    if (lane == 0) {
      mbar_arrive_expect_tx(full(s), uint32_t(live << p.box_shift) * (2 * kRow + 8 * kNG));
      ++fetched[s];
    }
    __syncwarp();
    const uint32_t stage = base + s * kStage;
    const int piece = lane >> 2, kind = lane & 3;
    if (piece < live) {
      if (page < 0 || page >= p.pages) {   // nothing outside the cache is read
        report_timeout(kSiteKv4Page);
        page = 0;
      }
      const int position = at.tile * kKv4Tile + (piece << p.box_shift);
      // (the cache has fewer than 2^31 rows)
      const int row = (page * p.kv_heads + at.kv) * p.page + (position - kv4_page_of(p, position) * p.page);
      if (kind < 2)
        tma_load_3d(stage + kind * kCodes + piece * p.box * kRow, kind ? &map_v : &map_k, full(s), 0, row / (128 / kRow), 0);
      else
        bulk_load(stage + 2 * kCodes + (kind - 2) * kScales + piece * p.box * kNG * 4,
                  (kind == 2 ? p.k_scales : p.v_scales) + static_cast<long long>(row) * kNG, uint32_t(p.box) * kNG * 4, full(s));
    }
  };
  Kv4Walk ahead = walk;
  bool ahead_some = ahead.step(p);
  int ahead_page = 0;
  {
    int behind = 0;
    auto advance = [&](int tile) {
      for (; behind < tile && ahead_some; ++behind) ahead_some = ahead.next_tile(p);
    };
    for (int s = warp; s < kStages; s += kKv4Warps) {        // the first tiles
      advance(s);
      if (ahead_some) issue(ahead, s, load_page(ahead));
    }
    advance((warp >= int(kKv4Lag) ? warp : warp + kKv4Warps) - int(kKv4Lag) + kStages);
    if (ahead_some) ahead_page = load_page(ahead);
  }
  {
    // ---------------------------------------------------------- attention
    // sequences without a position: nothing to attend to, the output row is zero
    for (int b = block; b < p.batch; b += blocks) {
      if (kv4_length(p, b)) continue;
      for (int i = threadIdx.x; i < p.heads * kD / 8; i += kKv4Threads)
        reinterpret_cast<uint4*>(p.out)[static_cast<long long>(b) * p.heads * kD / 8 + i] = make_uint4(0, 0, 0, 0);
      if (p.lse)
        for (int i = threadIdx.x; i < p.heads; i += kKv4Threads)
          p.lse[static_cast<long long>(b) * p.heads + i] = -INFINITY;
      if (p.cuts_by_row)
        for (int i = threadIdx.x; i < p.kv_heads * p.head_blocks; i += kKv4Threads)
          p.cuts[b * p.kv_heads * p.head_blocks + i] = make_int4(0, 0, 0, 0);
    }
    const int g = lane >> 2, t = lane & 3;
    // ldmatrix: lane l gives the address of row l & 7 of matrix l >> 3, which are (positions 0-7, 8-15) x
    // (an even, the next odd 16-byte chunk); chunks are swizzled, chunk ^ bits 7-9 of the offset.
    const uint32_t matrix_row = (warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * kRow + (lane >> 4) * 16;
    constexpr uint32_t kSubBytes = kKv4Warps * 16 * kRow;       // a multiple of 1024: the swizzle repeats
    const uint32_t matrix_offset = matrix_row ^ (((matrix_row >> 7) & 7) << 4);
    const int position0 = warp * 16 + g;                        // first row of the lane's scores
    // -8 in the form of the codes, for even and odd channels
    const uint32_t minus_eight[4] = {0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u};
    uint32_t it = 0, stage = 0, parity = 0;     // of the next tile: its number, stage and round
    bool ok = true;
    int4 cut = make_int4(0, 0, 0, 0);
    // The query rows of a piece are copied to shared memory while the piece before it is worked on.
    auto fetch_query = [&](const Kv4Walk& at) {
      if (warp >= kNT) return;
      const int in_block = warp * 8 + g, in_group = at.hb * kHeads + in_block;
      const __nv_bfloat16* src = p.q + at.b * p.q_batch +
                                 (at.kv * p.group_heads + (in_group < p.group_heads ? in_group : 0)) * p.q_head;
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_u32(&raw_query[warp][j][lane])),
                     "l"(src + 32 * j + 8 * t)
                     : "memory");
    };
    bool more = walk.step(p);
    if (more) {
      fetch_query(walk);
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    Kv4Walk after = walk;
    for (; more; walk = after) {
      const int head0 = walk.kv * p.group_heads + walk.hb * kHeads;     // first query head of the block
      const int heads_here = min(kHeads, p.group_heads - walk.hb * kHeads);
      if (warp < kNT) {
        // Query fragments of eight heads: lane (g, t) prepares channels 32 j + 8 t + (0..7) of head
        // 8 warp + g, which are the words it will read back.
        float x[kChunks][8], top = 0.0f, sums[kNG];
#pragma unroll
        for (int i = 0; i < kNG; ++i) sums[i] = 0.0f;
        const bool live = warp * 8 + g < heads_here;
        uint4 raw[kChunks];      // written by this very lane, which has waited for its copies
#pragma unroll
        for (int j = 0; j < kChunks; ++j) raw[j] = raw_query[warp][j][lane];
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[j][2 * e] = live ? bf16_lo(w[e]) : 0.0f;
            x[j][2 * e + 1] = live ? bf16_hi(w[e]) : 0.0f;
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            top = fmaxf(top, fabsf(x[j][e]));
            sums[j * kNG / kChunks] += x[j][e];
          }
        }
#pragma unroll
        for (int o = 1; o < 4; o *= 2) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
          for (int i = 0; i < kNG; ++i) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], o);
        }
        // power of two that brings the head's largest element to [2^11, 2^12)
        int exponent = top > 0.0f && top < INFINITY ? 11 - ilogbf(top) : 0;
        exponent = min(exponent, 100);
        const float up = exp2f(static_cast<float>(exponent));
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = (e & 1) ? up * 0.0625f : up;      // odd nibbles enter 16 times too large
            const __half2 h = __floats2half2_rn(x[j][e] * f, x[j][e + 4] * f);
            w[e] = *reinterpret_cast<const uint32_t*>(&h);
          }
          query[warp][j][lane] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (t == 0) {
          factors[warp * 8 + g][0] = ldexpf(p.scale_log2, 24 - exponent);     // 2^24: the codes' unit
#pragma unroll
          for (int i = 0; i < kNG; ++i) factors[warp * 8 + g][1 + i] = sums[i] * p.scale_log2;
        }
      }
      more = after.step(p);
      if (more) fetch_query(after);
      __syncthreads();
      float score_factor[kNT][2], zero_factor[kNT][2][kNG];    // lane (g, t): heads 2 t and 2 t + 1 of a tile
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          score_factor[n][c] = factors[n * 8 + 2 * t + c][0];
#pragma unroll
          for (int i = 0; i < kNG; ++i) zero_factor[n][c][i] = factors[n * 8 + 2 * t + c][1 + i];
        }
      float acc[kNT][kMT][4], zeros[kNT][2][kNG], ref[kNT][2], sum[kNT][2];
#pragma unroll
      for (int n = 0; n < kNT; ++n) {
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][i][e] = 0.0f;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          ref[n][c] = kKv4NoScore;
          sum[n][c] = 0.0f;
#pragma unroll
          for (int i = 0; i < kNG; ++i) zeros[n][c][i] = 0.0f;
        }
      }
      float shift[kNT][kNG][4];      // the -8's part of the accumulators, which takes it in every few tiles
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int i = 0; i < kNG; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) shift[n][i][e] = 0.0f;
      for (int tile = walk.first; tile < walk.first + walk.count; ++tile, ++it) {
        if (ok && it >= kKv4Lag && warp == int(it % kKv4Warps)) {
          // the stage of tile it - kKv4Lag, in the round before this one's if it lies behind this one's stage
          const bool wrapped = stage < kKv4Lag;
          const uint32_t free = wrapped ? stage + kStages - kKv4Lag : stage - kKv4Lag;
          ok = __all_sync(0xffffffffu, mbar_wait(empty(free), wrapped ? parity ^ 1u : parity, 0x911));
          if (ok && ahead_some) {
            issue(ahead, int(free), ahead_page);
            for (int i = 0; i < kKv4Warps && ahead_some; ++i) ahead_some = ahead.next_tile(p);
            if (ahead_some) ahead_page = load_page(ahead);
          }
        }
        const uint32_t s = stage;
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(full(s), parity, 0x912));
        if (++stage == kStages) {
          stage = 0;
          parity ^= 1u;
        }
        const int live = walk.length - tile * kKv4Tile;     // positions of the tile that exist
        if (ok && warp * 16 < live) {
          const uint32_t keys = base + s * kStage, values = keys + kCodes;
          const uint32_t key_scales = values + kCodes, value_scales = key_scales + kScales;
          float dot[kKv4Sub][kNT][kNG][4];
#pragma unroll
          for (int u = 0; u < kKv4Sub; ++u)
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int i = 0; i < kNG; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) dot[u][n][i][e] = 0.0f;
#pragma unroll
          for (int jj = 0; jj < kChunks / 2; ++jj) {
            uint32_t w[kKv4Sub][4];
#pragma unroll
            for (int u = 0; u < kKv4Sub; ++u) load_matrices<false>((keys + u * kSubBytes + matrix_offset) ^ (jj << 5), w[u]);
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              const int j = 2 * jj + q, i = j * kNG / kChunks;
              uint4 qf[kNT];
#pragma unroll
              for (int n = 0; n < kNT; ++n) qf[n] = query[n][j][lane];
#pragma unroll
              for (int u = 0; u < kKv4Sub; ++u)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const uint32_t lo = half ? w[u][2 * q] >> 8 : w[u][2 * q], hi = half ? w[u][2 * q + 1] >> 8 : w[u][2 * q + 1];
                  const uint32_t a[4] = {lo & 0x000f000fu, hi & 0x000f000fu, lo & 0x00f000f0u, hi & 0x00f000f0u};
#pragma unroll
                  for (int n = 0; n < kNT; ++n)
                    mma_f16(dot[u][n][i], a, half ? qf[n].z : qf[n].x, half ? qf[n].w : qf[n].y);
                }
            }
          }
          float score[kKv4Sub][kNT][4];
          uint32_t value_pair[kKv4Sub][2][kNG];
#pragma unroll
          for (int u = 0; u < kKv4Sub; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const int position = u * (kKv4Warps * 16) + position0 + 8 * r;
              uint32_t pair[kNG];
              load_pairs<kNG>(key_scales + position * (kNG * 4), pair);
              load_pairs<kNG>(value_scales + position * (kNG * 4), value_pair[u][r]);
#pragma unroll
              for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  float x = dot[u][n][0][2 * r + c] * bf16_lo(pair[0]), z = bf16_hi(pair[0]) * zero_factor[n][c][0];
#pragma unroll
                  for (int i = 1; i < kNG; ++i) {
                    x = fmaf(dot[u][n][i][2 * r + c], bf16_lo(pair[i]), x);
                    z = fmaf(bf16_hi(pair[i]), zero_factor[n][c][i], z);
                  }
                  score[u][n][2 * r + c] = fmaf(x, score_factor[n][c], z);
                }
            }
          if (live < kKv4Tile) {
            // what lies behind the sequence, NaN included, weighs nothing
#pragma unroll
            for (int u = 0; u < kKv4Sub; ++u)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (u * (kKv4Warps * 16) + position0 + 8 * r >= live) {
#pragma unroll
                  for (int n = 0; n < kNT; ++n) score[u][n][2 * r] = score[u][n][2 * r + 1] = -INFINITY;
#pragma unroll
                  for (int i = 0; i < kNG; ++i) value_pair[u][r][i] = 0;
                }
          }
          // The reference point of a head's exponentials lies kKv4Top below the largest score plus logarithm of
          // the value's magnitude (an upper bound: the exponent and one) when it was last set, and is set
          // again only when one exceeds that by kKv4Room (most tiles need neither the shuffles nor the
          // rescaling).  FP16 keeps products of weight and scale down to 2^-30 of the largest of weight and
          // magnitude.  A group whose scale is NaN is NaN in the result whatever it weighs: its
          // zero, which may be infinite, does not count.
          float level[kKv4Sub][2];
#pragma unroll
          for (int u = 0; u < kKv4Sub; ++u)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float size = kKv4Smallest;
#pragma unroll
              for (int i = 0; i < kNG; ++i)
                size = fmaxf(size, max_or_nan(fabsf(bf16_lo(value_pair[u][r][i])), fabsf(bf16_hi(value_pair[u][r][i]))));
              level[u][r] = __uint_as_float(0x4b000000u | __float_as_uint(size) >> 23) - (8388608.0f + 126.0f);
            }
          bool raise = false;
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) raise |= !(fabsf(ref[n][c]) < kKv4Coarse);
#pragma unroll
          for (int u = 0; u < kKv4Sub; ++u)
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                raise |= score[u][n][e] + level[u][e >> 1] > ref[n][e & 1] + (kKv4Top + kKv4Room);
          if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                // the largest score, and relative to it (exactly) the largest score and logarithm
                float m = -INFINITY, top = -INFINITY;
#pragma unroll
                for (int u = 0; u < kKv4Sub; ++u) m = fmaxf(m, fmaxf(score[u][n][c], score[u][n][2 + c]));
#pragma unroll
                for (int o = 4; o < 32; o *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
                for (int u = 0; u < kKv4Sub; ++u)
                  top = fmaxf(top, fmaxf((score[u][n][c] - m) + level[u][0], (score[u][n][2 + c] - m) + level[u][1]));
#pragma unroll
                for (int o = 4; o < 32; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                float next = m + (top - kKv4Top), f = 1.0f;
                if ((m - next) + top > kKv4Top + kKv4Room)        // rounded too far down (scores of 2^28)
                  next = __int_as_float(__float_as_int(next) + (next < 0.0f ? -1 : 1));
                if (next > ref[n][c]) {
                  f = exp2_approx(ref[n][c] - next);
                  ref[n][c] = next;
                }
                sum[n][c] *= f;
#pragma unroll
                for (int i = 0; i < kNG; ++i) zeros[n][c][i] *= f;
#pragma unroll
                for (int i = 0; i < kNG; ++i) {
                  shift[n][i][c] *= f;
                  shift[n][i][2 + c] *= f;
                }
#pragma unroll
                for (int i = 0; i < kMT; ++i) {
                  acc[n][i][c] *= f;
                  acc[n][i][2 + c] *= f;
                }
              }
          }
#pragma unroll
          for (int u = 0; u < kKv4Sub; ++u) {
            float (&weight)[kNT][4] = score[u];
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                weight[n][e] = exp2_approx(score[u][n][e] - ref[n][e & 1]);
                sum[n][e & 1] += weight[n][e];
              }
            uint32_t pf[kNT][kNG][2];
#pragma unroll
            for (int i = 0; i < kNG; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                const float scale = bf16_lo(value_pair[u][r][i]) * kKv4Unit;
                const float zero = fmaf(8.0f, bf16_lo(value_pair[u][r][i]), bf16_hi(value_pair[u][r][i]));
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
                  const __half2 h = __floats2half2_rn(weight[n][2 * r] * scale, weight[n][2 * r + 1] * scale);
                  pf[n][i][r] = transpose_8x8(*reinterpret_cast<const uint32_t*>(&h));
#pragma unroll
                  for (int c = 0; c < 2; ++c) zeros[n][c][i] = fmaf(weight[n][2 * r + c], zero, zeros[n][c][i]);
                }
              }
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
              for (int i = 0; i < kNG; ++i) mma_f16(shift[n][i], minus_eight, pf[n][i][0], pf[n][i][1]);
            // A chunk of 32 channels: lane (g, t) holds channels 4 g .. 4 g + 3 of positions 2 t, 2 t + 1 (and + 8);
            // two tiles of 16 channels, row g the even and row g + 8 the odd channel (16 times too large).
#pragma unroll
            for (int jj = 0; jj < kChunks / 2; ++jj) {
              uint32_t w[4];
              load_matrices<true>((values + u * kSubBytes + matrix_offset) ^ (jj << 5), w);
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const int j = 2 * jj + q, i = j * kNG / kChunks;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                  const uint32_t lo = half ? w[2 * q] >> 8 : w[2 * q], hi = half ? w[2 * q + 1] >> 8 : w[2 * q + 1];
                  const uint32_t a[4] = {lo & 0x000f000fu, lo & 0x00f000f0u, hi & 0x000f000fu, hi & 0x00f000f0u};
#pragma unroll
                  for (int n = 0; n < kNT; ++n) mma_f16(acc[n][2 * j + half], a, pf[n][i][0], pf[n][i][1]);
                }
              }
            }
          }
        }
        if ((tile & 3) == 3 || tile + 1 == walk.first + walk.count) {
#pragma unroll
          for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
              for (int i = 0; i < kMT; ++i) acc[n][i][e] += shift[n][i * kNG / kMT][e];
#pragma unroll
              for (int i = 0; i < kNG; ++i) shift[n][i][e] = 0.0f;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");    // the next query, if this warp asked for it
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(s));
      }
      // ---- the warps' parts of this piece meet, four heads (those of one accumulator column) at a time
      const bool whole = walk.count == walk.tiles;
      if (walk.first == 0) {
        cut = make_int4(0, 0, 0, 0);
        if (!whole) {
          const long long row_end = walk.base + static_cast<long long>(walk.row + 1) * walk.units;
          cut = make_int4(walk.b, walk.row, kv4_block_of(start.total, start.runs, row_end - 1), 1 + block);
        }
        if (threadIdx.x == 0 && p.cuts_by_row) p.cuts[walk.b * p.kv_heads * p.head_blocks + walk.row] = cut;
      }
      const int slot = walk.first == 0 ? 1 : 0;   // part 0: the row began in an earlier block
#pragma unroll
      for (int n = 0; n < kNT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (8 * n + c >= heads_here) continue;      // (for all threads: no head of the row is in this round)
          if (n | c) __syncthreads();
#pragma unroll
          for (int o = 4; o < 32; o *= 2) sum[n][c] += __shfl_xor_sync(0xffffffffu, sum[n][c], o);
#pragma unroll
          for (int i = 0; i < kNG; ++i)
#pragma unroll
            for (int o = 4; o < 32; o *= 2) zeros[n][c][i] += __shfl_xor_sync(0xffffffffu, zeros[n][c][i], o);
          float* mine = join + (warp * 4 + t) * kPitch + g * 4;
          constexpr float even = 0x1p24f / kKv4Unit, odd = 0x1p20f / kKv4Unit;     // the units of codes and weights
#pragma unroll
          for (int j = 0; j < kChunks; ++j) {
            const float zero = zeros[n][c][j * kNG / kChunks];
            *reinterpret_cast<float4*>(mine + 32 * j) =
                make_float4(fmaf(acc[n][2 * j][c], even, zero), fmaf(acc[n][2 * j][2 + c], odd, zero),
                            fmaf(acc[n][2 * j + 1][c], even, zero), fmaf(acc[n][2 * j + 1][2 + c], odd, zero));
          }
          if (g == 0) {
            join_ml[(warp * 4 + t) * 2] = ref[n][c];
            join_ml[(warp * 4 + t) * 2 + 1] = sum[n][c];
          }
          __syncthreads();
          static_assert(kKv4Threads == 4 * 32 && kD / 4 <= 32, "a thread joins four channels of one head");
          const int place = threadIdx.x / (kD / 4), channel = (threadIdx.x - place * (kD / 4)) * 4;
          const int head = 8 * n + 2 * place + c;
          if (place >= 4 || head >= heads_here) continue;
          float m = -INFINITY;
#pragma unroll
          for (int w = 0; w < kKv4Warps; ++w) m = fmaxf(m, join_ml[(w * 4 + place) * 2]);
          float total = 0.0f;
          float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
          for (int w = 0; w < kKv4Warps; ++w) {
            const float mw = join_ml[(w * 4 + place) * 2], lw = join_ml[(w * 4 + place) * 2 + 1];
            const float f = exp2f(mw - m);
            const float4 x = *reinterpret_cast<const float4*>(join + (w * 4 + place) * kPitch + channel);
            total = fmaf(lw, f, total);
            o.x = fmaf(x.x, f, o.x);
            o.y = fmaf(x.y, f, o.y);
            o.z = fmaf(x.z, f, o.z);
            o.w = fmaf(x.w, f, o.w);
          }
          if (whole) {
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            const long long at = static_cast<long long>(walk.b) * p.heads + head0 + head;
            *reinterpret_cast<uint2*>(p.out + at * kD + channel) =
                make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
            if (p.lse && channel == 0) p.lse[at] = (m + log2f(total)) * 0.69314718055994531f;
          } else {
            const long long at = (static_cast<long long>(block) * 2 + slot) * kHeads + head;
            *reinterpret_cast<float4*>(p.parts + at * kD + channel) = o;
            if (channel == 0) {
              float* ml = p.parts + static_cast<long long>(blocks) * 2 * kHeads * kD + at * 2;
              ml[0] = m;
              ml[1] = total;
            }
          }
        }
      // (the next piece writes the join area behind the barrier that follows its query)
    }
    // (a block that begins no row, or ends the last one that it begins, leaves nothing to join)
    if (threadIdx.x == 0 && !p.cuts_by_row) p.cuts[block] = cut;
    // After a wait that gave up, nothing may still be in flight into this block's shared memory.
    if (__syncthreads_or(!ok))
      for (int s = 0; s < kStages; ++s)
        if (fetched[s]) mbar_wait(full(s), (fetched[s] - 1) & 1u, 0x913);
  }
}

// Joins the parts of a row that was cut, in a fixed order; blockIdx.x counts the entries of `cuts`.  How many parts a
// row has depends on the lengths, which only the device knows (one long sequence among many short ones is
// spread over almost all blocks), so a block decides what it does: of a row of up to kFewParts parts the
// first block of each eight heads takes one head a warp, and the others leave; of a longer one every block takes
// kJoinHeads heads, with the parts dealt out to its warps, which meet in shared memory.  (When the host chose, by the
// average number of parts: one sequence of 131072 positions beside 63 of 16 took 50 us, now 25; 200 sequences of
// 0 to 8191 28 and 25, 2 x 262144 192 and 189; 64 x 4096 70 and 71.5, for the blocks that leave.)
constexpr int kJoinWarps = 8, kJoinHeads = 2, kFewParts = 16;
template <int kD, int kHeads>
__global__ void __launch_bounds__(32 * kJoinWarps) kv4_join_kernel(const Kv4Attend p, int blocks) {
  constexpr int kPerLane = kD / 32;
  __shared__ float sums[kJoinWarps][kD], ml_shared[kJoinWarps][2];
  grid_dependents_may_launch();
  grid_dependency_wait();
  const int4 cut = p.cuts[blockIdx.x];
  if (!cut.w) return;
  const int first = cut.w - 1, last = cut.z;
  const bool few = last - first < kFewParts;
  const int heads_here = few ? kJoinWarps : kJoinHeads, groups = kJoinWarps / heads_here;
  if (int(blockIdx.y) * heads_here >= kHeads) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = blockIdx.y * heads_here + warp % heads_here, group = warp / heads_here;
  const float* parts_ml = p.parts + static_cast<long long>(blocks) * 2 * kHeads * kD;
  float m = -INFINITY, total = 0.0f, o[kPerLane];
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) o[e] = 0.0f;
  constexpr int kBatch = 8;      // parts whose loads are in flight together
  for (int c0 = first + group; c0 <= last; c0 += kBatch * groups) {
    float x[kBatch][kPerLane], mc[kBatch], lc[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = c0 + u * groups;
      const long long at = (static_cast<long long>(c) * 2 + (c == first ? 1 : 0)) * kHeads + head;
      mc[u] = -INFINITY;
      lc[u] = 0.0f;
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) x[u][e] = 0.0f;
      if (c <= last) {
        const float2 ml = *reinterpret_cast<const float2*>(parts_ml + at * 2);
        mc[u] = ml.x;
        lc[u] = ml.y;
        if (kPerLane == 4) {
          const float4 v = *reinterpret_cast<const float4*>(p.parts + at * kD + lane * 4);
          x[u][0] = v.x; x[u][1] = v.y; x[u][2 % kPerLane] = v.z; x[u][3 % kPerLane] = v.w;
        } else {
          const float2 v = *reinterpret_cast<const float2*>(p.parts + at * kD + lane * 2);
          x[u][0] = v.x; x[u][1] = v.y;
        }
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) top = fmaxf(top, mc[u]);
    const float back = m == -INFINITY ? (total == 0.0f ? 0.0f : 1.0f) : exp2f(m - top);
    total *= back;
#pragma unroll
    for (int e = 0; e < kPerLane; ++e) o[e] *= back;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const float f = mc[u] == -INFINITY ? (lc[u] == 0.0f ? 0.0f : 1.0f) : exp2f(mc[u] - top);
      total = fmaf(lc[u], f, total);
#pragma unroll
      for (int e = 0; e < kPerLane; ++e) o[e] = fmaf(x[u][e], f, o[e]);
    }
    m = top;
  }
#pragma unroll
  for (int e = 0; e < kPerLane; ++e) sums[warp][lane * kPerLane + e] = o[e];
  if (lane == 0) {
    ml_shared[warp][0] = m;
    ml_shared[warp][1] = total;
  }
  __syncthreads();
  const int kv = cut.y / p.head_blocks, hb = cut.y - kv * p.head_blocks;
  const int in_group0 = hb * kHeads + blockIdx.y * heads_here;       // first head of the block, within its cached head
  for (int i = threadIdx.x; i < heads_here * kD; i += 32 * kJoinWarps) {
    const int h = i / kD, channel = i - h * kD;
    if (in_group0 + h >= p.group_heads) break;
    float top = -INFINITY, all = 0.0f, sum = 0.0f;
    for (int w = h; w < kJoinWarps; w += heads_here) top = fmaxf(top, ml_shared[w][0]);
    for (int w = h; w < kJoinWarps; w += heads_here) {
      const float mg = ml_shared[w][0], lg = ml_shared[w][1];
      const float f = mg == -INFINITY ? (lg == 0.0f ? 0.0f : 1.0f) : exp2f(mg - top);
      all = fmaf(lg, f, all);
      sum = fmaf(sums[w][channel], f, sum);
    }
    const long long at = static_cast<long long>(cut.x) * p.heads + kv * p.group_heads + in_group0 + h;
    p.out[at * kD + channel] = __float2bfloat16(all == 0.0f ? 0.0f : sum / all);
    if (p.lse && channel == 0) p.lse[at] = (top + log2f(all)) * 0.69314718055994531f;
  }
}

int check_kv4_cache(const char* what, const trinity_sm100_kv4_cache& c) {
  if (!c.k_codes || !c.k_scales || !c.v_codes || !c.v_scales) return fail(TRINITY_SM100_E_INVALID, "%s: null cache pointer", what);
  if (!aligned16(c.k_codes) || !aligned16(c.k_scales) || !aligned16(c.v_codes) || !aligned16(c.v_scales))
    return fail(TRINITY_SM100_E_INVALID, "%s: cache pointers must be 16-byte aligned", what);
  if (c.head_dim != 64 && c.head_dim != 128)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "%s: head_dim %d (64 and 128 are supported)", what, c.head_dim);
  if ((c.group != 32 && c.group != 64 && c.group != 128) || c.group > c.head_dim)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "%s: groups of %d channels (32, 64 and 128, at most head_dim)", what, c.group);
  if (c.pages <= 0 || c.kv_heads <= 0 || c.page <= 0) return fail(TRINITY_SM100_E_INVALID, "%s: empty cache", what);
  if (c.page % 16) return fail(TRINITY_SM100_E_UNSUPPORTED, "%s: a page of %d positions (multiples of 16)", what, c.page);
  if (static_cast<long long>(c.pages) * c.kv_heads > INT32_MAX / c.page)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "%s: the cache has 2^31 rows or more", what);
  return 0;
}

Kv4Rows kv4_rows(const trinity_sm100_kv4_cache& c, const trinity_sm100_kv4_rows& r) {
  Kv4Rows p = {};
  p.codes[0] = static_cast<uint8_t*>(c.k_codes);
  p.codes[1] = static_cast<uint8_t*>(c.v_codes);
  p.scales[0] = static_cast<__nv_bfloat162*>(c.k_scales);
  p.scales[1] = static_cast<__nv_bfloat162*>(c.v_scales);
  p.slots = reinterpret_cast<const long long*>(r.slots);
  p.tokens = r.tokens;
  p.positions = static_cast<long long>(c.pages) * c.page;
  p.token_stride[0] = r.k_token_stride;
  p.token_stride[1] = r.v_token_stride;
  p.head_stride[0] = r.k_head_stride;
  p.head_stride[1] = r.v_head_stride;
  p.kv_heads = c.kv_heads;
  p.page = c.page;
  p.group_shift = __builtin_ctz(c.group);
  p.heads_shift = (c.kv_heads & (c.kv_heads - 1)) == 0 ? __builtin_ctz(c.kv_heads) : -1;
  p.page_shift = (c.page & (c.page - 1)) == 0 ? __builtin_ctz(c.page) : -1;
  return p;
}

// What a thread takes: eight channels of one row while the GPU is not full of such threads (least
// latency), else sixteen of two rows where rows start on 32 bytes, and eight of four where they do not
// (four times the bytes in flight; sixteen channels take half the work on addresses for each).
struct Kv4Grid {
  int words, batch;
  dim3 blocks;
  Kv4Grid(long long tokens, const trinity_sm100_kv4_cache& c, bool wide, int sm_count) {
    const long long lanes = tokens * c.kv_heads * (c.head_dim / 8), resident = 2048ll * sm_count;
    words = lanes > resident && wide ? 2 : 1;
    batch = lanes > resident ? 4 / words : 1;
    blocks = dim3(unsigned((lanes + 256 * words * batch - 1) / (256 * words * batch)), 2);
  }
};
// Whether every row of the keys and values starts on a multiple of `bytes` (the stride of an axis with
// one entry has no meaning).
bool kv4_rows_start_on(int bytes, const trinity_sm100_kv4_rows& r, int element, int kv_heads) {
  const uintptr_t pointers = reinterpret_cast<uintptr_t>(r.k) | reinterpret_cast<uintptr_t>(r.v);
  const long long strides = (r.tokens > 1 ? r.k_token_stride | r.v_token_stride : 0) |
                            (kv_heads > 1 ? r.k_head_stride | r.v_head_stride : 0);
  return pointers % bytes == 0 && strides % (bytes / element) == 0;
}

int check_kv4_rows(const char* what, const trinity_sm100_kv4_cache& c, const trinity_sm100_kv4_rows& r) {
  if (int rc = check_kv4_cache(what, c)) return rc;
  if (!r.k || !r.v || !r.slots) return fail(TRINITY_SM100_E_INVALID, "%s: null pointer", what);
  if (r.tokens <= 0) return fail(TRINITY_SM100_E_INVALID, "%s: empty extent", what);
  if (r.tokens > INT32_MAX / (16 * c.kv_heads)) return fail(TRINITY_SM100_E_UNSUPPORTED, "%s: too many tokens", what);
  if (reinterpret_cast<uintptr_t>(r.slots) % 8) return fail(TRINITY_SM100_E_INVALID, "%s: slots must be 8-byte aligned", what);
  return 0;
}

template <int kD, int kNG, int kNT>
int launch_kv4_attend(const Kv4Attend& p, const CUtensorMap& map_k, const CUtensorMap& map_v, int blocks, cudaStream_t stream) {
  static unsigned long long opted = 0;
  constexpr int kSmem = kv4_smem_bytes<kD, kNG, kNT>();
  static_assert(kSmem <= 232448, "exceeds the 227 KB shared-memory limit");
  auto kernel = kv4_attend_kernel<kD, kNG, kNT>;
  if (int rc = opt_in_shared_memory(reinterpret_cast<const void*>(kernel), kSmem, &opted, "kv4_decode")) return rc;
  {
    KernelLaunch launch(dim3(blocks), dim3(kKv4Threads), kSmem, stream);
    cudaError_t e = cudaLaunchKernelEx(&launch.config, kernel, map_k, map_v, p);
    if (e != cudaSuccess) return fail(TRINITY_SM100_E_CUDA, "kv4_attend launch: %s", cudaGetErrorString(e));
    count_launch();
  }
  if (blocks > 1) {
    const unsigned rows = unsigned(p.batch) * p.kv_heads * p.head_blocks;
    KernelLaunch launch(dim3(p.cuts_by_row ? rows : unsigned(blocks), 8 * kNT / kJoinHeads), dim3(32 * kJoinWarps), 0, stream);
    cudaError_t e = cudaLaunchKernelEx(&launch.config, kv4_join_kernel<kD, 8 * kNT>, p, blocks);
    if (e != cudaSuccess) return fail(TRINITY_SM100_E_CUDA, "kv4_join launch: %s", cudaGetErrorString(e));
    count_launch();
  }
  return check_launch("kv4_decode");
}

int kv4_blocks(int sm_count, int block_heads) { return kv4_per_sm(block_heads / 8) * sm_count; }

}  // namespace
}  // namespace trinity_sm100

using namespace trinity_sm100;

extern "C" int trinity_sm100_kv4_append(const trinity_sm100_kv4_cache* cache, const trinity_sm100_kv4_rows* rows,
                                        void* stream_handle) {
  if (!cache || !rows) return fail(TRINITY_SM100_E_INVALID, "kv4_append: null argument block");
  const trinity_sm100_kv4_rows& r = *rows;
  if (int rc = check_kv4_rows("kv4_append", *cache, r)) return rc;
  if (reinterpret_cast<uintptr_t>(r.k) % 2 || reinterpret_cast<uintptr_t>(r.v) % 2)
    return fail(TRINITY_SM100_E_INVALID, "kv4_append: a pointer is not aligned to its element type");
  int sm_count = 0;
  if (int rc = require_sm100(&sm_count)) return rc;
  Kv4Rows p = kv4_rows(*cache, r);
  p.in[0] = static_cast<const __nv_bfloat16*>(r.k);
  p.in[1] = static_cast<const __nv_bfloat16*>(r.v);
  const bool vectors = kv4_rows_start_on(16, r, 2, cache->kv_heads);
  const Kv4Grid grid(r.tokens, *cache, kv4_rows_start_on(32, r, 2, cache->kv_heads), sm_count);
  KernelLaunch launch(grid.blocks, dim3(256), 0, static_cast<cudaStream_t>(stream_handle));
  cudaError_t e;
#define TRINITY_KV4_APPEND(D)                                                                            \
  e = grid.words == 2   ? cudaLaunchKernelEx(&launch.config, kv4_append_kernel<D, 2, true, 2>, p)        \
      : grid.batch == 4 ? (vectors ? cudaLaunchKernelEx(&launch.config, kv4_append_kernel<D, 1, true, 4>, p)   \
                                   : cudaLaunchKernelEx(&launch.config, kv4_append_kernel<D, 1, false, 4>, p)) \
      : vectors         ? cudaLaunchKernelEx(&launch.config, kv4_append_kernel<D, 1, true, 1>, p)        \
                        : cudaLaunchKernelEx(&launch.config, kv4_append_kernel<D, 1, false, 1>, p);
  if (cache->head_dim == 128) {
    TRINITY_KV4_APPEND(128)
  } else {
    TRINITY_KV4_APPEND(64)
  }
#undef TRINITY_KV4_APPEND
  if (e != cudaSuccess) return fail(TRINITY_SM100_E_CUDA, "kv4_append launch: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("kv4_append");
}

extern "C" int trinity_sm100_kv4_read(const trinity_sm100_kv4_cache* cache, const trinity_sm100_kv4_rows* rows,
                                      int32_t out_dtype, void* stream_handle) {
  if (!cache || !rows) return fail(TRINITY_SM100_E_INVALID, "kv4_read: null argument block");
  const trinity_sm100_kv4_rows& r = *rows;
  if (int rc = check_kv4_rows("kv4_read", *cache, r)) return rc;
  if (out_dtype != TRINITY_SM100_BF16 && out_dtype != TRINITY_SM100_FP32)
    return fail(TRINITY_SM100_E_INVALID, "kv4_read: unknown output dtype %d", out_dtype);
  const int element = out_dtype == TRINITY_SM100_FP32 ? 4 : 2;
  if (!kv4_rows_start_on(16, r, element, cache->kv_heads)) return fail(TRINITY_SM100_E_INVALID, "kv4_read: output rows must start on 16 bytes");
  int sm_count = 0;
  if (int rc = require_sm100(&sm_count)) return rc;
  Kv4Rows p = kv4_rows(*cache, r);
  p.out[0] = r.k;
  p.out[1] = r.v;
  p.out_f32 = out_dtype == TRINITY_SM100_FP32;
  const Kv4Grid grid(r.tokens, *cache, kv4_rows_start_on(32, r, element, cache->kv_heads), sm_count);
  KernelLaunch launch(grid.blocks, dim3(256), 0, static_cast<cudaStream_t>(stream_handle));
  cudaError_t e;
#define TRINITY_KV4_READ(D)                                                                        \
  e = grid.words == 2   ? cudaLaunchKernelEx(&launch.config, kv4_read_kernel<D, 2, 2>, p)           \
      : grid.batch == 4 ? cudaLaunchKernelEx(&launch.config, kv4_read_kernel<D, 1, 4>, p)           \
                        : cudaLaunchKernelEx(&launch.config, kv4_read_kernel<D, 1, 1>, p);
  if (cache->head_dim == 128) {
    TRINITY_KV4_READ(128)
  } else {
    TRINITY_KV4_READ(64)
  }
#undef TRINITY_KV4_READ
  if (e != cudaSuccess) return fail(TRINITY_SM100_E_CUDA, "kv4_read launch: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("kv4_read");
}

extern "C" size_t trinity_sm100_kv4_decode_workspace_bytes(int32_t heads, int32_t kv_heads, int32_t head_dim) {
  int sm_count = 0;
  if (heads <= 0 || kv_heads <= 0 || head_dim <= 0 || heads % kv_heads || require_sm100(&sm_count)) return 0;
  const int group_heads = heads / kv_heads;
  const size_t blocks = kv4_blocks(sm_count, 8);      // the most that any layout uses
  return blocks * 2 * (group_heads > 8 ? 16 : 8) * (size_t(head_dim) + 2) * 4 + blocks * sizeof(int4);
}

extern "C" int trinity_sm100_kv4_decode(const trinity_sm100_kv4_cache* cache, const trinity_sm100_kv4_decode_args* args,
                                        void* stream_handle) {
  if (!cache || !args) return fail(TRINITY_SM100_E_INVALID, "kv4_decode: null argument block");
  const trinity_sm100_kv4_cache& c = *cache;
  const trinity_sm100_kv4_decode_args& a = *args;
  if (int rc = check_kv4_cache("kv4_decode", c)) return rc;
  if (!a.q || !a.out || !a.page_table || !a.lengths) return fail(TRINITY_SM100_E_INVALID, "kv4_decode: null pointer");
  if (a.batch <= 0 || a.heads <= 0 || a.max_pages <= 0) return fail(TRINITY_SM100_E_INVALID, "kv4_decode: empty extent");
  if (a.heads % c.kv_heads)
    return fail(TRINITY_SM100_E_INVALID, "kv4_decode: %d query heads do not divide over %d cached ones", a.heads, c.kv_heads);
  if (a.table_stride < a.max_pages) return fail(TRINITY_SM100_E_INVALID, "kv4_decode: table stride smaller than its row");
  if (!aligned16(a.q) || (a.batch > 1 && a.q_batch_stride % 8) || (a.heads > 1 && a.q_head_stride % 8))
    return fail(TRINITY_SM100_E_INVALID, "kv4_decode: query rows must start on 16 bytes");
  if (!aligned16(a.out) || !aligned16(a.workspace)) return fail(TRINITY_SM100_E_INVALID, "kv4_decode: pointers must be 16-byte aligned");
  if (reinterpret_cast<uintptr_t>(a.page_table) % 4 || reinterpret_cast<uintptr_t>(a.lengths) % 4 ||
      reinterpret_cast<uintptr_t>(a.lse) % 4)
    return fail(TRINITY_SM100_E_INVALID, "kv4_decode: a pointer is not aligned to its element type");
  if (static_cast<long long>(a.max_pages) * c.page > INT32_MAX - kKv4Tile)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "kv4_decode: a table row covers 2^31 positions or more");
  const int group_heads = a.heads / c.kv_heads;
  const int block_heads = group_heads > 8 ? 16 : 8, head_blocks = (group_heads + block_heads - 1) / block_heads;
  if (((static_cast<long long>(a.max_pages) * c.page + kKv4Tile - 1) / kKv4Tile + kKv4RowUnits) * c.kv_heads * head_blocks > INT32_MAX)
    return fail(TRINITY_SM100_E_UNSUPPORTED, "kv4_decode: a sequence of up to %lld positions is too long for %d heads",
                static_cast<long long>(a.max_pages) * c.page, a.heads);
  // (behind the checks of the layout: the size of the workspace is 0 for one that is refused)
  if (!a.workspace) return fail(TRINITY_SM100_E_INVALID, "kv4_decode: null workspace");
  int sm_count = 0;
  if (int rc = require_sm100(&sm_count)) return rc;
  const size_t need = trinity_sm100_kv4_decode_workspace_bytes(a.heads, c.kv_heads, c.head_dim);
  if (a.workspace_bytes < need)
    return fail(TRINITY_SM100_E_INVALID, "kv4_decode: workspace of %zu bytes, %zu needed", a.workspace_bytes, need);
  Kv4Attend p;
  p.q = static_cast<const __nv_bfloat16*>(a.q);
  p.k_scales = static_cast<const __nv_bfloat162*>(c.k_scales);
  p.v_scales = static_cast<const __nv_bfloat162*>(c.v_scales);
  p.table = static_cast<const int*>(a.page_table);
  p.lengths = static_cast<const int*>(a.lengths);
  p.out = static_cast<__nv_bfloat16*>(a.out);
  p.lse = static_cast<float*>(a.lse);
  p.parts = static_cast<float*>(a.workspace);
  p.q_batch = a.q_batch_stride;
  p.q_head = a.q_head_stride;
  p.table_stride = a.table_stride;
  p.batch = a.batch;
  p.heads = a.heads;
  p.kv_heads = c.kv_heads;
  p.group_heads = group_heads;
  p.head_blocks = head_blocks;
  p.pages = c.pages;
  p.page = c.page;
  p.max_pages = a.max_pages;
  p.box = kKv4Tile;                     // positions a copy fetches: the largest power of two that pages and tiles share
  while (c.page % p.box) p.box /= 2;
  p.box_shift = __builtin_ctz(p.box);
  p.page_shift = (c.page & (c.page - 1)) == 0 ? __builtin_ctz(c.page) : -1;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  CUtensorMap map_k, map_v;
  const uint64_t lines = static_cast<uint64_t>(c.pages) * c.kv_heads * c.page * (c.head_dim / 2) / 128;
  const uint32_t box_lines = p.box * (c.head_dim / 2) / 128;
  if (int rc = make_tensor_map_3d(&map_k, c.k_codes, 2, 64, lines, 1, 128, 128 * lines, 64, box_lines, 1, 128)) return rc;
  if (int rc = make_tensor_map_3d(&map_v, c.v_codes, 2, 64, lines, 1, 128, 128 * lines, 64, box_lines, 1, 128)) return rc;
  const int blocks = kv4_blocks(sm_count, block_heads);
  p.cuts_by_row = static_cast<long long>(a.batch) * c.kv_heads * head_blocks <= blocks ? 1 : 0;
  p.cuts = reinterpret_cast<int4*>(p.parts + static_cast<size_t>(blocks) * 2 * block_heads * (c.head_dim + 2));
  cudaStream_t stream = static_cast<cudaStream_t>(stream_handle);
  const int groups = c.head_dim / c.group;
#define TRINITY_KV4(D, NG) \
  return block_heads == 8 ? launch_kv4_attend<D, NG, 1>(p, map_k, map_v, blocks, stream) \
                          : launch_kv4_attend<D, NG, 2>(p, map_k, map_v, blocks, stream);
  if (c.head_dim == 128) {
    if (groups == 1) TRINITY_KV4(128, 1)
    if (groups == 2) TRINITY_KV4(128, 2)
    TRINITY_KV4(128, 4)
  }
  if (groups == 1) TRINITY_KV4(64, 1)
  TRINITY_KV4(64, 2)
#undef TRINITY_KV4
}
