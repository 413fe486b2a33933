// Kernels of the 8-bit row operators: rows quantised to int8 with one fp32
// scale each, in place or into the pages of a cache, the pages read back, and
// the int8 matrix product with a scale per row and channel.
//
// One format throughout. A row x[0..d) is held as codes q and a scale s:
//   a = max |x_j|,  s = fl(a / 127) in fp32,  q_j = the integer nearest to the
//   real quotient x_j / s, ties to even, so |q_j| <= 127 and |x_j - s q_j| <=
//   s/2 up to the rounding of s.
// s is at most the largest number whose 127-fold is finite, so a finite row
// reads back finite. Rows whose s would be below the smallest normal number (a < 127 * 2^-126)
// are held as s = 0 with codes 0. A row with an infinity or a NaN has a scale
// that is not finite (inf or NaN) and codes 0: it reads back as NaN and never
// touches another row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace eb {

constexpr float kMinScale = 0x1p-126f;
constexpr float kMaxScale = 0x1.0204060000000p+121f;  // the largest s with 127 s finite

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// The scale of a row whose largest magnitude has the bits `amax` (of an fp32
// number without its sign; larger bits are larger magnitudes, NaN above inf).
__device__ __forceinline__ float row_scale(uint32_t amax) {
    float s = __fdiv_rn(__uint_as_float(amax), 127.0f);
    if (amax < 0x7F800000u) s = fminf(s, kMaxScale);
    return s < kMinScale ? 0.0f : s;  // NaN stays NaN (and positive)
}

// 1/s, or 0 where the codes are 0 whatever the row holds.
__device__ __forceinline__ float row_inverse(float s) {
    return s > 0.0f && s < __int_as_float(0x7f800000) ? __frcp_rn(s) : 0.0f;
}

// The integer nearest to x / s. t = x * inv is within 2^-16 of the quotient
// (|t| <= 127.5, inv is 1/s to half an ulp), so rint(t) is the answer unless t
// lies that near to a half; only there the quotient is taken in 64 bits, where
// its distance from a half decides exactly (x - (q + 1/2) s is a multiple of
// ulp(s)/2, so a quotient that is no tie is at least 2^-25 relative away).
__device__ __forceinline__ int row_code(float x, float s, float inv) {
    if (inv == 0.0f) return 0;
    const float t = x * inv;
    const float q = rintf(t);
    if (fabsf(t - q) > 0.5f - 0x1p-15f) return static_cast<int>(rint(static_cast<double>(x) / static_cast<double>(s)));
    return static_cast<int>(q);
}

// Where rows come from and where their codes go: row (part, t, head) of the
// call is `d` values at x[part] + t * stride_t + head * stride_h, and slot s
// of a cache is position s % page of page s / page. A plain quantisation has
// one part, one head, pages of one row and no slot list.
struct QuantParams {
    const void* x[2];
    int64_t x_stride_t[2], x_stride_h[2];  // elements
    int8_t* codes;
    float* scales;
    int64_t code_part, code_page, code_row, code_head;      // bytes
    int64_t scale_part, scale_page, scale_row, scale_head;  // elements
    const void* slots;  // [t], int32 or int64; null: row t goes to slot t
    int slots64;
    uint32_t t, parts, heads, d, page;
    int64_t num_slots;
};

__device__ __forceinline__ int64_t slot_of(const QuantParams& p, uint32_t t) {
    if (p.slots == nullptr) return t;
    return p.slots64 ? static_cast<const int64_t*>(p.slots)[t] : static_cast<const int32_t*>(p.slots)[t];
}

__device__ __forceinline__ float* scale_at(const QuantParams& p, uint32_t part, uint32_t slot, uint32_t head) {
    return p.scales + part * p.scale_part + static_cast<int64_t>(slot / p.page) * p.scale_page +
           static_cast<int64_t>(slot % p.page) * p.scale_row + head * p.scale_head;
}

// A slot given twice in one call keeps the last of its rows. Who writes is
// settled in the slot's own scale words before any row is written: one launch
// zeroes them, the next leaves the largest claim 0x80000001 + t there, and the
// row whose claim stands writes codes and scale. A scale is never negative, so
// no scale written in between is taken for a claim.
__device__ __forceinline__ uint32_t claim_of(uint32_t t) { return 0x80000001u + t; }

static __global__ void __launch_bounds__(256) cache_claim_kernel(const QuantParams p, int clear) {
    const uint64_t per_t = static_cast<uint64_t>(p.parts) * p.heads;
    const uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256u + threadIdx.x;
    if (i >= per_t * p.t) return;
    const uint32_t t = static_cast<uint32_t>(i / per_t), r = static_cast<uint32_t>(i % per_t);
    const int64_t s = slot_of(p, t);
    if (s < 0 || s >= p.num_slots) return;
    uint32_t* w = reinterpret_cast<uint32_t*>(scale_at(p, r / p.heads, static_cast<uint32_t>(s), r % p.heads));
    if (clear) *w = 0u;
    else atomicMax(w, claim_of(t));
}

// One warp per row: the largest magnitude, then the codes from a second read.
template <class T>
static __global__ void __launch_bounds__(256) quantize_rows_kernel(const QuantParams p, int claimed) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * 8u + (threadIdx.x >> 5);
    const uint64_t per_t = static_cast<uint64_t>(p.parts) * p.heads;
    if (row >= per_t * p.t) return;
    const uint32_t t = static_cast<uint32_t>(row / per_t), r = static_cast<uint32_t>(row % per_t);
    const uint32_t part = r / p.heads, head = r % p.heads;
    const int64_t s = slot_of(p, t);
    if (s < 0 || s >= p.num_slots) return;
    const uint32_t slot = static_cast<uint32_t>(s);
    float* const scale = scale_at(p, part, slot, head);
    if (claimed) {
        // Read by one lane, before any lane can write: the row's own claim
        // stands until lane 0 stores the scale below.
        uint32_t w = 0;
        if (lane == 0) w = *reinterpret_cast<volatile uint32_t*>(scale);
        if (__shfl_sync(0xffffffffu, w, 0) != claim_of(t)) return;
    }
    const T* x = static_cast<const T*>(p.x[part]) + t * p.x_stride_t[part] + head * p.x_stride_h[part];
    uint32_t amax = 0;
    for (uint32_t j = lane; j < p.d; j += 32) amax = max(amax, __float_as_uint(to_f32(x[j])) & 0x7FFFFFFFu);
    amax = __reduce_max_sync(0xffffffffu, amax);
    const float sc = row_scale(amax), inv = row_inverse(sc);
    int8_t* out = p.codes + part * p.code_part + static_cast<int64_t>(slot / p.page) * p.code_page +
                  static_cast<int64_t>(slot % p.page) * p.code_row + head * p.code_head;
    for (uint32_t j = lane; j < p.d; j += 32) out[j] = static_cast<int8_t>(row_code(to_f32(x[j]), sc, inv));
    if (lane == 0) *scale = sc;
}

// Reading pages back into packed rows. Sequence b owns the output rows
// offsets[b] .. offsets[b + 1]; position i of it is slot page_table[b][i /
// page] * page + i % page.
struct ReadParams {
    void* out[2];
    int64_t out_stride_t[2], out_stride_h[2];  // elements
    const int8_t* codes;
    const float* scales;
    int64_t code_part, code_page, code_row, code_head;
    int64_t scale_part, scale_page, scale_row, scale_head;
    const void* table;
    const void* offsets;
    int table64, offsets64;
    int64_t table_stride;
    uint32_t sequences, table_width, pages, page, parts, heads, d;
    uint32_t total;
    int zero_behind;  // rows past the last sequence: zeroed (a fresh output) or left as they are
};

__device__ __forceinline__ int64_t offset_of(const ReadParams& p, uint32_t b) {
    return p.offsets64 ? static_cast<const int64_t*>(p.offsets)[b] : static_cast<const int32_t*>(p.offsets)[b];
}

constexpr int64_t kRowBehind = -2;  // past the last sequence
constexpr int64_t kRowNoPage = -1;  // its page is not in the table or not a page of the cache

// The slot that output row t is read from. Whatever the table and the offsets
// hold, the answer is inside the cache or one of the two constants.
__device__ __forceinline__ int64_t read_slot(const ReadParams& p, uint32_t t) {
    uint32_t lo = 0, hi = p.sequences;  // the first b in [0, sequences] with offsets[b] > t, less one
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (offset_of(p, mid + 1u) > static_cast<int64_t>(t)) hi = mid;
        else lo = mid + 1u;
    }
    if (lo >= p.sequences) return kRowBehind;
    const int64_t i = static_cast<int64_t>(t) - offset_of(p, lo);
    if (i < 0) return kRowNoPage;
    const uint32_t pos = static_cast<uint32_t>(i);  // i <= t
    const uint32_t col = pos / p.page;
    if (col >= p.table_width) return kRowNoPage;
    const int64_t at = static_cast<int64_t>(lo) * p.table_stride + col;
    const int64_t pg = p.table64 ? static_cast<const int64_t*>(p.table)[at] : static_cast<const int32_t*>(p.table)[at];
    if (pg < 0 || pg >= static_cast<int64_t>(p.pages)) return kRowNoPage;
    return pg * p.page + pos % p.page;
}

template <class T>
static __global__ void __launch_bounds__(256) cache_read_kernel(const ReadParams p) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t row = static_cast<uint64_t>(blockIdx.x) * 8u + (threadIdx.x >> 5);
    const uint64_t per_t = static_cast<uint64_t>(p.parts) * p.heads;
    if (row >= per_t * p.total) return;
    const uint32_t t = static_cast<uint32_t>(row / per_t), r = static_cast<uint32_t>(row % per_t);
    const uint32_t part = r / p.heads, head = r % p.heads;
    const int64_t s = read_slot(p, t);
    if (s == kRowBehind && !p.zero_behind) return;
    T* out = static_cast<T*>(p.out[part]) + t * p.out_stride_t[part] + head * p.out_stride_h[part];
    if (s < 0) {
        for (uint32_t j = lane; j < p.d; j += 32) out[j] = from_f32<T>(0.0f);
        return;
    }
    const int64_t pg = s / p.page, at = s % p.page;
    const int8_t* q = p.codes + part * p.code_part + pg * p.code_page + at * p.code_row + head * p.code_head;
    const float sc = p.scales[part * p.scale_part + pg * p.scale_page + at * p.scale_row + head * p.scale_head];
    for (uint32_t j = lane; j < p.d; j += 32) out[j] = from_f32<T>(static_cast<float>(q[j]) * sc);
}

// The int8 product's arguments (int8_gemm.cuh).
struct GemmParams {
    const int8_t* a;
    const int8_t* b;
    int64_t a_pitch, b_pitch;
    const float* a_scales;
    const float* b_scales;
    const void* bias;
    int bias_type;  // ELIPS_B200_PRECISION_*
    void* out;
    int64_t out_pitch;  // elements
    uint32_t m, n, k;
};

__device__ __forceinline__ float bias_at(const void* bias, int type, uint32_t n) {
    if (type == 1) return __half2float(static_cast<const __half*>(bias)[n]);
    if (type == 4) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
    return static_cast<const float*>(bias)[n];
}

}  // namespace eb
