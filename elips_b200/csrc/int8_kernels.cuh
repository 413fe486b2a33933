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

// The integer nearest to x / s by a 64-bit division. A quotient of two fp32
// numbers that is no tie is at least 2^-25 (relative) away from one, because
// x - (q + 1/2) s is a multiple of half an ulp of s: the division decides.
__device__ __noinline__ int row_code_exact(float x, float s) {
    return static_cast<int>(rint(static_cast<double>(x) / static_cast<double>(s)));
}

// Adding 1.5 * 2^23 to a number below 2^22 rounds it to the nearest integer,
// ties to even, and leaves that integer in the low bits of the sum.
constexpr float kRound = 12582912.0f;

// V codes of one row, packed. inv is 1/s to half an ulp, so x * inv is within
// 2^-17 of the quotient (|x / s| < 127.5): its nearest integer is the code
// unless it lies that near to a half, and only then the exact division runs
// (for values that are half steps by their making, and else 1 in 2^15).
template <int V>
__device__ __forceinline__ void row_codes(const float (&x)[V], float s, float inv, uint32_t (&w)[(V + 3) / 4]) {
    uint32_t m[V];
    float off = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float r = fmaf(x[i], inv, kRound);
        off = fmaxf(off, fabsf(fmaf(x[i], inv, kRound - r)));
        m[i] = __float_as_uint(r);
    }
    if (off > 0.5f - 0x1p-16f) {
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = static_cast<uint32_t>(row_code_exact(x[i], s));
    }
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        uint32_t lo = m[i], hi = 0;
        if constexpr (V >= 2) lo = __byte_perm(m[i], m[i + 1], 0x0040);
        if constexpr (V >= 4) hi = __byte_perm(m[i + 2], m[i + 3], 0x0040);
        w[i / 4] = __byte_perm(lo, hi, 0x5410);
    }
}

// Division of numbers below 2^31 by a fixed divisor: a multiply, an add and a
// shift (mul = floor(2^32 (2^shift - d) / d) + 1 with 2^shift >= d).
struct FastDiv {
    uint32_t d = 1, mul = 1, shift = 0;
    __host__ __device__ FastDiv() {}
    __host__ explicit FastDiv(uint32_t divisor) : d(divisor) {
        while (shift < 31 && (1u << shift) < d) ++shift;
        mul = static_cast<uint32_t>((((uint64_t{1} << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// V elements as fp32, from one access of V * sizeof(T) bytes.
template <class T, int V>
__device__ __forceinline__ void load_row(const T* src, float (&x)[V]) {
    if constexpr (V == 1) {
        x[0] = to_f32(src[0]);
    } else if constexpr (sizeof(T) * V == 16) {
        const uint4 raw = *reinterpret_cast<const uint4*>(src);
        const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = to_f32(e[i]);
    } else {
        static_assert(V == 1, "rows are read 16 bytes or one element at a time");
    }
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
    uint32_t t, heads, d;
    uint32_t t0, groups;  // this launch: rows of t0 on, (t, part, head) groups of them
    FastDiv per_t, by_heads, page;
    int64_t num_slots;
    int dup;  // a slot may come twice: kDupNone, kDupScan or kDupClaim
};

enum DupCheck : int { kDupNone = 0, kDupScan = 1, kDupClaim = 2 };

__device__ __forceinline__ int64_t slot_of(const QuantParams& p, uint32_t t) {
    if (p.slots == nullptr) return t;
    return p.slots64 ? static_cast<const int64_t*>(p.slots)[t] : static_cast<const int32_t*>(p.slots)[t];
}

__device__ __forceinline__ float* scale_at(const QuantParams& p, uint32_t part, uint32_t slot, uint32_t head) {
    const uint32_t pg = p.page.div(slot), at = slot - pg * p.page.d;
    return p.scales + part * p.scale_part + pg * p.scale_page + at * p.scale_row + head * p.scale_head;
}

// The part, row and head of group g of this launch.
__device__ __forceinline__ void group_at(const QuantParams& p, uint32_t g, uint32_t& t, uint32_t& part, uint32_t& head) {
    const uint32_t i = p.per_t.div(g), r = g - i * p.per_t.d;
    t = p.t0 + i;
    part = p.by_heads.div(r);
    head = r - part * p.heads;
}

// A slot given twice in one call keeps the last of its rows. Up to
// kDupScanRows rows each row looks for its slot among the later ones (which
// stay in L1). Longer calls settle it in the slot's own scale words before any
// row is written: one launch zeroes them, the next leaves the largest claim
// 0x80000001 + t there, and the row whose claim stands writes codes and scale.
// A scale is never negative, so no scale written in between is taken for a
// claim; what the words held before does not matter.
constexpr uint32_t kDupScanRows = 256;

__device__ __forceinline__ uint32_t claim_of(uint32_t t) { return 0x80000001u + t; }

static __global__ void __launch_bounds__(256) cache_claim_kernel(const __grid_constant__ QuantParams p, int clear) {
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= p.groups) return;
    uint32_t t, part, head;
    group_at(p, g, t, part, head);
    const int64_t s = slot_of(p, t);
    if (s < 0 || s >= p.num_slots) return;
    uint32_t* w = reinterpret_cast<uint32_t*>(scale_at(p, part, static_cast<uint32_t>(s), head));
    if (clear) *w = 0u;
    else atomicMax(w, claim_of(t));
}

// G threads per row (8, a warp, or the whole block), each holding NV accesses
// of V values in registers: one read of the row, the largest magnitude over
// its threads, the codes. Rows wider than G * NV * V (only where G is the
// block) are read a second time for what did not fit.
template <class T, int V, int G, int NV>
static __global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantParams p) {
    __shared__ uint32_t block_max[8];
    constexpr uint32_t kPer = 256 / G;  // rows per block
    constexpr uint32_t kHeld = G * NV * V;
    const uint32_t gl = threadIdx.x % G;
    const uint32_t g = blockIdx.x * kPer + threadIdx.x / G;
    uint32_t t = 0, part = 0, head = 0;
    int64_t s = -1;
    if (g < p.groups) {
        group_at(p, g, t, part, head);
        s = slot_of(p, t);
    }
    // Rows of one warp stay together to the end: they share its votes.
    bool keep = s >= 0 && s < p.num_slots;
    const uint32_t slot = keep ? static_cast<uint32_t>(s) : 0u;
    float* const scale = scale_at(p, part, slot, head);
    const T* const x = static_cast<const T*>(p.x[part]) + t * p.x_stride_t[part] + head * p.x_stride_h[part];

    float v[NV][V];
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t e = (j * G + gl) * V;
        if (e < p.d && keep) {
            load_row<T, V>(x + e, v[j]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) v[j][i] = 0.0f;
        }
    }
    if (p.dup == kDupClaim) {
        // The row's own claim stands until it stores its scale below.
        if (keep) keep = *reinterpret_cast<volatile uint32_t*>(scale) == claim_of(t);
    } else if (p.dup == kDupScan && keep) {
        for (uint32_t i = t + 1u + gl; i < p.t; i += G) keep = keep && slot_of(p, i) != s;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) amax = max(amax, __float_as_uint(v[j][i]) & 0x7FFFFFFFu);
    if constexpr (G == 256) {
        for (uint32_t e = kHeld + gl * V; e < p.d; e += G * V) {
            float u[V];
            load_row<T, V>(x + e, u);
#pragma unroll
            for (int i = 0; i < V; ++i) amax = max(amax, __float_as_uint(u[i]) & 0x7FFFFFFFu);
        }
        if (__syncthreads_or(!keep)) return;
        amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        if ((threadIdx.x & 31u) == 0) block_max[threadIdx.x >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max(amax, block_max[i]);
    } else {
        const uint32_t kept = __ballot_sync(0xFFFFFFFFu, keep);
        if constexpr (G == 32) {
            keep = kept == 0xFFFFFFFFu;
            amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        } else {
            constexpr uint32_t kPeers = (1u << (G % 32)) - 1u;
            keep = ((kept >> (threadIdx.x & 31u & ~(G - 1u))) & kPeers) == kPeers;
#pragma unroll
            for (int o = G / 2; o > 0; o /= 2) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
        }
        if (!keep) return;
    }
    const float sc = row_scale(amax), inv = row_inverse(sc);
    const uint32_t pg = p.page.div(slot), at = slot - pg * p.page.d;
    int8_t* const out = p.codes + part * p.code_part + pg * p.code_page + at * p.code_row + head * p.code_head;
    auto put = [&](uint32_t e, const float (&u)[V]) {
        uint32_t w[(V + 3) / 4] = {};
        if (inv != 0.0f) row_codes<V>(u, sc, inv, w);
        if constexpr (V == 8) *reinterpret_cast<uint2*>(out + e) = make_uint2(w[0], w[V / 4 - 1]);
        else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(out + e) = w[0];
        else out[e] = static_cast<int8_t>(w[0]);
    };
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t e = (j * G + gl) * V;
        if (e < p.d) put(e, v[j]);
    }
    if constexpr (G == 256) {
        for (uint32_t e = kHeld + gl * V; e < p.d; e += G * V) {
            float u[V];
            load_row<T, V>(x + e, u);
            put(e, u);
        }
    }
    if (gl == 0) *scale = sc;
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
    uint32_t sequences, table_width, pages;
    uint32_t total, rows;                           // output rows, and those of one block
    FastDiv page, per_row, per_group, by_heads;     // accesses of V codes per output row and per (part, head)
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
    const uint32_t col = p.page.div(pos);
    if (col >= p.table_width) return kRowNoPage;
    const int64_t at = static_cast<int64_t>(lo) * p.table_stride + col;
    const int64_t pg = p.table64 ? static_cast<const int64_t*>(p.table)[at] : static_cast<const int32_t*>(p.table)[at];
    if (pg < 0 || pg >= static_cast<int64_t>(p.pages)) return kRowNoPage;
    return pg * p.page.d + (pos - col * p.page.d);
}

// int8 -> fp32 without the conversion unit: the byte with its sign bit turned
// (0 .. 255) in the low bits of 2^23 is 2^23 + byte, exactly.
__device__ __forceinline__ float code_f32(uint32_t turned, uint32_t byte) {
    return __uint_as_float(__byte_perm(turned, 0x4B000000u, 0x7440u | byte)) - 8388736.0f;  // 2^23 + 128
}

constexpr uint32_t kReadRows = 64;  // most output rows per block
constexpr int kReadBatch = 4;       // accesses a thread has under way

// A block reads `rows` output rows: first their slots, one thread each, then
// the codes, V at a time (16 bytes of output where everything is aligned so
// far), neighbouring threads on neighbouring codes of a row. One pass, bound
// by the bytes: 1 + sizeof(T) and 4 / dim per value.
template <class T, int V>
static __global__ void __launch_bounds__(256) cache_read_kernel(const __grid_constant__ ReadParams p) {
    __shared__ int64_t code_at[kReadRows], scale_at[kReadRows];
    const uint32_t t0 = blockIdx.x * p.rows, rows = min(p.rows, p.total - t0);
    if (threadIdx.x < rows) {
        const int64_t s = read_slot(p, t0 + threadIdx.x);
        int64_t code = s, scale = s;
        if (s >= 0) {
            const uint32_t pg = p.page.div(static_cast<uint32_t>(s)), at = static_cast<uint32_t>(s) - pg * p.page.d;
            code = pg * p.code_page + at * p.code_row;
            scale = pg * p.scale_page + at * p.scale_row;
        }
        code_at[threadIdx.x] = code;
        scale_at[threadIdx.x] = s < 0 ? s : scale;
    }
    __syncthreads();
    const uint32_t items = rows * p.per_row.d;
    for (uint32_t i0 = threadIdx.x; i0 < items; i0 += 256u * kReadBatch) {
        // The loads of a batch are issued before the first of its stores.
        uint32_t w[kReadBatch][(V + 3) / 4];
        float sc[kReadBatch];
        T* out[kReadBatch];
#pragma unroll
        for (int b = 0; b < kReadBatch; ++b) {
            const uint32_t i = i0 + 256u * b;
            out[b] = nullptr;
            if (i >= items) continue;
            const uint32_t row = p.per_row.div(i), r = i - row * p.per_row.d;
            const uint32_t group = p.per_group.div(r), e = (r - group * p.per_group.d) * V;
            const uint32_t part = p.by_heads.div(group), head = group - part * p.by_heads.d;
            const int64_t code = code_at[row];
            if (code == kRowBehind && !p.zero_behind) continue;
            out[b] = static_cast<T*>(p.out[part]) + (t0 + row) * p.out_stride_t[part] + head * p.out_stride_h[part] + e;
            sc[b] = 0.0f;
#pragma unroll
            for (int j = 0; j < (V + 3) / 4; ++j) w[b][j] = 0;
            if (code < 0) continue;
            const int8_t* q = p.codes + code + part * p.code_part + head * p.code_head + e;
            if constexpr (V == 8) {
                const uint2 u = __ldg(reinterpret_cast<const uint2*>(q));
                w[b][0] = u.x, w[b][V / 4 - 1] = u.y;
            } else if constexpr (V == 4) {
                w[b][0] = __ldg(reinterpret_cast<const uint32_t*>(q));
            } else if constexpr (V == 2) {
                w[b][0] = __ldg(reinterpret_cast<const uint16_t*>(q));
            } else {
                w[b][0] = static_cast<uint8_t>(__ldg(q));
            }
            sc[b] = __ldg(p.scales + scale_at[row] + part * p.scale_part + head * p.scale_head);
        }
#pragma unroll
        for (int b = 0; b < kReadBatch; ++b) {
            if (out[b] == nullptr) continue;
            alignas(16) T v[V];
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = from_f32<T>(code_f32(w[b][j / 4] ^ 0x80808080u, j % 4) * sc[b]);
            if constexpr (sizeof(T) * V == 16) *reinterpret_cast<uint4*>(out[b]) = *reinterpret_cast<const uint4*>(v);
            else if constexpr (sizeof(T) * V == 8) *reinterpret_cast<uint2*>(out[b]) = *reinterpret_cast<const uint2*>(v);
            else if constexpr (sizeof(T) * V == 4) *reinterpret_cast<uint32_t*>(out[b]) = *reinterpret_cast<const uint32_t*>(v);
            else *out[b] = v[0];
        }
    }
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
