// Kernels of the 8-bit row operators: rows quantised to int8 with one fp32
// scale each, in place or into the pages of a cache, the pages read back, and
// the int8 matrix product with a scale per row and channel.
//
// One format throughout. A row x[0..d) is held as codes q and a scale s:
//   a = max |x_j|,  s = fl(a / 127) in fp32,  q_j = the integer nearest to the
//   real quotient x_j / s, ties to even, so |q_j| <= 127 and |x_j - s q_j| <=
//   s/2 up to the rounding of s.
// s is at most the largest number whose 127-fold is finite, so a finite row
// reads back finite. Rows whose s would be below the smallest normal number (a
// < 127 * 2^-126) are held as s = 0 with codes 0. A row with an infinity or a
// NaN has a scale that is not finite (inf or NaN) and codes 0: it reads back
// as NaN and never touches another row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

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

// Adding 1.5 * 2^23 to a number below 2^22 rounds it to the nearest integer,
// ties to even, and leaves that integer in the low bits of the sum.
constexpr float kRound = 12582912.0f;

// r = kRound + q for a q next to the code of x: one step towards x / s if that
// is nearer, or as near and even. The remainder x - q s is exact: both are
// multiples of ulp(s) where |x| >= s, and x itself or (by Sterbenz) its
// difference from s where q is 0 or 1; where a q of 1 is one too many, the
// remainder is past -s/2 and rounds to no less, which still gives 0.
__device__ __forceinline__ float nearest_step(float r, float x, float s) {
    const float q = r - kRound;
    const float rem = fmaf(-q, s, x), twice = fabsf(rem + rem);
    const bool odd = (__float_as_uint(r) & 1u) != 0u;
    return twice > s || (twice == s && odd) ? r + copysignf(1.0f, rem) : r;
}

// What the codes of a row are made with: code = the integer nearest to x * inv,
// looked at once more near halves where `careful`.
struct RowScale {
    float s, inv;
    bool careful;
};

// inv is 0 where the codes are 0 whatever the row holds.
//
// 16-bit rows need no second look. With x of at most 11 bits and a the row's
// largest magnitude, 127 x / a is a half (k + 1/2) exactly or at least 1 / (254
// * 2^11) > 2^-19 of itself away from one, since 254 x - (2k + 1) a is a whole
// multiple of x's last bit. So only the exact halves are in doubt, and they
// are so because the stored s is not a / 127: x / s lies below the half where s
// was rounded up and above it where s was rounded down. An inverse a few ulps
// to that side of 127 / a (1/s rounded is within 2 ulps of it; 4 more make at
// most 2^-20) gives every code right. Where s is a / 127 exactly, a half is a
// tie, which 1/s keeps only if it is exact itself (in bf16 it always is);
// those few fp16 rows, and fp32 rows, take the second look.
template <class T>
__device__ __forceinline__ RowScale make_scale(uint32_t amax) {
    RowScale r;
    r.s = row_scale(amax);
    r.inv = r.s > 0.0f && r.s < __int_as_float(0x7f800000) ? __frcp_rn(r.s) : 0.0f;
    r.careful = true;
    if constexpr (sizeof(T) == 2) {
        const float over = fmaf(127.0f, r.s, -__uint_as_float(amax));  // the sign of s - a / 127
        r.careful = over == 0.0f && fmaf(r.inv, r.s, -1.0f) != 0.0f;
        if (over != 0.0f && r.inv != 0.0f) r.inv = __int_as_float(__float_as_int(r.inv) + (over > 0.0f ? -4 : 4));
    }
    return r;
}

// V codes of one row, packed. Near halves: inv is 1/s to half an ulp, so x *
// inv is within 2^-17 of the quotient (|x / s| < 127.5), and its nearest
// integer is the code unless it lies that near to a half.
template <int V>
__device__ __forceinline__ void row_codes(const float (&x)[V], const RowScale& rs, uint32_t (&w)[(V + 3) / 4]) {
    uint32_t m[V];
    if (!rs.careful) {
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = __float_as_uint(fmaf(x[i], rs.inv, kRound));
    } else {
        float r[V];
        float off = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            r[i] = fmaf(x[i], rs.inv, kRound);
            off = fmaxf(off, fabsf(fmaf(x[i], rs.inv, kRound - r[i])));
        }
        if (off > 0.5f - 0x1p-16f) {
#pragma unroll
            for (int i = 0; i < V; ++i) r[i] = nearest_step(r[i], x[i], rs.s);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) m[i] = __float_as_uint(r[i]);
    }
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        uint32_t lo = m[i], hi = 0;
        if constexpr (V >= 2) lo = __byte_perm(m[i], m[i + 1], 0x0040);
        if constexpr (V >= 4) hi = __byte_perm(m[i + 2], m[i + 3], 0x0040);
        w[i / 4] = __byte_perm(lo, hi, 0x5410);
    }
}

// One access to a row: 16 bytes of it, or one value where rows start anywhere.
template <class T, int V>
struct Access {
    uint4 raw;
    __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(const T* src) { raw = *reinterpret_cast<const uint4*>(src); }
    __device__ __forceinline__ void values(float (&x)[V]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                x[i] = __uint_as_float(w[i]);
            } else {
                const float2 f = pair(w[i]);
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            }
        }
    }
    static __device__ __forceinline__ float2 pair(uint32_t w) {
        if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
        else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
    // Zero for the elements outside [first, end).
    __device__ __forceinline__ void keep_only(int first, int end) {
        uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                if (i < first || i >= end) w[i] = 0;
            } else {
                if (2 * i < first || 2 * i >= end) w[i] &= 0xFFFF0000u;
                if (2 * i + 1 < first || 2 * i + 1 >= end) w[i] &= 0x0000FFFFu;
            }
        }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
    // The larger of `top` (a magnitude, NaN above all) and those held.
    __device__ __forceinline__ uint32_t top(uint32_t top) const {
        if constexpr (sizeof(T) == 4) {
            return max(max(max(raw.x & 0x7FFFFFFFu, raw.y & 0x7FFFFFFFu), max(raw.z & 0x7FFFFFFFu, raw.w & 0x7FFFFFFFu)), top);
        } else {
            // 16-bit magnitudes compare as whole numbers, two at a time
            const uint32_t m = __vmaxu2(__vmaxu2(raw.x & 0x7FFF7FFFu, raw.y & 0x7FFF7FFFu),
                                        __vmaxu2(raw.z & 0x7FFF7FFFu, raw.w & 0x7FFF7FFFu));
            return __vmaxu2(m, top);
        }
    }
    static __device__ __forceinline__ uint32_t bits32(uint32_t top) {
        if constexpr (sizeof(T) == 4) return top;
        const float2 f = pair(top);
        return max(__float_as_uint(f.x), __float_as_uint(f.y));
    }
};

template <class T>
struct Access<T, 1> {
    T raw;
    __device__ __forceinline__ void zero() { raw = from_f32<T>(0.0f); }
    __device__ __forceinline__ void load(const T* src) { raw = *src; }
    __device__ __forceinline__ void values(float (&x)[1]) const { x[0] = to_f32(raw); }
    __device__ __forceinline__ uint32_t top(uint32_t top) const { return max(top, __float_as_uint(to_f32(raw)) & 0x7FFFFFFFu); }
    static __device__ __forceinline__ uint32_t bits32(uint32_t top) { return top; }
};

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

// Programmatic dependent launch: a kernel may start while the one before it in
// the stream ends. Every kernel here waits with await_previous() until that one
// is complete and its writes are seen before it reads or writes global memory,
// and only then lets the next one start (let_next_start), so whatever a kernel
// finds running has itself seen the end of all before it. The one exception:
// a cache write after its claims reads rows and slots first, which nothing in
// between writes. Because a kernel may start before its inputs are written, none
// of them is read through the non-coherent path (__ldg), which is for data that
// stays as it is for as long as the kernel runs.
__device__ __forceinline__ void await_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Coherent loads that stay behind await_previous (volatile, as that is) and that
// the compiler may otherwise place as it does __ldg, before stores that they do
// not depend on among others: as plain loads, which may not pass a store, the
// batches of cache_read_kernel hold more registers and 131,072 rows of 2 x 8 x
// 128 bf16 take 156 us in place of 128.
__device__ __forceinline__ uint4 ld16(const void* at) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
    return v;
}
// Zero where `there` is negative: predicated, so that a batch of them is under
// way at once, on the value that a row's place is.
__device__ __forceinline__ uint2 ld8_if(const void* at, int64_t there = 0) {
    uint2 v;
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ge.s64 p, %3, 0;\n\tmov.u32 %0, 0;\n\tmov.u32 %1, 0;\n\t"
        "@p ld.global.v2.u32 {%0, %1}, [%2];\n\t}"
        : "=&r"(v.x), "=&r"(v.y)
        : "l"(at), "l"(there));
    return v;
}
__device__ __forceinline__ uint32_t ld4_if(const void* at, int64_t there = 0) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.s64 p, %2, 0;\n\tmov.u32 %0, 0;\n\t@p ld.global.u32 %0, [%1];\n\t}"
                 : "=&r"(v)
                 : "l"(at), "l"(there));
    return v;
}
__device__ __forceinline__ uint32_t ld2_if(const void* at, int64_t there = 0) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.s64 p, %2, 0;\n\tmov.u32 %0, 0;\n\t@p ld.global.u16 %0, [%1];\n\t}"
                 : "=&r"(v)
                 : "l"(at), "l"(there));
    return v;
}
__device__ __forceinline__ uint32_t ld1_if(const void* at, int64_t there = 0) {
    uint32_t v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.s64 p, %2, 0;\n\tmov.u32 %0, 0;\n\t@p ld.global.u8 %0, [%1];\n\t}"
                 : "=&r"(v)
                 : "l"(at), "l"(there));
    return v;
}
__device__ __forceinline__ float ld_float_if(const float* at, int64_t there = 0) { return __uint_as_float(ld4_if(at, there)); }

// A slot given twice in one call keeps the last of its rows. Up to
// kDupScanRows rows each row looks for its slot among the later ones (which
// stay in L1; 256 rows of 2 x 8 x 128 take 3.7 us, 300 with claims 3.2 but one
// launch more). Longer calls settle it before any row is written: a launch of
// its own leaves the largest claim 0x80000001 + t in the slot's scale words,
// and the row whose claim stands writes codes and scale. A scale is never
// negative, so neither one that is written in between nor one that was there
// is taken for a claim; of whatever else the words held (memory that no write
// has reached), a number that could be a claim is one only if its row has this
// slot, and then it loses to a later row's like any other.
constexpr uint32_t kDupScanRows = 256;

__device__ __forceinline__ uint32_t claim_of(uint32_t t) { return 0x80000001u + t; }

static __global__ void __launch_bounds__(256) cache_claim_kernel(const __grid_constant__ QuantParams p) {
    await_previous();
    let_next_start();
    const uint32_t g = blockIdx.x * 256u + threadIdx.x;
    if (g >= p.groups) return;
    uint32_t t, part, head;
    group_at(p, g, t, part, head);
    const int64_t s = slot_of(p, t);
    if (s < 0 || s >= p.num_slots) return;
    uint32_t* const w = reinterpret_cast<uint32_t*>(scale_at(p, part, static_cast<uint32_t>(s), head));
    const uint32_t claim = claim_of(t);
    uint32_t old = atomicMax(w, claim);
    // Mostly done: the word held a scale or an earlier claim. Else a later
    // row's claim, which stands, or a number that is none, which does not.
    while (old > claim) {
        const uint32_t other = old - claim_of(0);  // the row that `old` would be the claim of
        if (other < p.t && slot_of(p, other) == s) return;
        if (atomicCAS(w, old, claim) == old) return;
        old = atomicMax(w, claim);  // another row's claim came first
    }
}

// Whether a row after t has the same slot, by the G threads of the row (each
// sees its own share) or, where they are few, by the whole warp for one after
// the other of its rows, those of one t (its heads and parts) at once. The
// loops have no early end, so that their loads do not wait for each other.
template <int G>
__device__ __forceinline__ bool again_later(const QuantParams& p, uint32_t t, uint32_t slot, bool wanted, uint32_t gl) {
    bool again = false;
    if (G >= 32 || p.t <= 4 * G) {
#pragma unroll 4
        for (uint32_t i = t + 1u + gl; i < p.t; i += G) again |= slot_of(p, i) == static_cast<int64_t>(slot);
    } else if constexpr (G < 32) {
        const uint32_t lane = threadIdx.x & 31u;
        uint32_t last_t = 0xFFFFFFFFu;
        bool last = false;
#pragma unroll 1
        for (uint32_t r = 0; r < 32u / G; ++r) {
            if (!__shfl_sync(0xFFFFFFFFu, wanted ? 1 : 0, r * G)) continue;
            const uint32_t t_r = __shfl_sync(0xFFFFFFFFu, t, r * G), slot_r = __shfl_sync(0xFFFFFFFFu, slot, r * G);
            if (t_r != last_t) {
                bool found = false;
#pragma unroll 4
                for (uint32_t i = t_r + 1u + lane; i < p.t; i += 32) found |= slot_of(p, i) == static_cast<int64_t>(slot_r);
                last = __any_sync(0xFFFFFFFFu, found);
                last_t = t_r;
            }
            if (lane / G == r) again = last;
        }
    }
    return again;
}

// G threads per row (4, 8, a warp, or the whole block), each holding NV
// accesses of V values in registers: one read of the row, the largest
// magnitude over its threads, the codes. Rows wider than G * NV * V (only
// where G is the block) are read a second time for what did not fit. CACHE:
// rows go to slots; else row t of one matrix is row t of another.
//
// Bound by the bytes (sizeof(T) + 1 per value) once a value costs few
// instructions: 16384 x 1024 bf16 takes 8.4 us (6.0 TB/s), 4096 x 4096 fp32
// 13.6 us (6.2 TB/s), 10,000 x 768 fp32 7.6 us (5.0 TB/s, the launch a fourth
// of it); with a check for halves in every 16-bit value and a block per wide
// row the first took 13.2.
//
// SHIFT: rows that start anywhere. The 16-byte accesses are those that hold the
// row (what they hold beside it is set to zero; an access with one byte of the
// row is in memory wherever that byte is), and the codes, which start `off`
// values into the first access, are shifted into place through shared memory,
// so that they are stored V at a time too. Codes start on V bytes. 10,000 x 767
// bf16: 7.7 us, value by value 11.3 (10,000 x 768: 4.9); 60,000 x 67: 5.9 and
// 11.1.
template <class T, int V, int G, int NV, bool CACHE, bool SHIFT>
static __global__ void __launch_bounds__(256) quantize_rows_kernel(const __grid_constant__ QuantParams p) {
    static_assert(!SHIFT || V > 1, "single values need no shift");
    using Word = typename std::conditional<V == 8, uint64_t, uint32_t>::type;  // V codes
    __shared__ uint32_t block_max[8];
    __shared__ Word words[SHIFT ? 256 * NV + 1 : 1];
    constexpr uint32_t kHeld = G * NV * V;
    if (!CACHE || p.dup != kDupClaim) await_previous();
    const uint32_t gl = threadIdx.x % G;
    const uint32_t g = blockIdx.x * (256 / G) + threadIdx.x / G;
    uint32_t t = p.t0 + g, part = 0, head = 0, slot = t;
    // Rows of one warp stay together to the end: they share its votes.
    bool keep = g < p.groups;
    const T* x = static_cast<const T*>(p.x[0]);
    int8_t* out = p.codes;
    float* scale = p.scales;
    if constexpr (CACHE) {
        int64_t s = -1;
        if (keep) {
            group_at(p, g, t, part, head);
            s = slot_of(p, t);
        }
        keep = s >= 0 && s < p.num_slots;
        slot = keep ? static_cast<uint32_t>(s) : 0u;
        x = static_cast<const T*>(part != 0u ? p.x[1] : p.x[0]) +
            t * (part != 0u ? p.x_stride_t[1] : p.x_stride_t[0]) + head * (part != 0u ? p.x_stride_h[1] : p.x_stride_h[0]);
        scale = scale_at(p, part, slot, head);
        const uint32_t pg = p.page.div(slot), at = slot - pg * p.page.d;
        out += part * p.code_part + pg * p.code_page + at * p.code_row + head * p.code_head;
    } else {
        x += t * p.x_stride_t[0];
        out += t * p.code_page;
        scale += t;
    }

    const uint32_t off = SHIFT ? static_cast<uint32_t>(reinterpret_cast<uintptr_t>(x) % 16u / sizeof(T)) : 0u;
    Access<T, V> v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t e = (j * G + gl) * V;  // from `off` values before the row
        if (e < off + p.d && keep) v[j].load(x - off + e);
        else v[j].zero();
    }
    if constexpr (SHIFT) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = (j * G + gl) * V, first = static_cast<int>(off) - e, end = static_cast<int>(off + p.d) - e;
            if (first > 0 || end < V) v[j].keep_only(first, end);
        }
    }
    if constexpr (CACHE) {
        if (p.dup == kDupClaim) {
            // The row's own claim stands until it stores its scale below.
            await_previous();
            if (keep) keep = *reinterpret_cast<volatile uint32_t*>(scale) == claim_of(t);
        } else if (p.dup == kDupScan) {
            // Every lane takes part, whatever its row: the search votes.
            const bool again = again_later<G>(p, t, slot, keep, gl);
            keep = keep && !again;
        }
    }
    let_next_start();
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) top = v[j].top(top);
    if constexpr (G == 256 && !SHIFT) {
        for (uint32_t e = kHeld + gl * V; e < p.d && keep; e += G * V) {
            Access<T, V> u;
            u.load(x + e);
            top = u.top(top);
        }
    }
    uint32_t amax = Access<T, V>::bits32(top);
    if constexpr (G == 256) {
        if (__syncthreads_or(!keep)) return;
        amax = __reduce_max_sync(0xFFFFFFFFu, amax);
        if ((threadIdx.x & 31u) == 0) block_max[threadIdx.x >> 5] = amax;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = max(amax, block_max[i]);
    } else if constexpr (G == 32) {
        if (!__all_sync(0xFFFFFFFFu, keep)) return;
        amax = __reduce_max_sync(0xFFFFFFFFu, amax);
    } else {
        constexpr uint32_t kPeers = (1u << (G % 32)) - 1u;
        const uint32_t kept = __ballot_sync(0xFFFFFFFFu, keep);
        keep = ((kept >> (threadIdx.x & 31u & ~(G - 1u))) & kPeers) == kPeers;
#pragma unroll
        for (int o = G / 2; o > 0; o /= 2) amax = max(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
        if (!keep) return;
    }
    const RowScale rs = make_scale<T>(amax);
    auto put = [&](uint32_t e, const Access<T, V>& u) {
        uint32_t w[(V + 3) / 4] = {};
        if (rs.inv != 0.0f) {
            float f[V];
            u.values(f);
            row_codes<V>(f, rs, w);
        }
        if constexpr (V == 8) *reinterpret_cast<uint2*>(out + e) = make_uint2(w[0], w[V / 4 - 1]);
        else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(out + e) = w[0];
        else out[e] = static_cast<int8_t>(w[0]);
    };
    if constexpr (SHIFT) {
        Word* const mine = words + threadIdx.x / G * (G * NV);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            uint32_t w[V / 4] = {};
            if (rs.inv != 0.0f) {
                float f[V];
                v[j].values(f);
                row_codes<V>(f, rs, w);
            }
            if constexpr (V == 8) mine[j * G + gl] = static_cast<uint64_t>(w[V / 4 - 1]) << 32 | w[0];
            else mine[j * G + gl] = w[0];
        }
        if constexpr (G == 256) __syncthreads();
        else __syncwarp();
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t i = j * G + gl, e = i * V;
            if (e >= p.d) continue;
            // The next word is not needed where off is 0, and where it is past
            // the row's accesses no code of the row is taken from it.
            Word w = mine[i] >> (8u * off);
            if (off != 0u) w |= mine[i + 1] << (8u * (V - off));
            if (e + V <= p.d) {
                *reinterpret_cast<Word*>(out + e) = w;
            } else {
                for (uint32_t b = 0; e + b < p.d; ++b) out[e + b] = static_cast<int8_t>(w >> (8u * b));
            }
        }
    } else if constexpr (V > 1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t e = (j * G + gl) * V;
            if (e < p.d) put(e, v[j]);
        }
    } else {  // single values: their codes together, stored one by one
        float f[NV];
        uint32_t w[(NV + 3) / 4] = {};
#pragma unroll
        for (int j = 0; j < NV; ++j) f[j] = to_f32(v[j].raw);
        if (rs.inv != 0.0f) row_codes<NV>(f, rs, w);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t e = j * G + gl;
            if (e < p.d) out[e] = static_cast<int8_t>(w[j / 4] >> (8 * (j % 4)));
        }
    }
    if constexpr (G == 256 && !SHIFT) {
        for (uint32_t e = kHeld + gl * V; e < p.d; e += G * V) {
            Access<T, V> u;
            u.load(x + e);
            put(e, u);
        }
    }
    if (gl == 0) *scale = rs.s;
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
    uint32_t nx, ny, per_row;                       // a block's threads; accesses of V codes per output row
    FastDiv page, per_group, by_heads;              // ... and per (part, head)
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
    uint32_t lo = 0, hi = p.sequences;  // the number of sequences that end at or before row t
    while (lo < hi) {
        const uint32_t mid = (lo + hi) / 2u;
        if (offset_of(p, mid + 1u) > static_cast<int64_t>(t)) hi = mid;
        else lo = mid + 1u;
    }
    if (lo >= p.sequences) return kRowBehind;
    const int64_t i = static_cast<int64_t>(t) - offset_of(p, lo);
    if (i < 0 || i > static_cast<int64_t>(t)) return kRowNoPage;  // in front of the first sequence, or a bad offset
    const uint32_t pos = static_cast<uint32_t>(i);
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

// V codes, zeros where there are none (`there` is negative).
template <int V>
__device__ __forceinline__ void load_codes(const int8_t* src, int64_t there, uint32_t (&w)[(V + 3) / 4]) {
    if constexpr (V == 8) {
        const uint2 u = ld8_if(src, there);
        w[0] = u.x;
        w[V / 4 - 1] = u.y;
    } else if constexpr (V == 4) {
        w[0] = ld4_if(src, there);
    } else if constexpr (V == 2) {
        w[0] = ld2_if(src, there);
    } else {
        w[0] = ld1_if(src, there);
    }
}

constexpr uint32_t kReadRows = 64;      // most output rows per block
constexpr uint32_t kReadThreads = 512;  // most threads per block
constexpr int kReadBatch = 8;           // accesses a thread has under way

// A block reads `rows` output rows (a share of their columns, where they are
// wide): first their slots, one thread each, then
// the codes, V at a time (16 bytes of output where everything is aligned so
// far). Its threads are `ny` times `nx`: neighbours on neighbouring codes of a
// row, and each stays on its column (part, head and place in the row) while
// it walks down the rows, so that an access costs two additions of offsets and
// not the divisions. One pass, bound by the bytes: 1 + sizeof(T) and 4 / dim
// per value. What decides is that the loads of a batch are predicated and not
// branched around, so that all eight are under way before the first store:
// 131,072 rows of 2 x 8 x 128 bf16 took 167 us with a branch per load, 132 us
// with four and 126 us with eight predicated loads (814 MB, 6.4 TB/s).
template <class T, int V>
static __global__ void __launch_bounds__(kReadThreads) cache_read_kernel(const __grid_constant__ ReadParams p) {
    __shared__ longlong2 row_at[kReadRows];  // where a row's codes and scales start; x below 0: it has none
    await_previous();
    let_next_start();
    const uint32_t t0 = blockIdx.x * p.rows, rows = min(p.rows, p.total - t0);
    if (threadIdx.x < rows) {
        const int64_t s = read_slot(p, t0 + threadIdx.x);
        longlong2 at = make_longlong2(s == kRowBehind && p.zero_behind ? kRowNoPage : s, 0);
        if (s >= 0) {
            const uint32_t pg = p.page.div(static_cast<uint32_t>(s)), i = static_cast<uint32_t>(s) - pg * p.page.d;
            at.x = pg * p.code_page + i * p.code_row;
            at.y = pg * p.scale_page + i * p.scale_row;
        }
        row_at[threadIdx.x] = at;
    }
    __syncthreads();
    const uint32_t ty = threadIdx.x / p.nx, tx = threadIdx.x - ty * p.nx;
    if (ty >= p.ny) return;
    for (uint32_t c = blockIdx.y * p.nx + tx; c < p.per_row; c += gridDim.y * p.nx) {
        const uint32_t group = p.per_group.div(c), e = (c - group * p.per_group.d) * V;
        const uint32_t part = p.by_heads.div(group), head = group - part * p.by_heads.d;
        const int8_t* const codes = p.codes + part * p.code_part + head * p.code_head + e;
        const float* const scales = p.scales + part * p.scale_part + head * p.scale_head;
        const int64_t step = part != 0u ? p.out_stride_t[1] : p.out_stride_t[0];
        T* out = static_cast<T*>(part != 0u ? p.out[1] : p.out[0]) +
                 head * (part != 0u ? p.out_stride_h[1] : p.out_stride_h[0]) + e + (t0 + ty) * step;
        for (uint32_t r0 = ty; r0 < rows; r0 += kReadBatch * p.ny) {
            // The loads of a batch are issued before the first of its stores.
            longlong2 at[kReadBatch];
            uint32_t w[kReadBatch][(V + 3) / 4];
            float sc[kReadBatch];
#pragma unroll
            for (int b = 0; b < kReadBatch; ++b) at[b] = row_at[min(r0 + b * p.ny, rows - 1u)];
#pragma unroll
            for (int b = 0; b < kReadBatch; ++b) load_codes<V>(codes + at[b].x, at[b].x, w[b]);
#pragma unroll
            for (int b = 0; b < kReadBatch; ++b) sc[b] = ld_float_if(scales + at[b].y, at[b].x);
#pragma unroll
            for (int b = 0; b < kReadBatch; ++b) {
                if (r0 + b * p.ny < rows && at[b].x != kRowBehind) {
                    alignas(16) T v[V];
#pragma unroll
                    for (int j = 0; j < V; ++j) v[j] = from_f32<T>(code_f32(w[b][j / 4] ^ 0x80808080u, j % 4) * sc[b]);
                    if constexpr (sizeof(T) * V == 16) *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(v);
                    else if constexpr (sizeof(T) * V == 8) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(v);
                    else if constexpr (sizeof(T) * V == 4) *reinterpret_cast<uint32_t*>(out) = *reinterpret_cast<const uint32_t*>(v);
                    else *out = v[0];
                }
                out += p.ny * step;
            }
        }
    }
}

// cache_read_kernel for widths that no wide store divides, into outputs without
// gaps: the output rows of a block are one run of values, cut into 16-byte
// stores whatever rows they hold. A store's V values come from one row of codes
// or the ends of two (d >= V), whose words of V codes (rows of codes start on
// one) are shifted together. 24 sequences of up to 2,964 rows of 2 x 189 fp32:
// 23.3 us, value by value 31.8.
template <class T>
static __global__ void __launch_bounds__(256) cache_read_flat_kernel(const __grid_constant__ ReadParams p) {
    constexpr uint32_t V = 16 / sizeof(T);
    using Word = typename std::conditional<V == 8, unsigned long long, uint32_t>::type;
    __shared__ longlong2 row_at[kReadRows];
    auto ld_word = [](const Word* at) -> Word {
        if constexpr (V == 4) return ld4_if(at);
        const uint2 u = ld8_if(at);
        return static_cast<Word>(static_cast<uint64_t>(u.y) << 32 | u.x);
    };
    await_previous();
    let_next_start();
    const uint32_t t0 = blockIdx.x * p.rows, rows = min(p.rows, p.total - t0), part = blockIdx.y;
    if (threadIdx.x < rows) {
        const int64_t s = read_slot(p, t0 + threadIdx.x);
        longlong2 at = make_longlong2(s == kRowBehind && p.zero_behind ? kRowNoPage : s, 0);
        if (s >= 0) {
            const uint32_t pg = p.page.div(static_cast<uint32_t>(s)), i = static_cast<uint32_t>(s) - pg * p.page.d;
            at.x = pg * p.code_page + i * p.code_row;
            at.y = pg * p.scale_page + i * p.scale_row;
        }
        row_at[threadIdx.x] = at;
    }
    __syncthreads();
    const int8_t* const codes = p.codes + part * p.code_part;
    const float* const scales = p.scales + part * p.scale_part;
    const uint32_t heads = p.by_heads.d, d = p.per_group.d, run = rows * heads * d;
    T* const out = static_cast<T*>(part != 0u ? p.out[1] : p.out[0]) + static_cast<int64_t>(t0) * heads * d;
    for (uint32_t f = threadIdx.x * V; f < run; f += 256u * V) {
        // (row, head, place) of the first value, and the (row, head) after it
        const uint32_t g0 = p.per_group.div(f), e = f - g0 * d, left = d - e, g1 = g0 + 1u;
        const uint32_t r0 = p.by_heads.div(g0), h0 = g0 - r0 * heads;
        const uint32_t r1 = min(p.by_heads.div(g1), rows - 1u), h1 = g1 - p.by_heads.div(g1) * heads;
        const longlong2 at0 = row_at[r0], at1 = row_at[r1];
        // The first row's codes from the one or two words that hold them, what
        // is missing from the second row's first word.
        Word w = 0, next = 0;
        float s0 = 0.0f, s1 = 0.0f;
        if (at0.x >= 0) {
            const int8_t* const q = codes + at0.x + h0 * p.code_head + e;
            const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(q) % V);
            const Word* const from = reinterpret_cast<const Word*>(q - off);
            w = ld_word(from) >> (8u * off);
            if (off + min(V, left) > V) w |= ld_word(from + 1) << (8u * (V - off));
            s0 = ld_float_if(scales + at0.y + h0 * p.scale_head);
        }
        if (left < V) {
            if (at1.x >= 0) {
                next = ld_word(reinterpret_cast<const Word*>(codes + at1.x + h1 * p.code_head));
                s1 = ld_float_if(scales + at1.y + h1 * p.scale_head);
            }
            w = (w & ((Word{1} << (8u * left)) - 1u)) | next << (8u * left);
        }
        const uint32_t q[2] = {static_cast<uint32_t>(w), static_cast<uint32_t>(static_cast<uint64_t>(w) >> 32)};
        alignas(16) T v[V];
#pragma unroll
        for (uint32_t j = 0; j < V; ++j)
            v[j] = from_f32<T>(code_f32(q[j / 4] ^ 0x80808080u, j % 4) * (j >= left ? s1 : s0));
        if (f + V <= run && at0.x != kRowBehind && at1.x != kRowBehind) {
            *reinterpret_cast<uint4*>(out + f) = *reinterpret_cast<const uint4*>(v);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < V; ++j)
                if (f + j < run && (j >= left ? at1.x : at0.x) != kRowBehind) out[f + j] = v[j];
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
    int out_vec4, out_vec16;  // rows of out start on four elements, on 16 bytes
    // Rows that the product quantises itself (the dot kernel), in place of a:
    const void* x;
    int64_t x_pitch;  // elements
    int x_vec16;      // they start on 16 bytes and hold a whole number of them
};

__device__ __forceinline__ float bias_at(const void* bias, int type, uint32_t n) {
    if (type == 1) return __half2float(static_cast<const __half*>(bias)[n]);
    if (type == 4) return __bfloat162float(static_cast<const __nv_bfloat16*>(bias)[n]);
    return static_cast<const float*>(bias)[n];
}

}  // namespace eb
