// The int8 matrix product with a scale per row and channel,
//   out[i][j] = (sum_l a[i][l] b[j][l]) sa[i] sb[j] + bias[j],
// in three forms; the host picks one by sizes and a model of their times (dot_form
// and gemm_form in int8.cu).
//
//  * gemm_int8_dot_kernel: a few rows (the codes of single tokens). The
//    weight is read once, 16 bytes a lane, and multiplied with dp4a.
//  * gemm_int8_wide_kernel: rows up to a few hundred. The weight is the
//    128-lane operand of the tensor core and the rows its narrow one; a
//    cluster of CTAs shares one output tile and splits k, the partial sums
//    meeting in shared memory.
//  * gemm_int8_pair_kernel: many rows. Persistent CTA pairs, 256 x 256
//    outputs per MMA, the epilogue of one tile under the products of the next.
//
// The sums are exact in int32 whatever their order, so every form and every
// split gives the same bits: the conversion to fp32 (one rounding where the
// sum passes 2^24), sa, then sb and the bias by one fused multiply-add, and
// the rounding to the output's type.
#pragma once

#include <cstdint>

#include "int8_kernels.cuh"
#include "ptx.cuh"

namespace eb {

__device__ __forceinline__ float scaled(int32_t acc, float sa, float sb, float bias) {
    return fmaf(static_cast<float>(acc) * sa, sb, bias);
}

// -------------------------------------------------------------- a few rows

constexpr int kDotChannels = 4;  // weight rows per warp and step
constexpr uint32_t kDotCodeBytes = 32768;  // most codes of quantised rows in shared memory

// The block's quantisation of MR rows (m of them there) to codes in shared
// memory, padded with zeros to `pitch` bytes: 8 / MR warps a row.
template <int MR, class X, int V>
__device__ __forceinline__ void dot_quantize(const GemmParams& p, int8_t* codes, uint32_t pitch, uint32_t* warp_max,
                                             float* scales) {
    constexpr uint32_t kWarps = 8 / MR, kThreads = kWarps * 32;
    const uint32_t row = threadIdx.x / kThreads, tid = threadIdx.x % kThreads;
    const bool there = row < p.m;
    const X* x = static_cast<const X*>(p.x) + (there ? row : 0u) * p.x_pitch;
    uint32_t top = 0;
    for (uint32_t e = tid * V; e < p.k; e += kThreads * V) {
        Access<X, V> u;
        u.load(x + e);
        top = u.top(top);
    }
    const uint32_t top32 = __reduce_max_sync(0xFFFFFFFFu, Access<X, V>::bits32(top));
    if ((threadIdx.x & 31u) == 0) warp_max[threadIdx.x >> 5] = top32;
    __syncthreads();
    uint32_t amax = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWarps; ++i) amax = max(amax, warp_max[row * kWarps + i]);
    const RowScale rs = make_scale<X>(amax);
    if (tid == 0) scales[row] = rs.s;
    for (uint32_t e = tid * V; there && e < pitch; e += kThreads * V) {
        uint32_t w[(V + 3) / 4] = {};
        if (e < p.k && rs.inv != 0.0f) {
            Access<X, V> u;
            u.load(x + e);
            float f[V];
            u.values(f);
            row_codes<V>(f, rs, w);
        }
        int8_t* out = codes + row * pitch + e;
        if constexpr (V == 8) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[V / 4 - 1]);
        else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(out) = w[0];
        else *out = static_cast<int8_t>(w[0]);
    }
    __syncthreads();
}

// MR rows of a against every row of b. A block's warps form groups of `wk`
// that split k between them; a group takes kDotChannels rows of b. Rows of b
// start on 16 bytes and their last 16 bytes may be read whole. X is int8 (rows
// of codes that start on 16 bytes too, the bytes past k masked out) or a float
// type: each block then quantises the rows itself, a few thousand values that
// stay in L2, which costs about 1 us and saves a launch and the codes' memory.
template <int MR, class X, class T>
static __global__ void __launch_bounds__(256) gemm_int8_dot_kernel(const __grid_constant__ GemmParams p, uint32_t wk) {
    __shared__ int32_t part[8][MR * kDotChannels];
    extern __shared__ __align__(16) int8_t row_codes_smem[];
    constexpr bool kFloat = !std::is_same<X, int8_t>::value;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t group = (blockIdx.x * 8u + warp) / wk, kw = warp % wk;
    const uint32_t n0 = group * kDotChannels;
    const uint32_t chunks = (p.k + 15u) / 16u;
    const int8_t* br[kDotChannels];
#pragma unroll
    for (int c = 0; c < kDotChannels; ++c) br[c] = p.b + static_cast<int64_t>(min(n0 + c, p.n - 1u)) * p.b_pitch;
    __shared__ float row_scales[kFloat ? MR : 1];
    await_previous();
    let_next_start();
    if constexpr (kFloat) {
        __shared__ uint32_t warp_max[8];
        // The first weights are on their way while the rows are quantised.
#pragma unroll
        for (int c = 0; c < kDotChannels; ++c)
            if (kw * 32u + lane < chunks)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(br[c] + (kw * 32u + lane) * 16u));
        if (p.x_vec16) dot_quantize<MR, X, 16 / static_cast<int>(sizeof(X))>(p, row_codes_smem, chunks * 16u, warp_max, row_scales);
        else dot_quantize<MR, X, 1>(p, row_codes_smem, chunks * 16u, warp_max, row_scales);
    }
    int32_t acc[MR][kDotChannels] = {};
    const uint32_t tail = p.k & 15u;
#pragma unroll 4
    for (uint32_t i = kw * 32u + lane; i < chunks; i += wk * 32u) {
        uint4 w[kDotChannels];
#pragma unroll
        for (int c = 0; c < kDotChannels; ++c) w[c] = ld16(br[c] + i * 16u);
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            uint4 x;
            const uint32_t mm = min(static_cast<uint32_t>(m), p.m - 1u);
            if constexpr (kFloat) {
                x = *reinterpret_cast<const uint4*>(row_codes_smem + (mm * chunks + i) * 16u);
            } else {
                x = ld16(p.a + static_cast<int64_t>(mm) * p.a_pitch + i * 16u);
                if (tail != 0u && i == chunks - 1u) {
                    uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int keep = static_cast<int>(tail) - 4 * j;
                        xw[j] = keep >= 4 ? xw[j] : keep <= 0 ? 0 : xw[j] & ((1u << (8 * keep)) - 1u);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < kDotChannels; ++c) {
                int32_t s = acc[m][c];
                s = __dp4a(static_cast<int>(x.x), static_cast<int>(w[c].x), s);
                s = __dp4a(static_cast<int>(x.y), static_cast<int>(w[c].y), s);
                s = __dp4a(static_cast<int>(x.z), static_cast<int>(w[c].z), s);
                acc[m][c] = __dp4a(static_cast<int>(x.w), static_cast<int>(w[c].w), s);
            }
        }
    }
    int32_t mine = 0;  // lane m * kDotChannels + c keeps that sum
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int c = 0; c < kDotChannels; ++c) {
            const int32_t s = __reduce_add_sync(0xffffffffu, acc[m][c]);
            if (lane == static_cast<uint32_t>(m * kDotChannels + c)) mine = s;
        }
    if (wk > 1u) {
        if (lane < MR * kDotChannels) part[warp][lane] = mine;
        __syncthreads();
        if (kw != 0u) return;
        if (lane < MR * kDotChannels)
            for (uint32_t j = 1; j < wk; ++j) mine += part[warp + j][lane];
    }
    const uint32_t m = lane / kDotChannels, n = n0 + lane % kDotChannels;
    if (lane >= MR * kDotChannels || m >= p.m || n >= p.n) return;
    const float scale = kFloat ? row_scales[kFloat ? m : 0u] : p.a_scales[m];
    const float bias = p.bias == nullptr ? 0.0f : bias_at(p.bias, p.bias_type, n);
    static_cast<T*>(p.out)[m * p.out_pitch + n] = from_f32<T>(scaled(mine, scale, p.b_scales[n], bias));
}

// ------------------------------------------------------------- wide kernel

constexpr uint32_t kGemmStageK = 128;  // bytes of k per pipeline stage: one swizzle atom
constexpr uint32_t kWideChannels = 128;
constexpr uint32_t kWideMaxStages = 8;
constexpr int kWideThreads = 192;  // TMA, MMA and four epilogue warps

// A wait that must be sat out whatever else went wrong (an abort does not end
// it, only its own limit): for what is under way before a CTA exits.
__device__ __forceinline__ bool finish_wait(uint32_t bar, uint32_t parity) {
    const long long start = clock64();
    while (!mbar_try_wait(bar, parity)) {
        if (clock64() - start > kWaitTimeoutCycles) {
            record_device_error(kDevErrWaitTimeout);
            return false;
        }
    }
    return true;
}

// The last load issued to each stage (barriers `full0`, 8 bytes apart) lands.
__device__ __forceinline__ void land_loads(uint32_t full0, uint32_t issued_mask, uint32_t issued_parity) {
    while (issued_mask != 0u) {
        const uint32_t s = __ffs(issued_mask) - 1u;
        finish_wait(full0 + 8u * s, (issued_parity >> s) & 1u);
        issued_mask &= issued_mask - 1u;
    }
}

__device__ __forceinline__ int4 ld_cluster(uint32_t addr) {
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// Output tiles of 128 channels x BT rows. With S = 1 the CTAs are persistent:
// each takes every gridDim.x-th tile, its loads running on into the next tile
// while the epilogue empties the last one (two accumulators in TMEM). A thread
// of the epilogue owns a channel and stores its column of the tile straight
// from TMEM (a warp's stores of one row are neighbours). With S > 1 a cluster
// of S CTAs makes one tile, each summing its share of k; every CTA leaves its
// int32 tile in shared memory (over the pipeline's buffers, which are done)
// and sums BT / S of the rows over the cluster, four channels a lane.
template <int BT, int S, class T>
static __global__ void __launch_bounds__(kWideThreads)
    gemm_int8_wide_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x,
                          const __grid_constant__ GemmParams p, uint32_t stages, uint32_t n_rt, uint32_t tiles) {
    extern __shared__ uint8_t smem_raw[];
    // full and empty of every stage, full and empty of both accumulators, all MMAs done
    __shared__ __align__(8) uint64_t bars[2 * kWideMaxStages + 5];
    __shared__ float row_scales[4][BT];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int* const abort_flag = &abort_word;
    constexpr uint32_t kWBytes = kWideChannels * kGemmStageK;
    constexpr uint32_t kStageBytes = kWBytes + BT * kGemmStageK;
    constexpr uint32_t kAccCols = BT < 32 ? 32 : BT;  // the epilogue reads 32 columns at a time
    constexpr uint32_t kTmemCols = S == 1 ? 2 * kAccCols : kAccCols;
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t sbase = (raw + 1023u) & ~1023u;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t split = S == 1 ? 0u : blockIdx.x % S;  // = rank in the cluster
    const uint32_t tile0 = blockIdx.x / S, step = gridDim.x / S;
    const uint32_t kblocks = (p.k + kGemmStageK - 1u) / kGemmStageK;
    const uint32_t kb0 = static_cast<uint32_t>(static_cast<uint64_t>(kblocks) * split / S);
    const uint32_t kb1 = static_cast<uint32_t>(static_cast<uint64_t>(kblocks) * (split + 1u) / S);
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty = [&](uint32_t s) { return bar0 + 8u * (kWideMaxStages + s); };
    auto tfull = [&](uint32_t a) { return bar0 + 8u * (2 * kWideMaxStages + a); };
    auto tempty = [&](uint32_t a) { return bar0 + 8u * (2 * kWideMaxStages + 2 + a); };
    const uint32_t done = bar0 + 8u * (2 * kWideMaxStages + 4);

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tm_w);
        tma_prefetch_desc(&tm_x);
        for (uint32_t s = 0; s < stages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            mbar_init(tfull(a), 1);
            mbar_init(tempty(a), 4);
        }
        mbar_init(done, 1);
        abort_word = 0;
        fence_mbarrier_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_slot), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    await_previous();
    let_next_start();
    T* const out = static_cast<T*>(p.out);
    // Of a cluster's sums, the four channels of a lane: fetched while they are made.
    float sb4[4], bias4[4];
    if constexpr (S > 1) {
        const uint32_t n = tile0 / n_rt * kWideChannels + lane * 4u;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            sb4[c] = n + c < p.n ? p.b_scales[n + c] : 0.0f;
            bias4[c] = n + c < p.n && p.bias != nullptr ? bias_at(p.bias, p.bias_type, n + c) : 0.0f;
        }
    }

    if (warp == 0) {
        if (elect_one_sync()) {
            uint32_t stage = 0, phase = 0, issued_mask = 0, issued_parity = 0;
            bool ok = true;
            for (uint32_t t = tile0; ok && t < tiles; t += step) {
                const int32_t n0 = static_cast<int32_t>(t / n_rt * kWideChannels), m0 = static_cast<int32_t>(t % n_rt * BT);
                for (uint32_t kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait(empty(stage), phase ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(full(stage), kStageBytes);
                    const uint32_t dst = sbase + stage * kStageBytes;
                    const int32_t x = static_cast<int32_t>(kb * kGemmStageK);
                    tma_load_2d(dst, &tm_w, full(stage), x, n0);
                    tma_load_2d(dst + kWBytes, &tm_x, full(stage), x, m0);
                    issued_mask |= 1u << stage;
                    issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            land_loads(bar0, issued_mask, issued_parity);
        }
    } else if (warp == 1) {
        if (elect_one_sync()) {
            constexpr uint32_t idesc = make_idesc(2, 1, kWideChannels, BT);
            uint32_t stage = 0, phase = 0, iter = 0;
            bool ok = true;
            for (uint32_t t = tile0; ok && t < tiles; t += step, ++iter) {
                const uint32_t acc = iter & 1u;
                if (!mbar_wait(tempty(acc), ((iter >> 1) & 1u) ^ 1u, abort_flag)) break;
                tc_fence_after();
                for (uint32_t kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait(full(stage), phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t w = sbase + stage * kStageBytes, x = w + kWBytes;
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        tc_mma<MmaKind::I8>(tmem + acc * kAccCols, smem_desc_k128(w + 32u * k), smem_desc_k128(x + 32u * k),
                                            idesc, kb == kb0 && k == 0 ? 0u : 1u);
                    tc_commit(empty(stage));
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                tc_commit(tfull(acc));
            }
            // Nothing writes to TMEM once it is freed, whatever ended the loop.
            tc_commit(done);
            finish_wait(done, 0);
        }
    } else {
        const uint32_t quad = warp & 3u, row = quad * 32u + lane;  // TMEM lane = channel of the tile
        float* const scales = row_scales[quad];
        uint32_t iter = 0;
        for (uint32_t t = tile0; t < tiles; t += step, ++iter) {
            const uint32_t acc = iter & 1u;
            const uint32_t m0 = t % n_rt * BT, n = t / n_rt * kWideChannels + row;
            const uint32_t rows = m0 < p.m ? min(static_cast<uint32_t>(BT), p.m - m0) : 0u;
            const bool valid = n < p.n;
            for (uint32_t r = lane; r < BT; r += 32) scales[r] = r < rows ? p.a_scales[m0 + r] : 0.0f;
            float sb = 0.0f, bias = 0.0f;
            if (S == 1 && valid) {
                sb = p.b_scales[n];
                if (p.bias != nullptr) bias = bias_at(p.bias, p.bias_type, n);
            }
            __syncwarp();
            bool ok = mbar_wait(tfull(acc), (iter >> 1) & 1u, abort_flag);
            ok = __all_sync(0xFFFFFFFFu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t taddr = tmem + ((quad * 32u) << 16) + acc * kAccCols;
            T* dst = out + static_cast<int64_t>(m0) * p.out_pitch + n;
#pragma unroll 1
            for (uint32_t c = 0; c < BT; c += 32) {
                uint32_t v[32];
                __syncwarp();
                tmem_ld_32x32b_x32(taddr + c, v);
                tmem_wait_ld();
                if (S == 1 && c + 32 >= BT) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty(acc));
                }
                if (kb0 == kb1) {
#pragma unroll
                    for (uint32_t i = 0; i < 32; ++i) v[i] = 0;
                }
#pragma unroll
                for (uint32_t i = 0; i < (BT < 32 ? BT : 32); ++i) {
                    if constexpr (S == 1) {
                        const T o = from_f32<T>(scaled(static_cast<int32_t>(v[i]), scales[c + i], sb, bias));
                        if (valid && c + i < rows) *dst = o;
                        dst += p.out_pitch;
                    } else {
                        *reinterpret_cast<uint32_t*>(smem_raw + (sbase - raw) + ((c + i) * kWideChannels + row) * 4u) = v[i];
                    }
                }
            }
            __syncwarp();
        }
    }
    // TMEM goes back before this CTA waits for the others of its cluster: a CTA
    // of another launch that waits for TMEM on this SM, and whose own partner
    // holds the TMEM that a CTA of this cluster waits for, would never get it.
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
    if constexpr (S > 1) {
        __syncwarp();
        cluster_sync();
        const uint32_t m0 = tile0 % n_rt * BT, n = tile0 / n_rt * kWideChannels + lane * 4u;
        // Rows r of the tile with r % S == split, one warp per row and step.
        for (uint32_t r = split + S * warp; r < BT && m0 + r < p.m; r += S * (kWideThreads / 32)) {
            const uint32_t at = sbase + (r * kWideChannels + lane * 4u) * 4u;
            int4 part[S];
#pragma unroll
            for (int j = 0; j < S; ++j) part[j] = ld_cluster(mapa_shared(at, j));
            int32_t sum[4] = {};
#pragma unroll
            for (int j = 0; j < S; ++j) {
                sum[0] += part[j].x;
                sum[1] += part[j].y;
                sum[2] += part[j].z;
                sum[3] += part[j].w;
            }
            T o[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = from_f32<T>(scaled(sum[c], row_scales[0][r], sb4[c], bias4[c]));
            T* dst = out + static_cast<int64_t>(m0 + r) * p.out_pitch + n;
            if (p.out_vec4 && n + 4u <= p.n) {
                if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(o);
                else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(o);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (n + c < p.n) dst[c] = o[c];
            }
        }
        cluster_sync();  // the others may still read this CTA's sums
    }
}

// ------------------------------------------------------------- pair kernel

constexpr uint32_t kPairM = 256, kPairN = 256;
constexpr uint32_t kPairStages = 5;  // four lose 5 % on 8192^3, six do not fit
constexpr uint32_t kPairEpilogueWarps = 8;
constexpr int kPairThreads = 32 * (2 + kPairEpilogueWarps);
constexpr uint32_t kPairStageBytes = (kPairM / 2 + kPairN / 2) * kGemmStageK;
constexpr uint32_t kPairStoreBytes = 32 * 128;  // per epilogue warp: 32 rows of 128 bytes
constexpr uint32_t kPairStoreOffset = kPairStages * kPairStageBytes;
constexpr uint32_t kPairColsOffset = kPairStoreOffset + kPairEpilogueWarps * kPairStoreBytes;
constexpr uint32_t kPairBarOffset = kPairColsOffset + kPairEpilogueWarps * (kPairN / 2) * 8;
constexpr uint32_t kPairSmemBytes = 1024 + kPairBarOffset + 256;
static_assert(8 * (2 * kPairStages + 5) + 16 <= 256, "barrier area");
static_assert(kPairSmemBytes <= 232448, "shared memory");

template <class T>
struct Packed;
template <>
struct Packed<float> {
    static constexpr uint32_t per_word = 1;
};
template <>
struct Packed<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static constexpr uint32_t per_word = 2;
};
template <>
struct Packed<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static constexpr uint32_t per_word = 2;
};

// Tile order: columns of `kPairGroup` row tiles, so that the tiles under way
// at any time span about as many rows of a as of b and both stay in L2. The
// last tiles, where they are too few to give every pair one but halves of them
// fit one wave, are made as halves of 128 columns, which take 0.7 of a whole
// one's time: 4096^3 (3.46 waves) 48.9 -> 47.1 us, 10,000 x 1536 x 768 to fp32
// 20.7 -> 19.3.
constexpr uint32_t kPairGroup = 8;

struct PairUnit {
    uint32_t mt, n0, bn;  // row tile, first column, columns
};

__device__ __forceinline__ PairUnit pair_unit(uint32_t unit, uint32_t whole, uint32_t n_mt, uint32_t n_nt) {
    const uint32_t i = unit < whole ? unit : whole + (unit - whole) / 2u;
    const uint32_t per = kPairGroup * n_nt, g = i / per, r = i % per;
    const uint32_t rows = min(kPairGroup, n_mt - g * kPairGroup);
    PairUnit u;
    u.mt = g * kPairGroup + r % rows;
    u.n0 = r / rows * kPairN;
    u.bn = kPairN;
    if (unit >= whole) {
        u.bn = kPairN / 2;
        u.n0 += (unit - whole) % 2u * u.bn;
    }
    return u;
}

// Roles as in the search kernel: warp 0 loads, warp 1 of rank 0 issues the
// pair's MMAs, eight warps empty one accumulator while the other fills. A
// thread of the epilogue owns a row of a and half of the tile's columns; its
// results go through 128-byte rows of shared memory, so that a warp stores
// whole lines, 16 bytes a lane (one element where the output's rows start
// anywhere). The scales of the next tile are fetched under the current one.
template <class T>
static __global__ void __launch_bounds__(kPairThreads, 1)
    gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                          const __grid_constant__ GemmParams p, uint32_t n_mt, uint32_t n_nt, uint32_t whole,
                          uint32_t units) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t sbase = (raw + 1023u) & ~1023u;
    uint8_t* smem = smem_raw + (sbase - raw);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t rank = cluster_ctarank(), pair = cluster_id_x(), pairs = cluster_count_x();
    const bool leader = rank == 0;
    const uint32_t kblocks = (p.k + kGemmStageK - 1u) / kGemmStageK;

    const uint32_t bar0 = sbase + kPairBarOffset;
    auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (kPairStages + s); };
    auto tfull_bar = [&](uint32_t a) { return bar0 + 8u * (2 * kPairStages + a); };
    auto tempty_bar = [&](uint32_t a) { return bar0 + 8u * (2 * kPairStages + 2 + a); };
    const uint32_t mma_done_bar = bar0 + 8u * (2 * kPairStages + 4);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + kPairBarOffset + 8 * (2 * kPairStages + 5));
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    auto a_addr = [&](uint32_t s) { return sbase + s * kPairStageBytes; };
    auto b_addr = [&](uint32_t s) { return a_addr(s) + kPairM / 2 * kGemmStageK; };

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kPairStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), kPairEpilogueWarps * 2);
        }
        mbar_init(mma_done_bar, 1);
        *abort_flag = 0;
        fence_mbarrier_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), 2 * kPairN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    await_previous();
    let_next_start();

    if (warp == 0) {
        if (elect_one_sync()) {
            tma_prefetch_desc(&tm_a);
            tma_prefetch_desc(&tm_b);
            uint32_t stage = 0, phase = 0, issued_mask = 0, issued_parity = 0;
            bool ok = true;
            for (uint32_t i = pair; ok && i < units; i += pairs) {
                const PairUnit u = pair_unit(i, whole, n_mt, n_nt);
                const int32_t a_row = static_cast<int32_t>(u.mt * kPairM + rank * (kPairM / 2));
                const int32_t b_row = static_cast<int32_t>(u.n0 + rank * (u.bn / 2));
                for (uint32_t kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) {
                        ok = false;
                        break;
                    }
                    const int32_t x = static_cast<int32_t>(kb * kGemmStageK);
                    if (leader) mbar_arrive_expect_tx(full_bar(stage), (kPairM + u.bn) * kGemmStageK);
                    const uint32_t fb = mapa_shared(full_bar(stage), 0);
                    tma_load_2d_pair(a_addr(stage), &tm_a, fb, x, a_row);
                    tma_load_2d_pair(b_addr(stage), &tm_b, fb, x, b_row);
                    if (u.bn == kPairN)
                        tma_load_2d_pair(b_addr(stage) + kPairN / 4 * kGemmStageK, &tm_b, fb, x,
                                         b_row + static_cast<int32_t>(kPairN / 4));
                    issued_mask |= 1u << stage;
                    issued_parity = (issued_parity & ~(1u << stage)) | (phase << stage);
                    if (++stage == kPairStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // Every load must land before the CTAs exit; rank 0's barriers
            // count both CTAs' bytes, and the peer leaves only after the
            // closing cluster barrier.
            if (leader) land_loads(bar0, issued_mask, issued_parity);
        }
    } else if (warp == 1) {
        if (leader && elect_one_sync()) {
            uint32_t stage = 0, phase = 0, iter = 0;
            bool ok = true;
            for (uint32_t i = pair; ok && i < units; i += pairs, ++iter) {
                const uint32_t acc = iter & 1u;
                const uint32_t idesc = i < whole ? make_idesc(2, 1, kPairM, kPairN) : make_idesc(2, 1, kPairM, kPairN / 2);
                if (!mbar_wait_cluster(tempty_bar(acc), ((iter >> 1) & 1u) ^ 1u, abort_flag)) break;
                tc_fence_after();
                const uint32_t d = tmem_base + acc * kPairN;
                for (uint32_t kb = 0; kb < kblocks; ++kb) {
                    if (!mbar_wait(full_bar(stage), phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        tc_mma<MmaKind::I8, 2>(d, smem_desc_k128(a_addr(stage) + 32u * k),
                                               smem_desc_k128(b_addr(stage) + 32u * k), idesc, kb == 0 && k == 0 ? 0u : 1u);
                    tc_commit_pair_both(empty_bar(stage), 0x3);
                    if (++stage == kPairStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                tc_commit_pair_both(tfull_bar(acc), 0x3);
            }
            tc_commit_pair(mma_done_bar);
            finish_wait(mma_done_bar, 0);
        }
    } else {
        const uint32_t ew = warp - 2u, quad = warp & 3u, half = ew >> 2;
        constexpr uint32_t kHalf = kPairN / 2;       // columns of a warp (of a half tile: half)
        constexpr uint32_t kOwn = kHalf / 32;        // columns whose scales a lane fetches
        constexpr uint32_t kCols = 128 / sizeof(T);  // columns per 128 bytes of output
        constexpr uint32_t kPer = Packed<T>::per_word;
        uint8_t* const store = smem + kPairStoreOffset + ew * kPairStoreBytes;
        float2* const cols = reinterpret_cast<float2*>(smem + kPairColsOffset) + ew * kHalf;
        const uint32_t tempty0 = mapa_shared(tempty_bar(0), 0), tempty1 = mapa_shared(tempty_bar(1), 0);
        T* const out = static_cast<T*>(p.out);
        float sa = 0.0f;
        float2 sb[kOwn];  // scale and bias
        auto fetch = [&](uint32_t i) {
            const PairUnit u = pair_unit(i, whole, n_mt, n_nt);
            const uint32_t m = u.mt * kPairM + rank * (kPairM / 2) + quad * 32u + lane;
            sa = ld_float_if(p.a_scales + m, m < p.m ? 0 : -1);
#pragma unroll
            for (uint32_t j = 0; j < kOwn; ++j) {
                const uint32_t n = u.n0 + half * (u.bn / 2) + j * 32u + lane;
                const bool there = n < p.n && j * 32u < u.bn / 2;
                sb[j] = make_float2(ld_float_if(p.b_scales + n, there ? 0 : -1), 0.0f);
                if (there && p.bias != nullptr) sb[j].y = bias_at(p.bias, p.bias_type, n);
            }
        };
        if (pair < units) fetch(pair);
        uint32_t iter = 0;
        for (uint32_t i = pair; i < units; i += pairs, ++iter) {
            const PairUnit u = pair_unit(i, whole, n_mt, n_nt);
            const uint32_t acc = iter & 1u, groups = u.bn / 64;
            const uint32_t m_warp = u.mt * kPairM + rank * (kPairM / 2) + quad * 32u;
            const uint32_t n_half = u.n0 + half * (u.bn / 2);
            const float row_scale = sa;
#pragma unroll
            for (uint32_t j = 0; j < kOwn; ++j) cols[j * 32u + lane] = sb[j];
            if (i + pairs < units) fetch(i + pairs);
            __syncwarp();
            bool ok = mbar_wait(tfull_bar(acc), (iter >> 1) & 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t taddr = tmem_base + ((quad * 32u) << 16) + acc * kPairN + half * (u.bn / 2);
            const uint32_t rows = m_warp < p.m ? min(32u, p.m - m_warp) : 0u;
            // 32 columns at a time, the next ones on their way from TMEM.
            uint32_t v[2][32];
            tmem_ld_32x32b_x32(taddr, v[0]);
#pragma unroll
            for (uint32_t g = 0; g < kHalf / 32; ++g) {
                if (g >= groups) break;
                tmem_wait_ld();
                if (g + 1 < groups) {
                    tmem_ld_32x32b_x32(taddr + (g + 1) * 32u, v[(g + 1) & 1]);
                } else {  // all of the accumulator is in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(acc ? tempty1 : tempty0);
                }
                uint32_t w[32 / kPer];
#pragma unroll
                for (uint32_t j = 0; j < 32; j += 2) {
                    const float4 c = *reinterpret_cast<const float4*>(cols + g * 32u + j);  // scale, bias of two columns
                    const float f0 = scaled(static_cast<int32_t>(v[g & 1][j]), row_scale, c.x, c.y);
                    const float f1 = scaled(static_cast<int32_t>(v[g & 1][j + 1]), row_scale, c.z, c.w);
                    if constexpr (kPer == 2) {
                        w[j / 2] = Packed<T>::pack(f0, f1);
                    } else {
                        w[j] = __float_as_uint(f0);
                        w[(j + 1) % (32 / kPer)] = __float_as_uint(f1);
                    }
                }
                // 16-byte pieces of the 128-byte rows change places with the
                // row, so that neither side meets a bank conflict.
#pragma unroll
                for (uint32_t j = 0; j < 32 / kPer; j += 4) {
                    const uint32_t piece = (g * 32u % kCols) * sizeof(T) / 16u + j / 4u;
                    *reinterpret_cast<uint4*>(store + lane * 128u + ((piece ^ (lane & 7u)) * 16u)) =
                        make_uint4(w[j], w[j + 1], w[j + 2], w[j + 3]);
                }
                if ((g + 1) * 32u % kCols != 0u) continue;
                __syncwarp();
                const uint32_t n = n_half + (g + 1) * 32u - kCols;
                if (p.out_vec16 && n + kCols <= p.n) {
                    T* dst = out + static_cast<int64_t>(m_warp + lane / 8u) * p.out_pitch + n + (lane & 7u) * (16u / sizeof(T));
#pragma unroll
                    for (uint32_t r = 0; r < 32; r += 4) {
                        const uint32_t row = r + lane / 8u;
                        const uint4 x = *reinterpret_cast<const uint4*>(store + row * 128u + (((lane & 7u) ^ (row & 7u)) * 16u));
                        if (row < rows) *reinterpret_cast<uint4*>(dst) = x;
                        dst += 4 * p.out_pitch;
                    }
                } else if (n < p.n) {
                    for (uint32_t r = 0; r < rows; ++r) {
#pragma unroll
                        for (uint32_t q = 0; q < kCols; q += 32) {
                            const uint32_t byte = (q + lane) * sizeof(T), piece = (byte / 16u) ^ (r & 7u);
                            if (n + q + lane < p.n)
                                out[(m_warp + r) * p.out_pitch + n + q + lane] =
                                    *reinterpret_cast<const T*>(store + r * 128u + piece * 16u + byte % 16u);
                        }
                    }
                }
                __syncwarp();
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 2 * kPairN);
    }
}

// ------------------------------------------------- operands that TMA cannot read

// Copies rows whose start or pitch is no multiple of 16 bytes to rows of
// `pitch` bytes (a multiple of 16), zero past the width: one launch for one or
// both operands, four bytes a thread.
struct RepackParams {
    const int8_t* in[2];
    int8_t* out[2];
    int64_t in_pitch[2];
    uint32_t rows[2], k;
    FastDiv words;  // pitch / 4
};

static __global__ void __launch_bounds__(256) repack_codes_kernel(const __grid_constant__ RepackParams p) {
    await_previous();
    let_next_start();
    const uint32_t which = blockIdx.y;
    const uint32_t rows = which ? p.rows[1] : p.rows[0];
    const int8_t* const in = which ? p.in[1] : p.in[0];
    const int64_t in_pitch = which ? p.in_pitch[1] : p.in_pitch[0];
    const uint64_t blocks_of = (static_cast<uint64_t>(rows) * p.words.d + 255u) / 256u;
    for (uint64_t block = blockIdx.x; block < blocks_of; block += gridDim.x) {
        // Row and word of a block's first thread by a long division, once.
        const uint64_t i0 = block * 256u;
        const uint32_t r0 = static_cast<uint32_t>(i0 / p.words.d);
        const uint32_t c0 = static_cast<uint32_t>(i0 - static_cast<uint64_t>(r0) * p.words.d) + threadIdx.x;
        const uint32_t dr = p.words.div(c0), r = r0 + dr, c = (c0 - dr * p.words.d) * 4u;
        if (r >= rows) continue;
        const int8_t* src = in + r * in_pitch + c;
        uint32_t w = 0;
        if (c + 4u <= p.k) {
            // Four bytes from the two aligned words that hold them; the second
            // is read only where it holds one of them.
            const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(src)) & 3u;
            const uint32_t* at = reinterpret_cast<const uint32_t*>(src - off);
            const uint32_t lo = ld4_if(at), hi = ld4_if(at + 1, off != 0u ? 0 : -1);
            w = __funnelshift_r(lo, hi, 8u * off);
        } else {
            for (uint32_t j = 0; c + j < p.k; ++j) w |= static_cast<uint32_t>(static_cast<uint8_t>(src[j])) << (8u * j);
        }
        int8_t* out = which ? p.out[1] : p.out[0];
        *reinterpret_cast<uint32_t*>(out + (static_cast<uint64_t>(r) * p.words.d * 4u + c)) = w;
    }
}

}  // namespace eb
