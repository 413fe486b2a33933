// 8-bit row operators: quantise rows, multiply int8 matrices with a scale per
// row and channel, write rows into the pages of a cache and read them back.
// Kernels in int8_kernels.cuh; the C ABI at the end of this file.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>

#include "../../include/elips_b200.h"
#include "capi_util.cuh"
#include "engine.cuh"
#include "int8_gemm.cuh"
#include "int8_kernels.cuh"
#include "profiler.cuh"
#include "wait_selftest.cuh"

namespace eb {
namespace {

void launch_ok(const char* what) { check_cuda(cudaGetLastError(), ELIPS_B200_KERNEL_LAUNCH_FAILED, what); }

[[noreturn]] void bad(const std::string& what) { fail(ELIPS_B200_INVALID_ARGUMENT, what); }

uint32_t blocks_for(uint64_t items, uint32_t per_block) {
    const uint64_t b = (items + per_block - 1) / per_block;
    if (b > 0x7FFFFFFFull) bad("too many rows in one call");
    return static_cast<uint32_t>(b);
}

uint32_t cdiv(uint64_t a, uint64_t b) { return static_cast<uint32_t>((a + b - 1) / b); }

constexpr size_t kMaxDim = size_t{1} << 24;
constexpr size_t kMaxRows = 0x7FFFFFF0ull;
// Largest k whose sum of products of int8 values (at most 2^14 each) stays
// below 2^31.
constexpr size_t kMaxK = 131071;

void check_float_type(int type) {
    if (type != ELIPS_B200_PRECISION_FP32 && type != ELIPS_B200_PRECISION_FP16 && type != ELIPS_B200_PRECISION_BF16)
        bad("element types are fp32, fp16 and bf16");
}

void check_rows(size_t n, size_t d, int type) {
    check_float_type(type);
    if (d == 0 || d > kMaxDim) bad("row width must be in [1, 2^24]");
    if (n > kMaxRows) bad("too many rows in one call");
}

// fn is called with a value of the element type that `type` names.
template <class Fn>
void with_float_type(int type, Fn&& fn) {
    switch (type) {
        case ELIPS_B200_PRECISION_FP32: fn(float{}); return;
        case ELIPS_B200_PRECISION_FP16: fn(__half{}); return;
        case ELIPS_B200_PRECISION_BF16: fn(__nv_bfloat16{}); return;
        default: check_float_type(type);
    }
}

// A launch that may start while the kernel before it in the stream ends
// (early); it waits for that one itself (await_previous). After another call of
// the same kind: 64 x 100,000 x 384 scores 14.3 -> 12.0 us, prompts through a
// cache 45.7 -> 41.5, new tokens in a graph 5.4 -> 4.7.
struct LaunchConfig {
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr[2];
    LaunchConfig(dim3 grid, uint32_t threads, size_t smem, cudaStream_t stream, bool early = true) {
        cfg.gridDim = grid;
        cfg.blockDim = dim3(threads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cfg.attrs = attr;
        cfg.numAttrs = early ? 1 : 0;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
    }
    void clusters_of(uint32_t x) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = x;
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
    }
    template <class... K, class... A>
    void launch(void (*kernel)(K...), A&&... args) {
        check_cuda(cudaLaunchKernelEx(&cfg, kernel, static_cast<K>(args)...), ELIPS_B200_KERNEL_LAUNCH_FAILED, "kernel launch");
    }
};

template <class T, int V, int G, int NV, bool SHIFT>
void launch_rows(const QuantParams& p, cudaStream_t stream) {
    LaunchConfig cfg(dim3(blocks_for(p.groups, 256 / G)), 256, 0, stream);
    if (p.slots == nullptr) cfg.launch(quantize_rows_kernel<T, V, G, NV, false, SHIFT>, p);
    else cfg.launch(quantize_rows_kernel<T, V, G, NV, true, SHIFT>, p);
}

// Few threads with many accesses each: what a thread spends on finding its row
// is shared by more values, and up to 512 accesses a row needs no more than a
// warp. Wider rows take a block (1000 x 30,000 bf16: 26.2 us read twice with
// four accesses a thread, 17.4 held in sixteen), and so do rows too few to
// fill the SMs, whose time is that of one row (1 x 4096 bf16: 3.1 us with a
// warp, 1.7 with a block).
template <class T, int V, bool SHIFT>
void launch_rows_of(const QuantParams& p, cudaStream_t stream) {
    const uint32_t n = cdiv(p.d + (SHIFT ? V - 1 : 0), V);  // accesses per row
    const bool few = p.groups <= 1024;
    if constexpr (V > 1) {
        if (n <= 8) return launch_rows<T, V, 4, 2, SHIFT>(p, stream);
        if (n <= 16) return launch_rows<T, V, 4, 4, SHIFT>(p, stream);
    }
    if (n <= 32) launch_rows<T, V, 8, 4, SHIFT>(p, stream);
    else if (n > 64 && n <= 512 && few) launch_rows<T, V, 256, 2, SHIFT>(p, stream);
    else if (n <= 128) launch_rows<T, V, 32, 4, SHIFT>(p, stream);
    else if (n <= 256) launch_rows<T, V, 32, 8, SHIFT>(p, stream);
    else if (n <= 512) launch_rows<T, V, 32, 16, SHIFT>(p, stream);
    else if (n <= 1024) launch_rows<T, V, 256, 4, SHIFT>(p, stream);
    else launch_rows<T, V, 256, 16, SHIFT>(p, stream);
}

// fn(first row, groups) for runs of rows whose (part, head) groups are fewer
// than 2^30, what one launch indexes.
template <class Fn>
void in_runs(size_t t, uint32_t per_t, Fn&& fn) {
    const size_t step = std::max<size_t>(1, (size_t{1} << 30) / per_t);
    for (size_t t0 = 0; t0 < t; t0 += step) fn(static_cast<uint32_t>(t0), static_cast<uint32_t>(std::min(step, t - t0) * per_t));
}

void launch_quantize(int type, QuantParams p, uint32_t parts, cudaStream_t stream) {
    with_float_type(type, [&](auto tag) {
        using T = decltype(tag);
        constexpr uint32_t V = 16 / sizeof(T);
        // Rows are read 16 bytes at a time where their codes can be stored as
        // many at a time; as they are where each starts on 16 bytes and holds a
        // whole number of them, else shifted (where a block holds a row).
        uint64_t rows = p.d % V, codes = reinterpret_cast<uintptr_t>(p.codes);
        for (uint32_t i = 0; i < parts; ++i) {
            rows |= reinterpret_cast<uintptr_t>(p.x[i]) % 16;
            rows |= (static_cast<uint64_t>(p.x_stride_t[i]) | static_cast<uint64_t>(p.x_stride_h[i])) % V;
        }
        codes |= static_cast<uint64_t>(p.code_part | p.code_page | p.code_row | p.code_head);
        const bool wide = codes % V == 0, held = p.d + V - 1 <= 256u * 16u * V;
        in_runs(p.t, p.per_t.d, [&](uint32_t t0, uint32_t groups) {
            p.t0 = t0;
            p.groups = groups;
            if (wide && rows == 0) launch_rows_of<T, V, false>(p, stream);
            else if (wide && held) launch_rows_of<T, V, true>(p, stream);
            else launch_rows_of<T, 1, false>(p, stream);
        });
    });
    launch_ok("row quantisation launch");
}

void quantize_rows(const void* x, int type, size_t n, size_t d, int64_t x_pitch, int8_t* codes, size_t code_pitch,
                   float* scales, cudaStream_t stream) {
    if (n == 0) return;
    QuantParams p{};
    p.x[0] = x;
    p.x_stride_t[0] = n > 1 ? x_pitch : 0;
    p.codes = codes;
    p.scales = scales;
    p.code_page = static_cast<int64_t>(n > 1 ? code_pitch : 0);
    p.scale_page = 1;
    p.t = static_cast<uint32_t>(n);
    p.heads = 1;
    p.d = static_cast<uint32_t>(d);
    p.num_slots = static_cast<int64_t>(n);
    p.dup = kDupNone;
    Profiler::Scope prof("quantize_rows", stream, n);
    launch_quantize(type, p, 1, stream);
}

void check_cache(const elips_b200_cache& c) {
    if (c.parts < 1 || c.parts > 2) bad("a cache has one or two parts");
    if (c.pages < 0 || c.page_size < 1 || c.heads < 1 || c.dim < 1) bad("cache sizes must be positive");
    if (c.dim > static_cast<int64_t>(kMaxDim) || c.heads > (1 << 20) || c.parts * c.heads * c.dim > (1 << 30))
        bad("cache rows too wide");
    if (c.page_size > 0x7FFFFFFFll || c.pages > 0x7FFFFFFFll || c.pages * c.page_size > 0x7FFFFFFFll)
        bad("a cache holds fewer than 2^31 slots");
    if (c.pages > 0 && (c.codes == nullptr || c.scales == nullptr)) bad("cache without storage");
}

void check_cache_rows(const elips_b200_cache& c, const elips_b200_rows* rows, int type, size_t t) {
    check_float_type(type);
    if (t > kMaxRows) bad("too many rows in one call");
    for (int64_t i = 0; t > 0 && i < c.parts; ++i)
        if (rows[i].data == nullptr) bad("rows missing");
}

// The cache with 0 for the strides of axes of one entry, which address nothing.
elips_b200_cache plain_strides(elips_b200_cache c) {
    const int64_t sizes[4] = {c.parts, c.pages, c.page_size, c.heads};
    for (int i = 0; i < 4; ++i)
        if (sizes[i] == 1) c.code_strides[i] = c.scale_strides[i] = 0;
    return c;
}

template <class P>
void set_cache(P& p, const elips_b200_cache& c) {
    p.codes = static_cast<int8_t*>(c.codes);
    p.scales = c.scales;
    p.code_part = c.code_strides[0];
    p.code_page = c.code_strides[1];
    p.code_row = c.code_strides[2];
    p.code_head = c.code_strides[3];
    p.scale_part = c.scale_strides[0];
    p.scale_page = c.scale_strides[1];
    p.scale_row = c.scale_strides[2];
    p.scale_head = c.scale_strides[3];
    p.by_heads = FastDiv(static_cast<uint32_t>(c.heads));
    p.page = FastDiv(static_cast<uint32_t>(c.page_size));
}

void cache_write(const elips_b200_cache& given, const elips_b200_rows* rows, int type, size_t t, const void* slots,
                 int slots64, cudaStream_t stream) {
    const elips_b200_cache c = plain_strides(given);
    if (t == 0 || c.pages == 0) return;
    QuantParams p{};
    set_cache(p, c);
    for (int64_t i = 0; i < c.parts; ++i) {
        p.x[i] = rows[i].data;
        p.x_stride_t[i] = t > 1 ? rows[i].stride_row : 0;
        p.x_stride_h[i] = c.heads > 1 ? rows[i].stride_head : 0;
    }
    p.slots = slots;
    p.slots64 = slots64;
    p.t = static_cast<uint32_t>(t);
    p.heads = static_cast<uint32_t>(c.heads);
    p.d = static_cast<uint32_t>(c.dim);
    p.num_slots = c.pages * c.page_size;
    const uint32_t parts = static_cast<uint32_t>(c.parts);
    p.per_t = FastDiv(parts * p.heads);
    p.dup = t == 1 ? kDupNone : t <= kDupScanRows ? kDupScan : kDupClaim;
    const uint64_t items = static_cast<uint64_t>(t) * p.per_t.d;
    if (p.dup == kDupClaim) {
        Profiler::Scope prof("cache_claim", stream, items);
        in_runs(t, p.per_t.d, [&](uint32_t t0, uint32_t groups) {
            p.t0 = t0;
            p.groups = groups;
            LaunchConfig cfg(dim3(blocks_for(groups, 256)), 256, 0, stream);
            cfg.launch(cache_claim_kernel, p);
        });
        launch_ok("cache claim launch");
    }
    Profiler::Scope prof("cache_write", stream, items);
    launch_quantize(type, p, parts, stream);
}

// The most codes per access (a power of two, at most 16 bytes of output) that
// the sizes and strides of a read allow.
template <class T>
uint32_t read_width(const ReadParams& p, const elips_b200_cache& c) {
    uint64_t bits = static_cast<uint64_t>(c.dim) | reinterpret_cast<uintptr_t>(c.codes);
    for (int i = 0; i < 4; ++i) bits |= static_cast<uint64_t>(c.code_strides[i]);
    for (int64_t i = 0; i < c.parts; ++i) {
        bits |= static_cast<uint64_t>(p.out_stride_t[i] | p.out_stride_h[i]);
        bits |= reinterpret_cast<uintptr_t>(p.out[i]) / sizeof(T);
    }
    uint32_t v = 16 / sizeof(T);
    while (bits % v != 0) v /= 2;
    return v;
}

template <class T, int V>
void launch_read(ReadParams p, const elips_b200_cache& c, int num_sms, cudaStream_t stream) {
    p.per_group = FastDiv(static_cast<uint32_t>(c.dim) / V);
    p.per_row = static_cast<uint32_t>(c.parts * c.heads) * p.per_group.d;
    // A thread per access of a row, up to 256, and as many rows side by side as
    // leave the fewest threads of the last warp idle.
    p.nx = std::min(p.per_row, 256u);
    p.ny = 1;
    uint32_t threads = cdiv(p.nx, 32) * 32;
    for (uint32_t ny = 2; ny * p.nx <= 288; ++ny) {
        const uint32_t with = cdiv(ny * p.nx, 32) * 32;
        if (with < 128 || static_cast<uint64_t>(ny * p.nx) * threads >= static_cast<uint64_t>(p.ny * p.nx) * with) p.ny = ny, threads = with;
    }
    // Two batches of accesses a thread, the columns of wide rows in different
    // blocks. Fewer rows make four blocks an SM as long as that leaves a thread
    // three accesses, and one block an SM after that.
    const uint32_t shares = std::min(cdiv(p.per_row, p.nx), 65535u);
    const uint64_t work = static_cast<uint64_t>(p.total) * shares, sms = static_cast<uint32_t>(num_sms);
    uint64_t rows = std::max(cdiv(work, 4 * sms), std::min(3u * p.ny, cdiv(work, sms)));
    rows = std::min<uint64_t>(rows, std::min<uint64_t>(kReadRows, 2u * kReadBatch * p.ny));
    p.rows = static_cast<uint32_t>(rows);
    threads = std::max(threads, cdiv(p.rows, 32) * 32);
    LaunchConfig cfg(dim3(blocks_for(p.total, p.rows), shares), threads, 0, stream);
    cfg.launch(cache_read_kernel<T, V>, p);
}

// Whether the outputs are runs of values that start on 16 bytes, of rows no
// narrower than a store, and rows of codes start on as many bytes.
template <class T>
bool without_gaps(const ReadParams& p, const elips_b200_cache& c) {
    constexpr uint64_t V = 16 / sizeof(T);
    uint64_t codes = reinterpret_cast<uintptr_t>(c.codes);
    for (int i = 0; i < 4; ++i) codes |= static_cast<uint64_t>(c.code_strides[i]);
    if (codes % V != 0 || c.dim < static_cast<int64_t>(V) || c.heads * c.dim > (1 << 20)) return false;
    for (int64_t i = 0; i < c.parts; ++i) {
        if (reinterpret_cast<uintptr_t>(p.out[i]) % 16 != 0) return false;
        if (p.total > 1 && p.out_stride_t[i] != c.heads * c.dim) return false;
        if (c.heads > 1 && p.out_stride_h[i] != c.dim) return false;
    }
    return true;
}

template <class T>
void launch_read_flat(ReadParams p, const elips_b200_cache& c, int num_sms, cudaStream_t stream) {
    p.per_group = FastDiv(static_cast<uint32_t>(c.dim));
    // Rows in multiples of eight, so that every block starts on 16 bytes: two
    // stores a thread, four blocks an SM.
    const uint64_t row = static_cast<uint64_t>(c.heads * c.dim);
    uint64_t rows = std::max<uint64_t>(1, 512 * (16 / sizeof(T)) / row);
    rows = std::min<uint64_t>(rows, cdiv(static_cast<uint64_t>(p.total) * static_cast<uint64_t>(c.parts), 4u * static_cast<uint32_t>(num_sms)));
    p.rows = static_cast<uint32_t>(std::min<uint64_t>(kReadRows, (rows + 7) / 8 * 8));
    LaunchConfig cfg(dim3(blocks_for(p.total, p.rows), static_cast<uint32_t>(c.parts)), 256, 0, stream);
    cfg.launch(cache_read_flat_kernel<T>, p);
}

void cache_read(int num_sms, const elips_b200_cache& given, const elips_b200_sequences& q, const elips_b200_rows* out,
                int type, int zero_behind, cudaStream_t stream) {
    const elips_b200_cache c = plain_strides(given);
    if (q.total == 0) return;
    const size_t total = static_cast<size_t>(q.total);
    ReadParams p{};
    set_cache(p, c);
    for (int64_t i = 0; i < c.parts; ++i) {
        p.out[i] = const_cast<void*>(out[i].data);
        p.out_stride_t[i] = total > 1 ? out[i].stride_row : 0;
        p.out_stride_h[i] = c.heads > 1 ? out[i].stride_head : 0;
    }
    p.table = q.page_table;
    p.table64 = q.table_64bit;
    p.table_stride = q.table_stride;
    p.offsets = q.offsets;
    p.offsets64 = q.offsets_64bit;
    p.sequences = static_cast<uint32_t>(q.sequences);
    p.table_width = static_cast<uint32_t>(q.table_width);
    p.pages = static_cast<uint32_t>(c.pages);
    p.total = static_cast<uint32_t>(total);
    p.zero_behind = zero_behind;
    Profiler::Scope prof("cache_read", stream, static_cast<uint64_t>(total) * static_cast<uint64_t>(c.parts * c.heads));
    with_float_type(type, [&](auto tag) {
        using T = decltype(tag);
        const uint32_t v = read_width<T>(p, c);
        if (v <= 2 && v < 16 / sizeof(T) && without_gaps<T>(p, c)) return launch_read_flat<T>(p, c, num_sms, stream);
        if constexpr (sizeof(T) == 2) {
            if (v == 8) return launch_read<T, 8>(p, c, num_sms, stream);
        }
        if (v >= 4) launch_read<T, 4>(p, c, num_sms, stream);
        else if (v == 2) launch_read<T, 2>(p, c, num_sms, stream);
        else launch_read<T, 1>(p, c, num_sms, stream);
    });
    launch_ok("cache read launch");
}

bool on_16(const void* ptr, int64_t pitch_bytes, uint32_t rows) {
    return reinterpret_cast<uintptr_t>(ptr) % 16 == 0 && (rows <= 1 || pitch_bytes % 16 == 0);
}

// What a tensor map needs of a pitch that no row uses.
uint64_t map_pitch(int64_t pitch_bytes, uint64_t width_bytes, uint32_t rows) {
    return rows > 1 ? static_cast<uint64_t>(pitch_bytes) : (width_bytes + 15) / 16 * 16;
}

CUtensorMap code_map(const int8_t* codes, int64_t pitch, uint32_t rows, uint32_t k, uint32_t box_rows) {
    if (k == 0) return CUtensorMap{};  // nothing is loaded
    return make_operand_map(codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, k, rows, box_rows, map_pitch(pitch, k, rows));
}

template <int MR, class X, class T>
void launch_dot_rows(const GemmParams& p, int num_sms, cudaStream_t stream) {
    // Warps that split k between them until every SM has sixteen.
    const uint64_t groups = cdiv(p.n, kDotChannels);
    uint32_t wk = 1;
    while (wk < 8 && groups * wk < static_cast<uint64_t>(num_sms) * 16 && p.k > wk * 512u) wk *= 2;
    // Blocks that quantise their rows are spread over the SMs only by a plain
    // launch (1 x 4096 x 4096 after another, weights in L2: 4.4 us, early 5.3).
    constexpr bool codes = std::is_same<X, int8_t>::value;
    const size_t smem = codes ? 0 : static_cast<size_t>(p.m) * ((p.k + 15u) / 16u * 16u);
    LaunchConfig cfg(dim3(blocks_for(groups * wk, 8)), 256, smem, stream, codes);
    cfg.launch(gemm_int8_dot_kernel<MR, X, T>, p, wk);
    launch_ok("int8 product launch");
}

template <class X, class T>
void launch_dot(const GemmParams& p, int num_sms, cudaStream_t stream) {
    if (p.m == 1) launch_dot_rows<1, X, T>(p, num_sms, stream);
    else if (p.m == 2) launch_dot_rows<2, X, T>(p, num_sms, stream);
    else if (p.m <= 4) launch_dot_rows<4, X, T>(p, num_sms, stream);
    else launch_dot_rows<8, X, T>(p, num_sms, stream);
}

template <int BT, int S, class T>
void launch_wide_split(const GemmParams& p, int num_sms, cudaStream_t stream) {
    constexpr uint32_t stage_bytes = (kWideChannels + BT) * kGemmStageK;
    const uint32_t n_rt = cdiv(p.m, BT);
    const uint64_t all = static_cast<uint64_t>(cdiv(p.n, kWideChannels)) * n_rt;
    if (all > 0x7FFFFFFFull / S) bad("too many rows in one call");
    const uint32_t tiles = static_cast<uint32_t>(all), kblocks = cdiv(p.k, kGemmStageK);
    // A CTA has an SM to itself and keeps as much of k in flight as fits. Where
    // there are more tiles than SMs two share one, for eight warps to store what
    // the loads bring (64 x 100,000 x 384 to fp32: 17.8 us with one, 14.5 with
    // two); clusters of eight find room on every GPC only at two to an SM.
    const bool two = S == 8 || (S == 1 && tiles > static_cast<uint32_t>(num_sms));
    uint32_t stages = (two ? 111000u : 196608u) / stage_bytes;
    if (S > 1 || !two) stages = std::min(stages, std::max(1u, cdiv(kblocks, S)));
    stages = std::min<uint32_t>(stages, kWideMaxStages);
    const size_t smem = 1024 + std::max<size_t>(static_cast<size_t>(stages) * stage_bytes, S > 1 ? BT * kWideChannels * 4u : 0u);
    const CUtensorMap mw = code_map(p.b, p.b_pitch, p.n, p.k, kWideChannels);
    const CUtensorMap mx = code_map(p.a, p.a_pitch, p.m, p.k, BT);
    allow_dynamic_smem(reinterpret_cast<const void*>(gemm_int8_wide_kernel<BT, S, T>), smem);
    const uint32_t ctas = S == 1 ? std::min<uint32_t>(tiles, static_cast<uint32_t>(num_sms) * (two ? 2u : 1u)) : tiles * S;
    LaunchConfig cfg(dim3(ctas), kWideThreads, smem, stream);
    if (S > 1) cfg.clusters_of(S);
    cfg.launch(gemm_int8_wide_kernel<BT, S, T>, mw, mx, p, stages, n_rt, tiles);
}

template <int BT, class T>
void launch_wide(const GemmParams& p, int num_sms, uint32_t splits, cudaStream_t stream) {
    if (splits == 1) launch_wide_split<BT, 1, T>(p, num_sms, stream);
    else if (splits == 2) launch_wide_split<BT, 2, T>(p, num_sms, stream);
    else if (splits == 4) launch_wide_split<BT, 4, T>(p, num_sms, stream);
    else launch_wide_split<BT, 8, T>(p, num_sms, stream);
}

template <class T>
void launch_pair(const GemmParams& p, int num_sms, cudaStream_t stream) {
    const uint32_t n_mt = cdiv(p.m, kPairM), n_nt = cdiv(p.n, kPairN);
    if (static_cast<uint64_t>(n_mt) * n_nt > 0x3FFFFFFFull) bad("too many rows in one call");
    const CUtensorMap ma = code_map(p.a, p.a_pitch, p.m, p.k, kPairM / 2);
    const CUtensorMap mb = code_map(p.b, p.b_pitch, p.n, p.k, kPairN / 4);
    constexpr uint32_t smem = kPairSmemBytes;
    allow_dynamic_smem(reinterpret_cast<const void*>(gemm_int8_pair_kernel<T>), smem);
    const uint32_t all = static_cast<uint32_t>(num_sms) / 2, tiles = n_mt * n_nt, last = tiles % all;
    const uint32_t whole = 2 * last <= all ? tiles - last : tiles, units = whole + 2 * (tiles - whole);
    const uint32_t pairs = std::min(units, all);
    LaunchConfig cfg(dim3(pairs * 2), kPairThreads, smem, stream);
    cfg.clusters_of(2);
    cfg.launch(gemm_int8_pair_kernel<T>, ma, mb, p, n_mt, n_nt, whole, units);
}

// The form a product takes: rows per tile of the wide kernel (0: the pair
// kernel, 1: the dot kernel) and how many CTAs split k.
struct GemmForm {
    uint32_t rows = 0, splits = 1;
};

// The dot kernel is for single tokens. A warp takes four channels whatever k
// is, so what it spends on each counts where there are many (us on the device,
// to bf16, dot kernel / wide kernel with its best split):
//   1 row:  4096 x 4096 4.4 / 6.7, 8192 x 8192 13.0 / 14.4, 40,000 x 4096 28.4 /
//           29.7, 10,000 x 768 2.9 / 3.8, 50,000 x 1024 10.5 / 11.1, 60,000 x
//           1024 12.3 / 12.2, 100,000 x 768 16.3 / 14.6, 100,000 x 128 9.1 / 5.5,
//           1,000,000 x 128 79 / 33
//   2 rows: 4096 x 4096 5.3 / 6.8, 8192 x 4096 8.7 / 9.3, 10,000 x 768 3.8 / 3.7
//           (rows of floats 3.8 / 5.3), 16,000 x 4096 14.0 / 12.9, 100,000 x 768
//           21.8 / 14.8, 1,000,000 x 128 108 / 34
// From three rows on its dp4a takes over from the loads at about 2^25 products:
// 4 x 2048 x 2048 2.7 / 4.6, 8 x 1024 x 1024 2.7 / 3.8, 4 x 4096 x 4096 7.2 / 6.8,
// 8 x 4096 x 4096 8.5 / 6.9, 4 x 10,000 x 768 4.3 / 3.7.
bool dot_form(uint32_t m, uint32_t n, uint32_t k) {
    if (k == 0 || m > 8) return false;
    if (m == 1 && n <= uint64_t{52} * k) return true;
    if (m <= 2) return n <= 12288;
    return n <= 8192 && static_cast<uint64_t>(m) * n * k <= (1u << 25);
}

// Between the others the least time that a simple model gives, in us, from what
// was measured over sizes from 16 x 1024 x 1024 to 8192^3:
//  * wide: 4 for the launch and its ends; a CTA loads 127 KB/us, four fifths
//    of that when all SMs do; a cluster's summing costs 0.35 and 0.0145 a row.
//    With more tiles than SMs, each takes 0.2 and its loads or, if longer, its
//    stores (0.02 a row, a quarter more to fp32).
//  * pair: 4.5 for the launch and its ends, then waves of tiles at 0.36 per
//    128 of k (1670 T products/s, the tensor cores' pace at this power) + 1.2,
//    2.4 at least, 0.8 more to fp32; 0.7 of that for a last wave of half tiles.
// Measured on both sides (wide of 128 rows or as named / pair): 512 x 4096 x 4096
// 11.8 / 12.5, 1024 x 4096 x 4096 18.6 / 16.2, 64 x 100,000 x 384 to fp32 14.0 (64
// rows) / 20.7, 10,000 x 1536 x 768 21.8 / 14.7, to fp32 22.4 / 18.4.
GemmForm gemm_form(uint32_t m, uint32_t n, uint32_t k, bool fp32, int num_sms) {
    if (dot_form(m, n, k)) return {1, 1};
    const uint32_t kb = cdiv(k, kGemmStageK);
    const double sms = num_sms;
    GemmForm best{0, 1};
    double least = 1e30;
    if (kb > 0) {
        const uint64_t pairs = num_sms / 2, tiles = static_cast<uint64_t>(cdiv(m, kPairM)) * cdiv(n, kPairN);
        const double last = tiles % pairs == 0 ? 0 : 2 * (tiles % pairs) <= pairs ? 0.7 : 1;
        const double each = std::max(kb * 0.36 + 1.2, 2.4) + (fp32 ? 0.8 : 0);
        least = 4.5 + (static_cast<double>(tiles / pairs) + last) * each;
    }
    for (uint32_t rows = 16; rows <= 128; rows *= 2) {
        const uint64_t tiles = static_cast<uint64_t>(cdiv(n, kWideChannels)) * cdiv(m, rows);
        const double per_kb = (kWideChannels + rows) * kGemmStageK / 127e3;
        for (uint32_t splits = 1; splits <= 8; splits *= 2) {
            if (splits > 1 && (tiles * splits > static_cast<uint64_t>(num_sms) || splits > kb)) break;
            const double each = cdiv(kb, splits) * per_kb;
            const double us = tiles <= static_cast<uint64_t>(num_sms)
                                  ? 4 + each + (splits > 1 ? 0.35 + 0.0145 * rows : 0)
                                  : 4 + tiles / sms * (0.2 + std::max(1.25 * each, (fp32 ? 0.025 : 0.02) * rows));
            if (us < least) least = us, best = {rows, splits};
        }
        if (rows >= m) break;
    }
    return best;
}

template <class T>
void launch_gemm(const GemmParams& p, int num_sms, cudaStream_t stream) {
    const GemmForm f = gemm_form(p.m, p.n, p.k, sizeof(T) == 4, num_sms);
    if (f.rows == 0) launch_pair<T>(p, num_sms, stream);
    else if (f.rows == 1) launch_dot<int8_t, T>(p, num_sms, stream);
    else if (f.rows == 16) launch_wide<16, T>(p, num_sms, f.splits, stream);
    else if (f.rows == 32) launch_wide<32, T>(p, num_sms, f.splits, stream);
    else if (f.rows == 64) launch_wide<64, T>(p, num_sms, f.splits, stream);
    else launch_wide<128, T>(p, num_sms, f.splits, stream);
    launch_ok("int8 product launch");
}

void gemm_int8(int num_sms, GemmParams p, int out_type, cudaStream_t stream) {
    if (p.m == 0 || p.n == 0) return;
    // Operands whose rows do not start on 16 bytes are copied to rows that do:
    // one more pass over them.
    const bool a_ok = on_16(p.a, p.a_pitch, p.m), b_ok = on_16(p.b, p.b_pitch, p.n);
    const size_t pitch = (static_cast<size_t>(p.k) + 15) / 16 * 16;
    const size_t a_bytes = a_ok ? 0 : (p.m * pitch + 255) / 256 * 256, b_bytes = b_ok ? 0 : p.n * pitch;
    auto product = [&] {
        Profiler::Scope prof("gemm_int8", stream, static_cast<uint64_t>(p.m) * p.n);
        with_float_type(out_type, [&](auto tag) { launch_gemm<decltype(tag)>(p, num_sms, stream); });
    };
    if ((a_ok && b_ok) || p.k == 0) {
        product();
        return;
    }
    StreamScratch s(a_bytes + b_bytes, stream);
    {
        Profiler::Scope prof("repack_codes", stream, (a_ok ? 0u : p.m) + static_cast<uint64_t>(b_ok ? 0u : p.n));
        RepackParams r{};
        r.k = p.k;
        r.words = FastDiv(static_cast<uint32_t>(pitch / 4));
        uint32_t count = 0;
        uint64_t most = 0;
        auto add = [&](const int8_t*& codes, int64_t& from, uint32_t rows, uint8_t* to) {
            r.in[count] = codes;
            r.in_pitch[count] = from;
            r.rows[count] = rows;
            r.out[count] = reinterpret_cast<int8_t*>(to);
            most = std::max<uint64_t>(most, rows * (pitch / 4));
            codes = r.out[count++];
            from = static_cast<int64_t>(pitch);
        };
        if (!a_ok) add(p.a, p.a_pitch, p.m, s.get());
        if (!b_ok) add(p.b, p.b_pitch, p.n, s.get() + a_bytes);
        const uint32_t blocks = static_cast<uint32_t>(std::min<uint64_t>((most + 255) / 256, 1u << 20));
        LaunchConfig cfg(dim3(blocks, count), 256, 0, stream);
        cfg.launch(repack_codes_kernel, r);
        launch_ok("operand copy launch");
    }
    product();
}

// Runs of `width` bytes, one at each combination of up to four axes' steps.
struct Region {
    using Wide = __int128;  // no product of a size and a stride passes it
    uintptr_t base = 0;     // of the lowest run
    int64_t width = 0;
    int64_t count[4] = {1, 1, 1, 1};
    Wide step[4] = {};
    Wide all = 0;           // bytes from the first to behind the last of the runs
    // The same without the axes whose step is a multiple of `whole`.
    Wide extent(Wide whole) const {
        Wide e = width;
        for (int i = 0; i < 4; ++i)
            if (step[i] % whole != 0) e += (count[i] - 1) * step[i];
        return e;
    }
};

struct Axis {
    int64_t count;
    Region::Wide step;  // bytes
};

Region region(const void* p, int64_t width, std::initializer_list<Axis> axes) {
    Region r;
    r.width = r.all = width;
    Region::Wide base = reinterpret_cast<uintptr_t>(p);
    int i = 0;
    for (const Axis& a : axes) {
        if (a.count <= 0) r.width = 0;
        if (a.count > 1) {
            r.count[i] = a.count;
            r.step[i] = a.step < 0 ? -a.step : a.step;
            r.all += (a.count - 1) * r.step[i];
            if (a.step < 0) base += (a.count - 1) * a.step;
        }
        ++i;
    }
    r.base = static_cast<uintptr_t>(base);
    return r;
}

// Whether two regions share a byte. They do not where one ends before the
// other starts, or where for some step S all bytes of one are, modulo S, before
// or behind those of the other: columns side by side in one buffer, parts or
// heads that take turns, codes and scales of each page one after the other.
// Layouts that interlace in no such way are taken to share one.
bool overlap(const Region& a, const Region& b) {
    using Wide = Region::Wide;
    if (a.width <= 0 || b.width <= 0) return false;
    const Wide from_a = static_cast<Wide>(b.base) - static_cast<Wide>(a.base);
    if (from_a >= a.all || -from_a >= b.all) return false;
    for (int i = 0; i < 8; ++i) {
        const Wide s = i < 4 ? a.step[i] : b.step[i - 4];
        if (s <= 0) continue;
        const Wide ea = a.extent(s), eb = b.extent(s), ahead = (from_a % s + s) % s;
        if (ahead >= ea && ahead + eb <= s) return false;
    }
    return true;
}

int64_t type_bytes(int type) {
    return type == ELIPS_B200_PRECISION_INT8 ? 1 : type == ELIPS_B200_PRECISION_FP32 ? 4 : 2;
}

// The forms differ in what they have read when they first write (the dot
// kernel's blocks each read every row), so no output may lie on an input.
void check_gemm_apart(const elips_b200_gemm& g) {
    const int64_t a = type_bytes(g.a_type), o = type_bytes(g.out_type);
    const Region out = region(g.out, g.n * o, {{g.m, Region::Wide{g.out_stride} * o}});
    if (overlap(out, region(g.a, g.k * a, {{g.m, Region::Wide{g.a_stride} * a}})) ||
        overlap(out, region(g.b, g.k, {{g.n, g.b_stride}})) || overlap(out, region(g.b_scales, g.n * 4, {})) ||
        (g.a_type == ELIPS_B200_PRECISION_INT8 && overlap(out, region(g.a_scales, g.m * 4, {}))) ||
        (g.bias != nullptr && overlap(out, region(g.bias, g.n * type_bytes(g.bias_type), {}))))
        bad("the output shares memory with an input");
}

Region codes_region(const elips_b200_cache& c) {
    const int64_t* s = c.code_strides;
    return region(c.codes, c.dim, {{c.parts, s[0]}, {c.pages, s[1]}, {c.page_size, s[2]}, {c.heads, s[3]}});
}

Region scales_region(const elips_b200_cache& c) {
    Region::Wide s[4];
    for (int i = 0; i < 4; ++i) s[i] = Region::Wide{c.scale_strides[i]} * 4;
    return region(c.scales, 4, {{c.parts, s[0]}, {c.pages, s[1]}, {c.page_size, s[2]}, {c.heads, s[3]}});
}

Region rows_region(const elips_b200_cache& c, const elips_b200_rows& r, size_t t, int type) {
    const int64_t bytes = type_bytes(type);
    return region(r.data, c.dim * bytes, {{static_cast<int64_t>(t), Region::Wide{r.stride_row} * bytes},
                                          {c.heads, Region::Wide{r.stride_head} * bytes}});
}

// Claims overwrite scale words, and rows their codes, before other rows and
// slots have been read.
void check_write_apart(const elips_b200_cache& c, const elips_b200_rows* rows, int type, size_t t, const void* slots,
                       int slots64) {
    if (t == 0 || c.pages == 0) return;
    const Region codes = codes_region(c), scales = scales_region(c);
    const Region list = region(slots, static_cast<int64_t>(t) * (slots64 ? 8 : 4), {});
    bool shared = overlap(codes, scales) || overlap(list, codes) || overlap(list, scales);
    for (int64_t i = 0; i < c.parts; ++i) {
        const Region x = rows_region(c, rows[i], t, type);
        shared = shared || overlap(x, codes) || overlap(x, scales);
    }
    if (shared) bad("the cache shares memory with the rows or slots, or its codes with its scales");
}

void check_read_apart(const elips_b200_cache& c, const elips_b200_sequences& q, const elips_b200_rows* out, int type) {
    if (q.total == 0) return;
    const size_t total = static_cast<size_t>(q.total);
    const int64_t entry = q.table_64bit ? 8 : 4, columns = q.sequences > 0 ? q.table_width : 0;
    const Region inputs[4] = {c.pages > 0 ? codes_region(c) : Region{}, c.pages > 0 ? scales_region(c) : Region{},
                              region(q.page_table, columns * entry, {{q.sequences, Region::Wide{q.table_stride} * entry}}),
                              region(q.offsets, q.sequences > 0 ? (q.sequences + 1) * (q.offsets_64bit ? 8 : 4) : 0, {})};
    bool shared = c.parts == 2 && overlap(rows_region(c, out[0], total, type), rows_region(c, out[1], total, type));
    for (int64_t i = 0; i < c.parts; ++i) {
        const Region x = rows_region(c, out[i], total, type);
        for (const Region& in : inputs) shared = shared || overlap(x, in);
    }
    if (shared) bad("an output shares memory with what is read or with the other part's output");
}

void check_gemm(const elips_b200_gemm& g) {
    check_float_type(g.out_type);
    if (g.bias != nullptr) check_float_type(g.bias_type);
    const bool codes = g.a_type == ELIPS_B200_PRECISION_INT8;
    if (!codes) check_float_type(g.a_type);
    if (g.m < 0 || g.n < 0 || g.k < 0 || g.m > static_cast<int64_t>(kMaxRows) || g.n > static_cast<int64_t>(kMaxRows))
        bad("matrix sizes must be below 2^31");
    if (g.k > static_cast<int64_t>(kMaxK)) bad("k must be below 2^17: the int32 sum could overflow");
    if (!codes && g.k == 0) bad("rows to quantise must have a value");
    if (g.b_stride < g.k || g.out_stride < g.n || (codes && g.a_stride < g.k)) bad("neighbouring matrix rows overlap");
    if (g.m == 0 || g.n == 0) return;
    if (g.b_scales == nullptr || g.out == nullptr || (codes && g.a_scales == nullptr)) bad("operand missing");
    if (g.k > 0 && (g.a == nullptr || g.b == nullptr)) bad("operand missing");
    check_gemm_apart(g);
}

GemmParams gemm_params(const elips_b200_gemm& g) {
    GemmParams p{};
    p.a = static_cast<const int8_t*>(g.a);
    p.a_scales = g.a_scales;
    p.a_pitch = g.a_stride;
    p.b = g.b;
    p.b_pitch = g.b_stride;
    p.b_scales = g.b_scales;
    p.bias = g.bias;
    p.bias_type = g.bias_type;
    p.out = g.out;
    p.out_pitch = g.out_stride;
    p.m = static_cast<uint32_t>(g.m);
    p.n = static_cast<uint32_t>(g.n);
    p.k = static_cast<uint32_t>(g.k);
    const int64_t size = g.out_type == ELIPS_B200_PRECISION_FP32 ? 4 : 2;
    p.out_vec4 = reinterpret_cast<uintptr_t>(g.out) % (4 * size) == 0 && (p.m <= 1 || g.out_stride % 4 == 0);
    p.out_vec16 = on_16(g.out, g.out_stride * size, p.m);
    return p;
}

// The product over rows that are not quantised yet.
void linear_int8(int num_sms, const elips_b200_gemm& g, cudaStream_t stream) {
    GemmParams p = gemm_params(g);
    const size_t pitch = (static_cast<size_t>(p.k) + 15) / 16 * 16;
    // Few values: the dot kernel quantises them itself.
    if (gemm_form(p.m, p.n, p.k, g.out_type == ELIPS_B200_PRECISION_FP32, num_sms).rows == 1 &&
        p.m * pitch <= kDotCodeBytes && on_16(p.b, p.b_pitch, p.n)) {
        p.x = g.a;
        p.x_pitch = p.m > 1 ? g.a_stride : 0;
        Profiler::Scope prof("linear_int8", stream, static_cast<uint64_t>(p.m) * p.n);
        with_float_type(g.a_type, [&](auto xt) {
            using X = decltype(xt);
            p.x_vec16 = on_16(g.a, g.a_stride * static_cast<int64_t>(sizeof(X)), p.m) && p.k % (16 / sizeof(X)) == 0;
            with_float_type(g.out_type, [&](auto tag) { launch_dot<X, decltype(tag)>(p, num_sms, stream); });
        });
        return;
    }
    const size_t code_bytes = (p.m * pitch + 255) / 256 * 256;
    StreamScratch s(code_bytes + p.m * sizeof(float), stream);
    int8_t* codes = reinterpret_cast<int8_t*>(s.get());
    float* scales = reinterpret_cast<float*>(s.get() + code_bytes);
    quantize_rows(g.a, g.a_type, p.m, p.k, g.a_stride, codes, pitch, scales, stream);
    p.a = codes;
    p.a_pitch = static_cast<int64_t>(pitch);
    p.a_scales = scales;
    gemm_int8(num_sms, p, g.out_type, stream);
}

cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

}  // namespace

void int8_wait_selftest(int device, long long budget) {
    if (budget < 1 || budget > kWaitTimeoutCycles) bad("wait budget must be in [1, 2^31] cycles");
    DeviceGuard g(device);
    device_props(device);
    wait_selftest_kernel<<<1, 32>>>(budget);
    launch_ok("wait self-test launch");
    check_cuda(cudaDeviceSynchronize(), ELIPS_B200_KERNEL_LAUNCH_FAILED, "wait self-test");
}

int take_int8_error(int device) {
    DeviceGuard g(device);
    int code = 0;
    check_cuda(cudaMemcpyFromSymbol(&code, g_device_error, sizeof(int)), ELIPS_B200_TRANSFER_FAILED, "read device error");
    if (code != 0) {
        const int zero = 0;
        check_cuda(cudaMemcpyToSymbol(g_device_error, &zero, sizeof(int)), ELIPS_B200_TRANSFER_FAILED,
                   "clear device error");
    }
    return code;
}

}  // namespace eb

using eb::guarded;

extern "C" {

int elips_b200_int8_wait_selftest(int device, uint64_t cycles) {
    return guarded([&] { eb::int8_wait_selftest(device, static_cast<long long>(cycles)); });
}

int elips_b200_quantize_rows(int device, const void* x, int type, size_t n, size_t d, int64_t x_stride, int8_t* codes,
                             size_t code_stride, float* scales, void* stream) {
    if (n > 0 && (x == nullptr || codes == nullptr || scales == nullptr)) return ELIPS_B200_INVALID_ARGUMENT;
    return guarded([&] {
        eb::check_rows(n, d, type);
        if (code_stride < d) eb::bad("codes of neighbouring rows overlap");
        const int64_t rows = static_cast<int64_t>(n), width = static_cast<int64_t>(d), bytes = eb::type_bytes(type);
        const eb::Region in = eb::region(x, width * bytes, {{rows, eb::Region::Wide{x_stride} * bytes}});
        const eb::Region out = eb::region(codes, width, {{rows, static_cast<eb::Region::Wide>(code_stride)}});
        const eb::Region held = eb::region(scales, rows * 4, {});
        if (eb::overlap(in, out) || eb::overlap(in, held) || eb::overlap(out, held))
            eb::bad("rows, codes and scales share memory");
        eb::DeviceGuard g(device);
        eb::device_props(device);
        eb::quantize_rows(x, type, n, d, x_stride, codes, code_stride, scales, eb::as_stream(stream));
    });
}

int elips_b200_gemm_int8(int device, const elips_b200_gemm* args, void* stream) {
    if (args == nullptr) return ELIPS_B200_INVALID_ARGUMENT;
    return guarded([&] {
        eb::check_gemm(*args);
        if (args->m == 0 || args->n == 0) return;
        eb::DeviceGuard g(device);
        const int num_sms = eb::device_props(device).num_sms;
        if (args->a_type == ELIPS_B200_PRECISION_INT8)
            eb::gemm_int8(num_sms, eb::gemm_params(*args), args->out_type, eb::as_stream(stream));
        else
            eb::linear_int8(num_sms, *args, eb::as_stream(stream));
    });
}

int elips_b200_gemm_int8_form(int64_t m, int64_t n, int64_t k, int out_type, int num_sms, int* rows_out, int* splits_out) {
    if (rows_out == nullptr || splits_out == nullptr) return ELIPS_B200_INVALID_ARGUMENT;
    return guarded([&] {
        eb::check_float_type(out_type);
        const int64_t most = static_cast<int64_t>(eb::kMaxRows);
        if (m < 1 || n < 1 || k < 0 || m > most || n > most || k > static_cast<int64_t>(eb::kMaxK) || num_sms < 2)
            eb::bad("no such product");
        const eb::GemmForm f = eb::gemm_form(static_cast<uint32_t>(m), static_cast<uint32_t>(n), static_cast<uint32_t>(k),
                                             out_type == ELIPS_B200_PRECISION_FP32, num_sms);
        *rows_out = static_cast<int>(f.rows);
        *splits_out = static_cast<int>(f.splits);
    });
}

int elips_b200_cache_write(int device, const elips_b200_cache* cache, const elips_b200_rows* rows, int type, size_t t,
                           const void* slots, int slots_64bit, void* stream) {
    if (cache == nullptr || (t > 0 && rows == nullptr)) return ELIPS_B200_INVALID_ARGUMENT;
    return guarded([&] {
        eb::check_cache(*cache);
        eb::check_cache_rows(*cache, rows, type, t);
        if (t > 0 && slots == nullptr) eb::bad("slots missing");
        eb::check_write_apart(*cache, rows, type, t, slots, slots_64bit);
        eb::DeviceGuard g(device);
        eb::device_props(device);
        eb::cache_write(*cache, rows, type, t, slots, slots_64bit, eb::as_stream(stream));
    });
}

int elips_b200_cache_read(int device, const elips_b200_cache* cache, const elips_b200_sequences* sequences,
                          const elips_b200_rows* out, int type, int zero_behind, void* stream) {
    if (cache == nullptr || sequences == nullptr) return ELIPS_B200_INVALID_ARGUMENT;
    const elips_b200_sequences& q = *sequences;
    if (q.total < 0 || q.sequences < 0 || q.table_width < 0 || (q.total > 0 && out == nullptr))
        return ELIPS_B200_INVALID_ARGUMENT;
    return guarded([&] {
        eb::check_cache(*cache);
        eb::check_cache_rows(*cache, out, type, static_cast<size_t>(q.total));
        if (q.sequences > static_cast<int64_t>(eb::kMaxRows) || q.table_width > static_cast<int64_t>(eb::kMaxRows))
            eb::bad("page table too large");
        if (q.total > 0 && q.sequences > 0 && q.offsets == nullptr) eb::bad("offsets missing");
        if (q.total > 0 && q.sequences > 0 && q.table_width > 0 && q.page_table == nullptr) eb::bad("page table missing");
        eb::check_read_apart(*cache, q, out, type);
        eb::DeviceGuard g(device);
        eb::cache_read(eb::device_props(device).num_sms, *cache, q, out, type, zero_behind, eb::as_stream(stream));
    });
}

}  // extern "C"
