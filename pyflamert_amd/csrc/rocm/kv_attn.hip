// Attention over a paged key/value cache: a prefix that every request shares,
// and each request's own tokens up to the query's.  No counterpart in the
// reference.
#include <cmath>

#include "kv_attn.hpp"

#pragma clang fp contract(off)

namespace {

using pfr::attn::Args;
using pfr::attn::Kind;
using pfr::attn::kWaves;
using pfr::attn::kWideKeys;
using pfr::attn::kWideRows;

// A wave joins a row, where a launch of its own does that.
template <class QT>
__global__ __launch_bounds__(256) void k_kv_attn_join(Args a) {
    const int64_t rows = (int64_t)a.T * a.Hq, R = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (R >= rows) return;
    const int t = (int)(R / a.Hq);
    const bool own = a.whole || (a.B > 0 && t >= a.start[0] && t < a.start[a.B]);
    pfr::attn::join_row<QT, false>(a, R, t, a.p_splits + (own ? a.o_splits : 0));
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits of `keys` keys, each of `chunk` keys (a multiple of `round`), for
// about `want` of them, and at most kMaxParts.
constexpr int kMaxParts = 24;
void split_keys(int64_t want, int64_t round, int64_t keys, int32_t* splits, int32_t* chunk) {
    int64_t s = ceil_div(keys, round);
    s = want < s ? want : s;
    s = s > kMaxParts ? kMaxParts : s;
    const int64_t c = s > 0 ? ceil_div(ceil_div(keys, s), round) * round : round;
    *splits = (int32_t)(s > 0 ? ceil_div(keys, c) : 0);
    *chunk = (int32_t)c;
}

// Own keys of so many blocks at most go to a wave each: with one to a workgroup,
// 67 requests of one key, 32 heads, took 77 us, 36 so.
constexpr int kSoloBlocks = 8;
// And, of a 16-bit cache, up to so many keys where a CU's share is kSoloItems of one
// tile of rows each: the waves then stand in for each other, and none waits for
// the rest of its workgroup (200 requests, 32 heads, bf16, up to 301 keys: 151 us
// with a workgroup to each, 107 so; up to 501: 186, 169; up to 701: 223, 228;
// up to 1001: 291, 314.  300 requests of up to 301 keys in float32: 148, 154.
// With half as many items, 64 requests of up to 1024 keys: 144, 164).
constexpr int kSoloKeys = 512, kSoloItems = 16;
// Rows of a key head that the workgroups that come last join themselves; more
// take a launch, for that joins them side by side (14 rows of 24 parts: 87 us
// in the workgroups, 24 so; 4 rows of 5: 9 us, 12 so).
constexpr int kJoinRows = 8;
// And parts of a row that they join behind a launch of its own for the prefix
// (128 requests, 64 heads, 10 parts: 219 us, with a launch 214; 59 requests of
// one head, 24 parts: 44 us, 31; 118 requests, 12 heads, 2 parts: 23 us, 25).
constexpr int kJoinParts = 4;

// The kernels of a call and their workgroups; one launch where both parts take the same kernel.
struct Plan {
    Kind prefix = pfr::attn::kNarrow1, own = pfr::attn::kNarrow1;
    int64_t prefix_blocks = 0, own_blocks = 0;
};

// Which kernels, and how the work is cut into workgroups.
Plan plan(int num_cu, bool half, bool half_cache, int64_t max_added, int64_t max_length, int64_t room, Args& a) {
    using namespace pfr::attn;
    Plan p;
    const int64_t rows = (int64_t)a.T * a.G, own_rows = max_added * a.G;  // of a key head
    // Float32 rows go 16 to a wave however many they are: with 32 a wave's
    // registers leave one workgroup to a CU where two hide each other's loads
    // (64 requests, 8 heads of 96 for 64 of q, 2752 keys: 121 us with 32, 100 so).
    const auto kind = [&](int64_t n) { return half && a.D <= 128 && n > 16 ? (n > 32 ? kWide : kNarrow2) : kNarrow1; };
    const auto tile = [](Kind k) { return k == kWide ? kWideRows : (k == kNarrow2 ? 32 : 16); };
    const int64_t block = half ? kBlock<__bf16> : kBlock<float>, round = kWaves * block, wide_round = 4 * kWideKeys;

    p.own = kind(own_rows);
    a.whole = a.B > 0 && p.own == kWide && rows >= kWideRows * a.B && a.prefix_len + room < INT32_MAX - 4096;
    if (a.whole) {
        const int64_t tiles = rows / kWideRows + a.B + 2;
        a.o_tiles = (int32_t)ceil_div(own_rows, kWideRows);
        a.o_splits = 1;
        a.o_chunk = INT32_MAX;
        // Where a CU has few tiles, in equal shares of one workgroup a CU; with
        // many, a tile to a workgroup and no scratch.
        if (a.B + 2 <= kShareGroups && tiles * a.Hkv < 8 * num_cu) {
            p.own = kShares;
            a.shares = num_cu > a.Hkv ? num_cu / a.Hkv : 1;
            a.items = (int32_t)tiles;
            // parts as memory goes: 256 MB of them, at least three
            const int64_t parts = (int64_t(256) << 20) / ((int64_t)a.T * a.Hq * a.D * 4);
            a.parts = (int32_t)(parts < 3 ? 3 : (parts > kMaxParts ? kMaxParts : parts));
            p.own_blocks = (int64_t)a.shares * a.Hkv;
            return p;
        }
    } else {
        p.prefix = kind(rows);
        if (a.B > 0 && p.prefix != kWide && p.own != kWide) p.prefix = p.own = p.prefix > p.own ? p.prefix : p.own;
        a.p_tiles = (int32_t)ceil_div(rows, tile(p.prefix));
        a.o_tiles = a.B > 0 ? (int32_t)ceil_div(own_rows, tile(p.own)) : 0;
        const int64_t prefix_items = (int64_t)a.Hkv * a.p_tiles, own_items = (int64_t)a.Hkv * a.B * a.o_tiles;
        if (p.prefix != kWide && p.own != kWide) {
            // Chunks of one size, four workgroups to a CU if all requests were of
            // max_length; two with float32 rows, whose few keys a round and
            // longer start want more keys to a workgroup (8 requests, 32
            // heads of 128 behind 4096 keys, float32: 64 us with four, 58 so).
            const int64_t keys = prefix_items * a.prefix_len + own_items * max_length;
            const int64_t c = ceil_div(ceil_div(keys, (half ? 4 : 2) * num_cu), round) * round;
            split_keys(ceil_div(a.prefix_len, c), round, a.prefix_len, &a.p_splits, &a.p_chunk);
            split_keys(ceil_div(max_length, c), round, max_length, &a.o_splits, &a.o_chunk);
        } else {
            split_keys(ceil_div(num_cu, prefix_items), wide_round, a.prefix_len, &a.p_splits, &a.p_chunk);
            // one wide workgroup fills a CU; narrow ones eight to a CU, so that
            // requests of uneven lengths even out (128 requests of up to 2048
            // keys, 8 heads: 224 us with four, 220 so)
            if (a.B > 0)
                split_keys(ceil_div((p.own == kWide ? 1 : 8) * num_cu, own_items), p.own == kWide ? wide_round : round, max_length,
                           &a.o_splits, &a.o_chunk);
        }
        p.prefix_blocks = (int64_t)a.Hkv * a.p_tiles * a.p_splits;
        // a wave for a request's own keys where there are few of them and many requests, or very many of them
        const bool few = max_length <= kSoloBlocks * block && own_items >= 4 * num_cu;
        const bool many = half_cache && max_length <= kSoloKeys && a.o_tiles == 1 && own_items >= kSoloItems * num_cu;
        if (a.B > 0 && p.own != kWide && (few || many)) {
            a.solo = 1;
            split_keys(1, block, max_length, &a.o_splits, &a.o_chunk);
        }
    }
    if (a.B > 0) {
        const int64_t each = (int64_t)a.Hkv * (a.B + (a.whole ? 2 : 0)) * (a.o_splits > 0 ? a.o_splits : 1);
        while (a.o_tiles > 1 && each * a.o_tiles >= (1 << 22)) a.o_tiles = (a.o_tiles + 1) / 2;  // workgroups take several
        p.own_blocks = a.o_splits > 0 ? ceil_div(each * a.o_tiles, a.solo ? kWaves : 1) : 0;
    }
    return p;
}

__global__ void k_kv_attn_zero(uint32_t* p, int n) {
    const int i = (int)(blockIdx.x * blockDim.x + threadIdx.x);
    if (i < n) p[i] = 0;
}

// The context's zeros, and n arrival counters, which every launch leaves at zero, behind them.
constexpr int64_t kZeros = 256;
char* zeros(pfr_ctx* ctx, int64_t n) {
    const size_t had = ctx->scratch[8].bytes, want = (size_t)kZeros + (size_t)(n < 16384 ? 16384 : n) * sizeof(uint32_t);
    void* p = ctx->scratch[8].ensure(want);
    if (ctx->scratch[8].bytes != had) {
        const int words = (int)(ctx->scratch[8].bytes / sizeof(uint32_t));
        hipLaunchKernelGGL(k_kv_attn_zero, dim3((unsigned)ceil_div(words, 256)), dim3(256), 0, ctx->stream,
                           static_cast<uint32_t*>(p), words);
        PFR_HIP(hipGetLastError());
    }
    return static_cast<char*>(p);
}

void enqueue(pfr_ctx* ctx, const pfr_kv* kv, pfr_dtype dtype, const Args& a, Kind kind, int64_t blocks) {
    using pfr::attn::launch;
    if (blocks == 0) return;
    pfr::require(blocks < (1 << 24), "kv attention: extent too large");
    hipStream_t s = ctx->stream;
    if (dtype == PFR_BF16) launch<__bf16, __bf16>(s, a, kind, (unsigned)blocks);
    else if (dtype == PFR_F16) launch<_Float16, _Float16>(s, a, kind, (unsigned)blocks);
    else if (kv->dtype == PFR_BF16) launch<float, __bf16>(s, a, kind, (unsigned)blocks);
    else if (kv->dtype == PFR_F16) launch<float, _Float16>(s, a, kind, (unsigned)blocks);
    else launch<float, float>(s, a, kind, (unsigned)blocks);
}

void attention_dev(pfr_ctx* ctx, const pfr_kv* kv, const void* q, pfr_dtype dtype, int64_t T, int64_t heads, int64_t ldq,
                   float scale, const int32_t* prefix_table, int64_t prefix_len, const int32_t* table, int64_t table_w,
                   int64_t table_ld, int64_t B, const int32_t* lengths, const int32_t* start, int64_t max_added,
                   int64_t max_length, void* out, int64_t ldo) {
    pfr::require(T >= 0 && B >= 0 && prefix_len >= 0 && table_w >= 0, "kv attention: negative extent");
    pfr::require(heads >= 1 && heads % kv->heads == 0, "kv attention: query heads must be a multiple of the cache's heads");
    if (dtype != PFR_F32 && dtype != kv->dtype)
        throw pfr::Error(PFR_ERR_UNSUPPORTED, "kv attention: queries are float32 or of the cache's type");
    pfr::require(ldq >= heads * kv->dim && ldo >= heads * kv->dim, "kv attention: token stride below heads * dim");
    pfr::require(std::isfinite(scale), "kv attention: scale must be finite");
    pfr::require(T == 0 || (q && out), "kv attention: null q/out");
    pfr::require(prefix_len == 0 || prefix_table, "kv attention: null prefix table");
    pfr::require(B == 0 || (lengths && start), "kv attention: null lengths/start");
    pfr::require(B == 0 || table_w == 0 || table, "kv attention: null table");
    pfr::require(table_ld >= table_w, "kv attention: table row stride below its width");
    pfr::require(max_added >= 0 && max_length >= 0, "kv attention: negative bound");
    // rows and positions are 32-bit, and so are a launch's threads
    pfr::require(T <= (1 << 25) / heads && table_w <= INT32_MAX && B < (1 << 24) / kv->heads, "kv attention: extent too large");
    pfr::require(ldq < (int64_t(1) << 40) && ldo < (int64_t(1) << 40), "kv attention: extent too large");
    const int64_t es = dtype == PFR_F32 ? 4 : 2, row = heads * kv->dim;
    pfr::require(T == 0 || pfr::disjoint(q, ((T - 1) * ldq + row) * es, out, ((T - 1) * ldo + row) * es),
                 "kv attention: out overlaps q");
    const int64_t room = table_w * kv->page_size;
    pfr::require(room <= pfr::kMaxKeys && prefix_len <= pfr::kMaxKeys, "kv attention: extent too large");
    pfr::bind(ctx);
    if (T == 0) return;

    Args a{};
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.k = kv->k;
    a.v = kv->v;
    a.head_stride = kv->head_stride;
    a.map.page = pfr::FastDiv((uint32_t)kv->page_size);
    a.map.pages = (uint32_t)kv->pages;
    a.map.page_stride = kv->page_stride;
    a.map.token_stride = kv->token_stride;
    a.D = (int32_t)kv->dim;
    a.Hkv = (int32_t)kv->heads;
    a.Hq = (int32_t)heads;
    a.G = a.Hq / a.Hkv;
    a.group = pfr::FastDiv((uint32_t)a.G);
    a.T = (int32_t)T;
    a.scale = scale == 0.0f ? 1.0f : std::fabs(scale) * 1.44269504088896340736f;
    a.sign = scale == 0.0f ? 0.0f : (scale < 0.0f ? -1.0f : 1.0f);
    a.prefix_table = prefix_table;
    a.prefix_len = (int32_t)prefix_len;
    a.table = table;
    a.table_ld = table_ld;
    a.table_w = (int32_t)table_w;
    a.lengths = lengths;
    a.start = start;
    a.B = (int32_t)B;
    // bounds: what a request may add and hold
    if (max_added == 0 || max_added > T) max_added = T;
    if (max_length == 0 || max_length > room) max_length = room;
    const Plan p = plan(ctx->num_cu, dtype != PFR_F32, kv->dtype != PFR_F32, max_added, max_length, room, a);

    const bool in_shares = p.own == pfr::attn::kShares;
    const int64_t parts = in_shares ? a.parts : a.p_splits + a.o_splits, rows = T * heads;
    if (!a.whole || in_shares) {
        const size_t o = (size_t)(parts * rows * kv->dim) * sizeof(float);
        char* ws = static_cast<char*>(ctx->scratch[7].ensure(o + (size_t)(parts * rows) * sizeof(float2) + 16));
        a.part_o = reinterpret_cast<float*>(ws);
        a.part_ml = reinterpret_cast<float2*>(ws + o);
    }
    a.zeros = zeros(ctx, a.Hkv * (in_shares ? a.items : B + 2));
    auto* arrived = reinterpret_cast<uint32_t*>(const_cast<char*>(a.zeros) + kZeros);
    const bool one = p.prefix == p.own;  // (a call in shares has no launch for the prefix)
    const auto by = [](int64_t n) { return pfr::FastDiv((uint32_t)(n > 0 ? n : 1)); };
    a.by_heads = by(a.Hkv);
    a.by_p_tiles = by(a.p_tiles);
    a.by_o_tiles = by(a.o_tiles);
    a.by_fours = by(a.D / 4);
    a.by_requests = by(a.B + (a.whole ? 2 : 0));
    // the workgroups that come last join the rows, where there is little to join
    if (a.part_o != nullptr && p.own != pfr::attn::kWide && p.own_blocks > 0 &&
        (in_shares || (!one && parts <= kJoinParts) || (one && !a.solo && B + 2 <= 64 && T * a.G <= kJoinRows)))
        a.arrived = arrived;
    a.p_items = (int32_t)p.prefix_blocks;
    enqueue(ctx, kv, dtype, a, p.prefix, p.prefix_blocks + (one ? p.own_blocks : 0));
    if (!one) {
        a.p_items = 0;
        enqueue(ctx, kv, dtype, a, p.own, p.own_blocks);
    }
    if (a.part_o != nullptr && a.arrived == nullptr) {
        const dim3 grid((unsigned)ceil_div(rows, 4)), wg(256);
        if (dtype == PFR_BF16) hipLaunchKernelGGL(k_kv_attn_join<__bf16>, grid, wg, 0, ctx->stream, a);
        else if (dtype == PFR_F16) hipLaunchKernelGGL(k_kv_attn_join<_Float16>, grid, wg, 0, ctx->stream, a);
        else hipLaunchKernelGGL(k_kv_attn_join<float>, grid, wg, 0, ctx->stream, a);
    }
    PFR_HIP(hipGetLastError());
}

}  // namespace

extern "C" {

int pfr_kv_attention_dev(pfr_ctx* ctx, const pfr_kv* kv, const void* q, pfr_dtype dtype, int64_t T, int64_t heads,
                         int64_t ldq, float scale, const int32_t* prefix_table, int64_t prefix_len, const int32_t* table,
                         int64_t table_w, int64_t table_ld, int64_t B, const int32_t* lengths, const int32_t* start,
                         int64_t max_added, int64_t max_length, void* out, int64_t ldo) {
    return pfr::guarded([&] {
        pfr::require(kv != nullptr, "null kv cache");
        attention_dev(ctx, kv, q, dtype, T, heads, ldq, scale, prefix_table, prefix_len, table, table_w, table_ld, B,
                      lengths, start, max_added, max_length, out, ldo);
    });
}

}  // extern "C"
