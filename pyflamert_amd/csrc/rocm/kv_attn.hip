// Attention over a paged key/value cache: a prefix that every request shares,
// and each request's own tokens up to the query's.  No counterpart in the
// reference.
#include <cmath>

#include "common.hpp"
#include "kv.hpp"

#pragma clang fp contract(off)

namespace {

using pfr::FastDiv;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;   // waves of a workgroup
constexpr int kBlock = 32;  // keys of a wave's block

struct AttnArgs {
    const void* q;
    int64_t ldq;
    void* out;
    int64_t ldo;
    const void* k;
    const void* v;
    int64_t head_stride;
    pfr::PageMap map;
    FastDiv group;  // by the query heads of a key head
    int32_t D, G, Hkv, Hq;
    int32_t T;
    float scale;  // of the scores, times log2 e
    const int32_t* prefix_table;
    int32_t prefix_len;
    const int32_t* table;
    int64_t table_ld;
    int32_t table_w;
    const int32_t* lengths;
    const int32_t* start;
    int32_t B;
    // prefix items: Hkv * p_tiles * p_splits workgroups, p_chunk keys a split;
    // then own items: Hkv * B * o_tiles * o_splits, o_chunk keys a split
    int32_t p_tiles, p_splits, p_chunk, o_tiles, o_splits, o_chunk;
    float* part_o;    // [p_splits + o_splits][T * Hq][D]
    float2* part_ml;  // [p_splits + o_splits][T * Hq]
};

template <class T>
struct Mfma16;
template <>
struct Mfma16<__bf16> {
    typedef __bf16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f4 dot(V8 a, V8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Mfma16<_Float16> {
    typedef _Float16 V8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f4 dot(V8 a, V8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

template <int BYTES>
struct Raw;
template <>
struct Raw<8> {
    typedef u2 T;
};
template <>
struct Raw<16> {
    typedef u4 T;
};

template <class T>
constexpr uint32_t exp_bits() {
    return sizeof(T) == 4 ? 0x7f800000u : (std::is_same<T, _Float16>::value ? 0x7c00u : 0x7f80u);
}

// The operands of one block of kBlock keys and RT tiles of 16 query rows, and
// the running output, in registers.  Lane = 16 g + n.
//
// Scores are S^T = K Q^T, 16 keys x 16 rows a tile: the matrix unit leaves row
// n's scores of keys 4 g + i of the tile in the lane's registers i.  That is
// where the second product, O^T = V^T P^T, wants its right operand if its
// sum runs over the keys in the order (g; tile 0's 4 g .. 4 g + 3, tile 1's),
// so P goes from one product into the other without leaving its lane, and a
// row's statistics, its P and its O^T column share the lane's n.
template <class QT, class KT, int DP, int RT, bool FULL>
struct Tiles {
    static constexpr bool kHalf = sizeof(QT) == 2;         // 16-bit products; else float32 ones
    static constexpr int VE = 16 / (int)sizeof(KT);         // elements of a 16-byte load
    static constexpr int KS = DP / (4 * VE);                // key loads per lane and tile
    static constexpr int VV = VE < DP / 16 ? VE : DP / 16;  // contiguous values of a lane per load
    static constexpr int CC = DP / 16 / VV;                 // value loads per lane and key
    static constexpr int NT = DP / 16;                      // 16-wide column tiles of O: tile c * VV + e
    typedef typename Raw<VV * (int)sizeof(KT)>::T VRaw;
    typedef QT QV __attribute__((ext_vector_type(VE)));
    typedef QT QVu __attribute__((ext_vector_type(VE), aligned(sizeof(QT))));
    typedef KT KV __attribute__((ext_vector_type(VE)));

    QV q[RT][KS];
    KV k[2][KS];
    VRaw v[8][CC];
    f4 o[RT][NT];

    // element e of load s of a lane is d = (4 s + g) VE + e, for rows of Q and of K alike
    __device__ __forceinline__ void load_q(int rt, const QT* row, bool valid, int g, int D) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = (4 * s + g) * VE;
            q[rt][s] = QV(0);
            if (valid && (FULL || d < D)) q[rt][s] = *reinterpret_cast<const QVu*>(row + d);
        }
    }
    __device__ __forceinline__ void load_k(int t, const KT* row, int g, int D) {
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = (4 * s + g) * VE;
            if (FULL || d < D) k[t][s] = *reinterpret_cast<const KV*>(row + d);
            else k[t][s] = KV(0);
        }
    }
    // value register j is key 4 g + j of tile 0 (j < 4) or 4 g + j - 4 of tile
    // 1, columns (16 c + n) VV ..
    __device__ __forceinline__ void load_v(int j, const KT* row, int n, int D) {
#pragma unroll
        for (int c = 0; c < CC; ++c) {
            const int d = (16 * c + n) * VV;
            if (FULL || d < D) v[j][c] = *reinterpret_cast<const VRaw*>(row + d);
            else v[j][c] = VRaw(0);
        }
    }
    __device__ __forceinline__ void zero_v(int j) {
#pragma unroll
        for (int c = 0; c < CC; ++c) v[j][c] = VRaw(0);
    }
    // whether value register j holds an infinity or a NaN
    __device__ __forceinline__ bool nonfinite_v(int j) const {
        constexpr uint32_t E = exp_bits<KT>();
        bool bad = false;
#pragma unroll
        for (int c = 0; c < CC; ++c)
#pragma unroll
            for (int w = 0; w < (int)sizeof(VRaw) / 4; ++w) {
                const uint32_t x = v[j][c][w];
                bad |= (x & E) == E;
                if constexpr (sizeof(KT) == 2) bad |= ((x >> 16) & E) == E;
            }
        return bad;
    }
    __device__ __forceinline__ f4 scores(int rt, int t) const {
        f4 acc = f4(0.0f);
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if constexpr (kHalf) {
                acc = Mfma16<KT>::dot(k[t][s], q[rt][s], acc);
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    acc = __builtin_amdgcn_mfma_f32_16x16x4f32((float)k[t][s][e], q[rt][s][e], acc, 0, 0, 0);
            }
        }
        return acc;
    }
    // o += V^T p for the lane's eight keys, p in the order of v's registers.
    // With 16-bit products p is rounded to the cache's type (its error, half a
    // step a weight and averaged over the keys, is the size of the output's
    // own rounding); the sum of the weights keeps 32 bits.
    __device__ __forceinline__ void add(int rt, const float (&p)[8]) {
        if constexpr (kHalf) {
            typename Mfma16<KT>::V8 pv;
#pragma unroll
            for (int j = 0; j < 8; ++j) pv[j] = (KT)p[j];
#pragma unroll
            for (int c = 0; c < CC; ++c)
#pragma unroll
                for (int e = 0; e < VV; ++e) {
                    // the lane's column e of its eight keys, two keys a register
                    u4 col;
#pragma unroll
                    for (int x = 0; x < 4; ++x)
                        col[x] = __builtin_amdgcn_perm(v[2 * x + 1][c][e / 2], v[2 * x][c][e / 2],
                                                       (e & 1) ? 0x07060302u : 0x05040100u);
                    o[rt][c * VV + e] = Mfma16<KT>::dot(__builtin_bit_cast(typename Mfma16<KT>::V8, col), pv, o[rt][c * VV + e]);
                }
        } else {
            typedef KT VK __attribute__((ext_vector_type(VV)));
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < CC; ++c) {
                    const VK x = __builtin_bit_cast(VK, v[j][c]);
#pragma unroll
                    for (int e = 0; e < VV; ++e)
                        o[rt][c * VV + e] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)x[e], p[j], o[rt][c * VV + e], 0, 0, 0);
                }
        }
    }
};

// The largest over the four lanes that hold a row.
__device__ __forceinline__ float row_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float row_sum(float x) {
    x = x + __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}
__device__ __forceinline__ float finite_max(float m) { return m == -INFINITY ? 0.0f : m; }

// One workgroup's rows against keys [lo, hi) of one table.  Rows r0 .. of the
// n_rows that start at token t0: row r is query head r % G of token t0 + r / G.
// lim0 and per_token: row r sees keys below lim0 + per_token * (r / G).
// Writes the rows' part `part`.
template <class QT, class KT, int DP, int RT, bool FULL>
__device__ __forceinline__ void attend(const AttnArgs& a, float* lds, int h, int t0, int r0, int n_rows,
                                       const int32_t* __restrict__ table, int table_w, int lo, int hi, int lim0,
                                       int per_token, int part) {
    typedef Tiles<QT, KT, DP, RT, FULL> TT;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n = lane & 15, g = lane >> 4;
    TT x;
    float m[RT], l[RT];
    int lim[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int r = r0 + rt * 16 + n;
        const bool valid = r < n_rows;
        const int dt = (int)a.group.div((uint32_t)(valid ? r : 0));
        const int hq = h * a.G + (valid ? r : 0) - dt * a.G;
        x.load_q(rt, static_cast<const QT*>(a.q) + (int64_t)(t0 + dt) * a.ldq + (int64_t)hq * a.D, valid, g, a.D);
        lim[rt] = valid ? lim0 + per_token * dt : 0;
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int i = 0; i < TT::NT; ++i) x.o[rt][i] = f4(0.0f);
    }
    // all rows see the keys below this
    const int min_lim = lim0 + per_token * (int)a.group.div((uint32_t)r0);
    const KT* kp = static_cast<const KT*>(a.k) + (int64_t)h * a.head_stride;
    const KT* vp = static_cast<const KT*>(a.v) + (int64_t)h * a.head_stride;

    for (int k0 = lo + w * kBlock; k0 < hi; k0 += kWaves * kBlock) {
        // lane i (and i + 32) finds key i
        const int key = k0 + (lane & 31);
        int64_t off = key < hi ? pfr::key_offset(a.map, table, table_w, key) : -1;
        const uint32_t okm = (uint32_t)__ballot(off >= 0);
        off = off < 0 ? 0 : off;  // the pool's first row is there to be read
        if (okm == 0) continue;
#pragma unroll
        for (int t = 0; t < 2; ++t) x.load_k(t, kp + __shfl((long long)off, 16 * t + n), g, a.D);
#pragma unroll
        for (int u = 0; u < 8; ++u) x.load_v(u, vp + __shfl((long long)off, (u < 4 ? 0 : 16) + 4 * g + (u & 3)), n, a.D);

        const bool partly = k0 + kBlock > min_lim;
        uint32_t poison = 0;
        if (okm != ~0u) {
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (!((okm >> ((u < 4 ? 0 : 16) + 4 * g + (u & 3))) & 1)) x.zero_v(u);
        }
        if (partly) {
            // A key that only some rows see must not reach the others, and 0
            // times an infinity or a NaN would: such values are added row by row.
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const uint64_t b = __ballot(x.nonfinite_v(u));
#pragma unroll
                for (int gg = 0; gg < 4; ++gg)
                    if ((b >> (16 * gg)) & 0xffff) poison |= 1u << ((u < 4 ? 0 : 16) + 4 * gg + (u & 3));
            }
            if (min_lim > k0) poison &= ~0u << (min_lim - k0);
            if (poison) {
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if ((poison >> ((u < 4 ? 0 : 16) + 4 * g + (u & 3))) & 1) x.zero_v(u);
            }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float s[8];
            const f4 s0 = x.scores(rt, 0), s1 = x.scores(rt, 1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = s0[i] * a.scale;
                s[4 + i] = s1[i] * a.scale;
            }
            if (partly || okm != ~0u) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int kk = (u < 4 ? 0 : 16) + 4 * g + (u & 3);
                    if (!((okm >> kk) & 1) || k0 + kk >= lim[rt]) s[u] = -INFINITY;
                }
            }
            float mx = s[0];
#pragma unroll
            for (int u = 1; u < 8; ++u) mx = fmaxf(mx, s[u]);
            const float mn = fmaxf(m[rt], row_max(mx)), ms = finite_max(mn);
            const float alpha = __builtin_amdgcn_exp2f(m[rt] - ms);
            m[rt] = mn;
            float p[8], sum = 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                p[u] = __builtin_amdgcn_exp2f(s[u] - ms);
                sum = sum + p[u];
            }
            l[rt] = l[rt] * alpha + sum;
#pragma unroll
            for (int i = 0; i < TT::NT; ++i) x.o[rt][i] *= alpha;
            x.add(rt, p);
            for (uint32_t rest = poison; rest; rest &= rest - 1) {
                const int kk = __builtin_ctz(rest), u0 = (kk >> 4) * 4 + (kk & 3), g0 = (kk >> 2) & 3;
                float mine = 0.0f;
#pragma unroll
                for (int u = 0; u < 8; ++u) mine = u == u0 ? p[u] : mine;
                const float pk = __shfl(mine, 16 * g0 + n);
                const KT* row = vp + __shfl((long long)off, kk);
                if (((okm >> kk) & 1) && k0 + kk < lim[rt]) {
#pragma unroll
                    for (int c = 0; c < TT::CC; ++c)
#pragma unroll
                        for (int e = 0; e < TT::VV; ++e)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int d = (16 * c + 4 * g + i) * TT::VV + e;
                                if (FULL || d < a.D) x.o[rt][c * TT::VV + e][i] += pk * (float)row[d];
                            }
                }
            }
        }
    }

    // the waves' sums, joined
    float* sm = lds;                       // [kWaves][16 RT] maxima
    float* sl = lds + kWaves * 16 * RT;    // [kWaves][16 RT] sums
    float* so = lds + 2 * kWaves * 16 * RT;  // [kWaves][16][64 VV's columns + 4]
    constexpr int kCols = 16 * TT::VV, kPitch = kCols + 4;
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        l[rt] = row_sum(l[rt]);
        if (g == 0) {
            sm[w * 16 * RT + rt * 16 + n] = m[rt];
            sl[w * 16 * RT + rt * 16 + n] = l[rt];
        }
    }
    __syncthreads();
    const int64_t rows_all = (int64_t)a.T * a.Hq;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        if (r0 + rt * 16 >= n_rows) break;
        float M = -INFINITY;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) M = fmaxf(M, sm[i * 16 * RT + rt * 16 + n]);
        const float f = __builtin_amdgcn_exp2f(m[rt] - finite_max(M));
        if (w == 0 && g == 0 && r0 + rt * 16 + n < n_rows) {
            float L = 0.0f;
#pragma unroll
            for (int i = 0; i < kWaves; ++i)
                L = L + sl[i * 16 * RT + rt * 16 + n] * __builtin_amdgcn_exp2f(sm[i * 16 * RT + rt * 16 + n] - finite_max(M));
            const int r = r0 + rt * 16 + n, dt = (int)a.group.div((uint32_t)r);
            const int64_t R = (int64_t)(t0 + dt) * a.Hq + h * a.G + (r - dt * a.G);
            a.part_ml[(int64_t)part * rows_all + R] = make_float2(M, L);
        }
#pragma unroll
        for (int c = 0; c < TT::CC; ++c) {
            float* mine = so + w * 16 * kPitch + n * kPitch;
#pragma unroll
            for (int e = 0; e < TT::VV; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[(4 * g + i) * TT::VV + e] = x.o[rt][c * TT::VV + e][i] * f;
            __syncthreads();
            for (int z = threadIdx.x; z < 16 * kCols; z += kWaves * 64) {
                const int rr = z / kCols, cc = z % kCols, r = r0 + rt * 16 + rr, d = c * kCols + cc;
                if (r < n_rows && d < a.D) {
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < kWaves; ++i) sum = sum + so[i * 16 * kPitch + rr * kPitch + cc];
                    const int dt = (int)a.group.div((uint32_t)r);
                    const int64_t R = (int64_t)(t0 + dt) * a.Hq + h * a.G + (r - dt * a.G);
                    a.part_o[((int64_t)part * rows_all + R) * a.D + d] = sum;
                }
            }
            __syncthreads();
        }
    }
}

template <int RT>
constexpr int lds_floats(int cols) {
    return 2 * kWaves * 16 * RT + kWaves * 16 * (cols + 4);
}

template <class QT, class KT, int DP, int RT, bool FULL>
__global__ __launch_bounds__(kWaves * 64) void k_kv_attn_prefix(AttnArgs a) {
    __shared__ float lds[lds_floats<RT>(16 * Tiles<QT, KT, DP, RT, FULL>::VV)];
    const int h = (int)blockIdx.x % a.Hkv, i = (int)blockIdx.x / a.Hkv;
    const int tile = i % a.p_tiles, split = i / a.p_tiles;
    int lo, hi;
    pfr::split_span(split, a.p_splits, a.p_chunk, a.prefix_len, &lo, &hi);
    attend<QT, KT, DP, RT, FULL>(a, lds, h, 0, tile * 16 * RT, a.T * a.G, a.prefix_table, INT32_MAX, lo, hi, a.prefix_len, 0, split);
}

template <class QT, class KT, int DP, int RT, bool FULL>
__global__ __launch_bounds__(kWaves * 64) void k_kv_attn_own(AttnArgs a) {
    __shared__ float lds[lds_floats<RT>(16 * Tiles<QT, KT, DP, RT, FULL>::VV)];
    const int h = (int)blockIdx.x % a.Hkv, b = (int)blockIdx.x / a.Hkv;
    const int tile0 = (int)blockIdx.y, split = (int)blockIdx.z;
    int t0, t1;
    pfr::request_tokens(a.start, b, a.T, &t0, &t1);
    const int n_rows = (t1 - t0) * a.G;
    if (n_rows == 0) return;
    const int lim0 = pfr::first_limit(a.lengths[b], t1 - t0);
    const int64_t room = (int64_t)a.table_w * a.map.page.d;
    for (int tile = tile0; tile * 16 * RT < n_rows; tile += a.o_tiles) {
        const int r0 = tile * 16 * RT, r1 = r0 + 16 * RT < n_rows ? r0 + 16 * RT : n_rows;
        const int end = pfr::keys_end(lim0, (int)a.group.div((uint32_t)(r1 - 1)), room);
        int lo, hi;
        pfr::split_span(split, a.o_splits, a.o_chunk, end, &lo, &hi);
        attend<QT, KT, DP, RT, FULL>(a, lds, h, t0, r0, n_rows, a.table + (int64_t)b * a.table_ld, a.table_w, lo, hi, lim0, 1,
                                     a.p_splits + split);
        __syncthreads();
    }
}

// One wave a row: the parts' sums joined, divided, rounded to the output's type.
template <class QT>
__global__ __launch_bounds__(256) void k_kv_attn_join(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t rows = (int64_t)a.T * a.Hq, R = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (R >= rows) return;
    const int t = (int)(R / a.Hq);
    const bool own = a.B > 0 && t >= a.start[0] && t < a.start[a.B];
    const int parts = a.p_splits + (own ? a.o_splits : 0);
    float M = -INFINITY;
    for (int p = lane; p < parts; p += 64) M = fmaxf(M, a.part_ml[p * rows + R].x);
    for (int o = 32; o; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    const float Ms = finite_max(M);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, L = 0.0f;
    for (int p = 0; p < parts; ++p) {
        const float2 ml = a.part_ml[p * rows + R];
        if (ml.x == -INFINITY && ml.y == 0.0f) continue;
        const float f = __builtin_amdgcn_exp2f(ml.x - Ms);
        L = L + f * ml.y;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = lane + 64 * i;
            if (d < a.D) acc[i] = acc[i] + f * a.part_o[(p * rows + R) * a.D + d];
        }
    }
    QT* o = static_cast<QT*>(a.out) + (int64_t)t * a.ldo + (R - (int64_t)t * a.Hq) * a.D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int d = lane + 64 * i;
        if (d < a.D) o[d] = (QT)(L == 0.0f ? 0.0f : acc[i] / L);
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits of `keys` keys so that `items` workgroups a split fill the chip, and
// the keys of each: whole rounds of the waves' blocks.
void split_keys(int num_cu, int64_t items, int64_t keys, int32_t* splits, int32_t* chunk) {
    const int64_t round = kWaves * kBlock;
    int64_t s = keys > 0 ? ceil_div(2 * num_cu, items > 0 ? items : 1) : 0;
    const int64_t most = ceil_div(keys, round);
    s = s > most ? most : s;
    const int64_t c = s > 0 ? ceil_div(ceil_div(keys, s), round) * round : round;
    *splits = (int32_t)(s > 0 ? ceil_div(keys, c) : 0);
    *chunk = (int32_t)c;
}

template <class QT, class KT, int DP, bool FULL>
void launch_rt(pfr_ctx* ctx, const AttnArgs& a, int p_rt, int o_rt) {
    hipStream_t s = ctx->stream;
    constexpr int kMost = sizeof(QT) == 2 && DP <= 128 ? 4 : (DP <= 128 ? 2 : 1);
    if (a.p_splits > 0) {
        const dim3 grid((unsigned)(a.Hkv * a.p_tiles * a.p_splits));
        if (p_rt == 1) hipLaunchKernelGGL((k_kv_attn_prefix<QT, KT, DP, 1, FULL>), grid, dim3(kWaves * 64), 0, s, a);
        else if (p_rt == 2) hipLaunchKernelGGL((k_kv_attn_prefix<QT, KT, DP, kMost < 2 ? kMost : 2, FULL>), grid, dim3(kWaves * 64), 0, s, a);
        else hipLaunchKernelGGL((k_kv_attn_prefix<QT, KT, DP, kMost, FULL>), grid, dim3(kWaves * 64), 0, s, a);
    }
    if (a.o_splits > 0) {
        const dim3 grid((unsigned)(a.Hkv * a.B), (unsigned)a.o_tiles, (unsigned)a.o_splits);
        if (o_rt == 1) hipLaunchKernelGGL((k_kv_attn_own<QT, KT, DP, 1, FULL>), grid, dim3(kWaves * 64), 0, s, a);
        else if (o_rt == 2) hipLaunchKernelGGL((k_kv_attn_own<QT, KT, DP, kMost < 2 ? kMost : 2, FULL>), grid, dim3(kWaves * 64), 0, s, a);
        else hipLaunchKernelGGL((k_kv_attn_own<QT, KT, DP, kMost, FULL>), grid, dim3(kWaves * 64), 0, s, a);
    }
    const int64_t rows = (int64_t)a.T * a.Hq;
    hipLaunchKernelGGL(k_kv_attn_join<QT>, dim3((unsigned)ceil_div(rows, 4)), dim3(256), 0, s, a);
    PFR_HIP(hipGetLastError());
}

template <class QT, class KT>
void launch_dim(pfr_ctx* ctx, const AttnArgs& a, int p_rt, int o_rt) {
    if (a.D == 128) launch_rt<QT, KT, 128, true>(ctx, a, p_rt, o_rt);
    else if (a.D <= 64) launch_rt<QT, KT, 64, false>(ctx, a, p_rt, o_rt);
    else if (a.D < 128) launch_rt<QT, KT, 128, false>(ctx, a, p_rt, o_rt);
    else launch_rt<QT, KT, 256, false>(ctx, a, p_rt, o_rt);
}

// Row tiles of 16 a wave takes at once: as many as there are, up to what its registers hold.
int row_tiles(int64_t rows, int most) { return rows <= 16 ? 1 : (rows <= 32 || most < 4 ? (most < 2 ? 1 : 2) : most); }

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

    AttnArgs a{};
    a.q = q;
    a.ldq = ldq;
    a.out = out;
    a.ldo = ldo;
    a.k = kv->k;
    a.v = kv->v;
    a.head_stride = kv->head_stride;
    a.map.page = FastDiv((uint32_t)kv->page_size);
    a.map.pages = (uint32_t)kv->pages;
    a.map.page_stride = kv->page_stride;
    a.map.token_stride = kv->token_stride;
    a.D = (int32_t)kv->dim;
    a.Hkv = (int32_t)kv->heads;
    a.Hq = (int32_t)heads;
    a.G = a.Hq / a.Hkv;
    a.group = FastDiv((uint32_t)a.G);
    a.T = (int32_t)T;
    a.scale = scale * 1.44269504088896340736f;
    a.prefix_table = prefix_table;
    a.prefix_len = (int32_t)prefix_len;
    a.table = table;
    a.table_ld = table_ld;
    a.table_w = (int32_t)table_w;
    a.lengths = lengths;
    a.start = start;
    a.B = (int32_t)B;

    const int most = dtype != PFR_F32 && kv->dim <= 128 ? 4 : (kv->dim <= 128 ? 2 : 1);
    const int64_t p_rows = T * a.G;
    const int p_rt = row_tiles(p_rows, most);
    a.p_tiles = (int32_t)ceil_div(p_rows, 16 * p_rt);
    split_keys(ctx->num_cu, a.Hkv * a.p_tiles, prefix_len, &a.p_splits, &a.p_chunk);

    // bounds: what a request may add and hold
    if (max_added == 0 || max_added > T) max_added = T;
    if (max_length == 0 || max_length > room) max_length = room;
    const int64_t o_rows = max_added * a.G;
    const int o_rt = row_tiles(o_rows, most);
    a.o_tiles = (int32_t)ceil_div(o_rows, 16 * o_rt);
    a.o_tiles = a.o_tiles > 65535 ? 65535 : a.o_tiles;
    if (B > 0) {
        split_keys(ctx->num_cu, B * a.Hkv * a.o_tiles, max_length, &a.o_splits, &a.o_chunk);
    }
    pfr::require((int64_t)a.Hkv * a.p_tiles * a.p_splits < (1 << 24), "kv attention: extent too large");
    const int64_t parts = a.p_splits + a.o_splits, rows = T * heads;
    const size_t ml = (size_t)(parts * rows) * sizeof(float2);
    char* ws = static_cast<char*>(ctx->scratch[7].ensure(ml + (size_t)(parts * rows * kv->dim) * sizeof(float) + 16));
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float2*>(ws + (size_t)(parts * rows * kv->dim) * sizeof(float));

    if (dtype == PFR_BF16) launch_dim<__bf16, __bf16>(ctx, a, p_rt, o_rt);
    else if (dtype == PFR_F16) launch_dim<_Float16, _Float16>(ctx, a, p_rt, o_rt);
    else if (kv->dtype == PFR_BF16) launch_dim<float, __bf16>(ctx, a, p_rt, o_rt);
    else if (kv->dtype == PFR_F16) launch_dim<float, _Float16>(ctx, a, p_rt, o_rt);
    else launch_dim<float, float>(ctx, a, p_rt, o_rt);
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
