// Attention of packed query rows over the 8-bit paged cache (see include/pigeon_hip.h: pgn_cached_attention).
//
// For a query row i of request r, with keys j of its block table, 8-bit bytes k8 / v8 and their page's scales s:
//   x_ij = scale * s_k(j) * (q_i . k8_j)        j <= pos_i (causal), j > pos_i - window
//   o_i  = sum_j 2^(x_ij log2e - m_i) s_v(j) v8_j / sum_j 2^(x_ij log2e - m_i)        m_i: running maximum
// The bytes become bf16 / fp16 (exact: e4m3 has four significant bits) on their way into the matrix instructions, so q
// keeps its 16 bits; scores, maxima, sums and the output accumulator are fp32, the probabilities are rounded to the
// 16-bit type for the second product and summed before that rounding.
//
// Operands without any exchange between lanes.  A wave takes 64 keys at a time, as four tiles of 16 for
// S^T = K Q^T.  Row m of tile t is key 16 (m >> 2) + 4 t + (m & 3), so that the result leaves lane group g (16 lanes, one
// per query row) with the keys 16 g .. 16 g + 15: as the second operand of O^T = V^T P^T they pair with 16 CONSECUTIVE
// tokens of a head dim, one 16-byte load from the transposed value page, and all of a lane's keys lie in one page, so
// both scales are one number per lane.  The contraction over head dims is permuted alike (lane group g owns bytes
// 16 g .. 16 g + 15 of each 64), which makes the key loads 16 bytes too.
#include "pgn_common.h"

#include "pgn_fp8.h"

namespace {

struct CachedArgs {
    const unsigned short* q;
    const unsigned char* k_pages;
    const unsigned char* v_pages;
    const float* k_scale;
    const float* v_scale;
    const int* table;
    const int* lens;
    const int* starts;
    unsigned short* out;
    float* part_o;                                           // of each split and row: unnormalised output, then maximum and sum
    float2* part_ml;
    int4* plans;                                             // of each request with few rows: tiles, splits, first slot
    float* big_part_o;
    float2* big_part_ml;
    int64_t table_stride, q_st, q_sh, o_st, o_sh;
    int T, R, Hq, Hkv, G, W, shift, N, causal, window;
    int few_split, few_slots, tiles_per_request;             // of the 16-row kernel
    int big_nsplit, big_tiles;                               // of the 128-row kernel
    int out_vec;                                             // rows of `out` begin on 8 bytes
    float c;                                                 // scale * log2(e)
};

template <int DT>
struct Mat;
template <>
struct Mat<PGN_BF16> {
    typedef bf16x8_t v8;
    typedef __attribute__((ext_vector_type(2))) __bf16 v2;
    static __device__ __forceinline__ f32x4_t mfma16(v8 a, v8 b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    template <bool HI>
    static __device__ __forceinline__ v2 cvt(unsigned w, float s) {
        return __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI);
    }
    static __device__ __forceinline__ f32x16_t mfma32(v8 a, v8 b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ __bf16 one(float f) { return (__bf16)f; }
};
template <>
struct Mat<PGN_F16> {
    typedef f16x8_t v8;
    typedef __attribute__((ext_vector_type(2))) _Float16 v2;
    static __device__ __forceinline__ f32x4_t mfma16(v8 a, v8 b, f32x4_t c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    template <bool HI>
    static __device__ __forceinline__ v2 cvt(unsigned w, float s) {
        return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, s, HI);
    }
    static __device__ __forceinline__ f32x16_t mfma32(v8 a, v8 b, f32x16_t c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ _Float16 one(float f) { return (_Float16)f; }
};

// 8 e4m3 bytes times a power of two -> 8 values of the 16-bit type
template <int DT>
__device__ __forceinline__ typename Mat<DT>::v8 widen8(unsigned lo, unsigned hi, float s) {
    typename Mat<DT>::v2 a = Mat<DT>::template cvt<false>(lo, s), b = Mat<DT>::template cvt<true>(lo, s);
    typename Mat<DT>::v2 c = Mat<DT>::template cvt<false>(hi, s), d = Mat<DT>::template cvt<true>(hi, s);
    typename Mat<DT>::v8 r = {a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    return r;
}

// 0x80 in every byte of w that is an e4m3 NaN
__device__ __forceinline__ unsigned nan_bytes(unsigned w) {
    return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
}

// mask of the bytes of word `word` of a lane's 16 whose key (first + 4 word + byte) lies in [lo, hi)
__device__ __forceinline__ unsigned key_bytes(int first, int word, int lo, int hi) {
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int key = first + 4 * word + j;
        m |= key >= lo && key < hi ? 0xffu << (8 * j) : 0u;
    }
    return m;
}

// Requests of up to this many rows (a row: a token and a query head of the KV head's group) go to the 16-row kernel, the
// others to the 128-row kernel, in one call if need be.  At head dim 128: 4 requests of 64 rows over 4096 keys of 4 KV
// heads take 28 us in the one and 41 in the other, 32 requests over 2048 keys 62 and 61; with 128 rows 40 and 45, and 103
// and 83.  With 8 KV heads 64 rows take 39 and 43, 96 and 88; 128 rows 64 and 47, 148 and 89.
#define PGN_CA_FEW_ROWS 64

// The rows of a workgroup: consecutive rows of one request, ROWS to a tile.  16-row tiles: a fixed number for every
// request.  128-row tiles leave each request the numbers floor(start * G / 128) + r and up, which is room for its
// ceil(n * G / 128) tiles whatever the lengths are, so the launch needs to know only the number of tokens and requests.
struct TileRows {
    int r, first, count, begin, n, len;                      // first row of the tile in its request, its valid rows
};

__device__ __forceinline__ bool request_rows(const CachedArgs& a, int r, TileRows& t) {
    t.r = r;
    if (a.starts == nullptr) {
        t.begin = r;
        t.n = 1;
    } else {
        t.begin = a.starts[r];
        const int end = a.starts[r + 1];
        if (t.begin < 0 || end < t.begin || end > a.T) return false;
        t.n = end - t.begin;
    }
    const int64_t room = (int64_t)a.W << a.shift;
    const int len = a.lens[r];
    t.len = len < 0 ? 0 : (len > room ? (int)room : len);
    return true;
}

__device__ __forceinline__ bool few_rows_tile(const CachedArgs& a, int tile, TileRows& t) {
    const int r = tile / a.tiles_per_request, local = tile - r * a.tiles_per_request;
    if (!request_rows(a, r, t)) return false;
    const int rows = t.n * a.G;
    if (a.starts != nullptr && rows > PGN_CA_FEW_ROWS) return false;
    t.first = local * 16;
    t.count = min(16, rows - t.first);
    return t.count > 0;
}

template <int ROWS>
__device__ __forceinline__ bool many_rows_tile(const CachedArgs& a, int tile, TileRows& t) {
    int lo = 0, hi = a.R;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)a.starts[mid] * a.G / ROWS + mid <= tile) lo = mid;
        else hi = mid;
    }
    if (!request_rows(a, lo, t) || t.n * a.G <= PGN_CA_FEW_ROWS) return false;
    const int64_t local = tile - ((int64_t)t.begin * a.G / ROWS + lo);
    if (local < 0 || local * ROWS >= t.n * a.G) return false;
    t.first = (int)local * ROWS;
    t.count = min(ROWS, t.n * a.G - t.first);
    return true;
}

// First key that the window leaves a token at `pos` (which may be negative: more queries than keys).
__device__ __forceinline__ int window_lo(const CachedArgs& a, int pos) {
    return a.window && pos >= a.window ? pos - a.window + 1 : 0;
}

// Keys that any row of the tile sees: [lo, hi).
__device__ __forceinline__ void key_range(const CachedArgs& a, const TileRows& t, int& lo, int& hi) {
    const int pos0 = t.len - t.n + t.first / a.G, pos1 = t.len - t.n + (t.first + t.count - 1) / a.G;
    hi = a.causal ? max(0, min(t.len, pos1 + 1)) : t.len;
    lo = window_lo(a, pos0);
}

// Splits have this many keys at least: two rounds of the 16-row kernel's four waves (256: 20.8 us against 16.2 for one
// request of 16000 keys of 8 heads, 10.4 against 8.2 for one of 257; 1024: 17.4), 8 tiles of the 128-row kernel.
#define PGN_CA_LEAST_KEYS 512

// Keys of a split of the 128-row kernel.  The launch says how many splits there are, from the width of the table; their size
// goes by the longest request, or by the window, so that a wide table leaves none of them idle.
__device__ __forceinline__ int split_keys(const CachedArgs& a, int lo, int hi, int nsplit) {
    int span = hi - (lo & ~63);
    if (nsplit > 1 && a.R > 1) {                             // then R is under 512
        int longest = 0;
        for (int r = threadIdx.x & 63; r < a.R; r += 64) longest = max(longest, a.lens[r]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) longest = max(longest, __shfl_xor(longest, off));
        longest = min(longest, a.W << a.shift);
        span = max(span, a.window ? min(longest, a.window) : longest);
    }
    const int units = ((max(span, 1) + nsplit - 1) / nsplit + PGN_CA_LEAST_KEYS - 1) / PGN_CA_LEAST_KEYS;
    return __builtin_amdgcn_readfirstlane(units * PGN_CA_LEAST_KEYS);
}

// Splits of the 16-row kernel.  All have one size, under which the call's tiles make as many workgroups as the CUs hold at a
// time, so that a long request among short ones gets its share of them (64 requests of 8 heads, one of 16367 keys, the
// others of 500: 30 us instead of 111 without).  Nothing of this is known to the host: the launch has that many slots, or
// one for each tile and that many, which is what any lengths can need, and every workgroup finds the tile and split of its
// slot by a prefix sum over the requests.  That costs 1 us of a short call (4 requests of 2000 keys: 19 us).
struct FewPlan {
    int r, tiles, splits, first_slot, keys;                  // of a request: 16-row tiles, splits of each, its first slot
};

// tiles of request r and the keys that one of them can see, counted from a multiple of 64
__device__ __forceinline__ void few_request(const CachedArgs& a, int r, int& tiles, int& span) {
    TileRows t;
    tiles = span = 0;
    if (r >= a.R || !request_rows(a, r, t)) return;
    const int rows = t.n * a.G;
    if (a.starts != nullptr && rows > PGN_CA_FEW_ROWS) return;
    tiles = (rows + 15) / 16;
    span = t.len;
    if (a.window && t.len > a.window)
        span = t.n == 1 ? t.len - ((t.len - a.window) & ~63) : min(t.len, a.window + t.n) + 63;
}

// Workgroups of the 16-row kernel that the CUs hold at a time, by its registers.
__host__ __device__ constexpr int few_resident(int D) { return D == 64 ? 768 : D == 128 ? 512 : 256; }

// The plan of the request that owns a slot, by all lanes of a wave; false: there is none.  512 requests at most.
template <int D>
__device__ __forceinline__ bool few_plan(const CachedArgs& a, int slot, FewPlan& p) {
    const int lane = threadIdx.x & 63, share = max(1, few_resident(D) / a.Hkv);
    int tiles, span, longest = 0, all = 0;
    int64_t total = 0;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
        few_request(a, r0 + lane, tiles, span);
        longest = max(longest, tiles > 0 ? span : 0);
        total += (int64_t)tiles * span;
        all += tiles;
    }
    for (int off = a.R > 32 ? 32 : a.R > 8 ? 16 : 4; off > 0 && a.R > 1; off >>= 1) {
        longest = max(longest, __shfl_xor(longest, off));
        total += __shfl_xor(total, off);
        all += __shfl_xor(all, off);
    }
    all = __builtin_amdgcn_readfirstlane(all);
    longest = __builtin_amdgcn_readfirstlane(longest);
    total = ((int64_t)__builtin_amdgcn_readfirstlane((int)(total >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)total);
    // where there are enough tiles, only one of twice the average is split; 64 splits at most (see the join)
    const float mean = fminf((float)total * ((all >= share ? 2.f : 1.f) / (float)share), (float)longest);
    p.keys = max(PGN_CA_LEAST_KEYS, (max((int)ceilf(mean), (longest + 63) / 64) + 255) / 256 * 256);
    if (a.R <= 64 && all < share && p.keys < longest) {
        // Rounded up for each request, the splits may be more than the share, and the last ones would run alone: the least size
        // under which they are not, of 64, one in each lane (138 us instead of 168 for 4 requests of 60000 to 131072 keys).
        const int step = max(256, p.keys / 64 / 256 * 256), size = p.keys + lane * step;
        const float per = 1.f / (float)size;
        int count = 0;
        for (int r = 0; r < a.R; ++r) {
            const int keys = __builtin_amdgcn_readlane(span, r), whole = (int)((float)keys * per), rest = keys - whole * size;
            count += __builtin_amdgcn_readlane(tiles, r) * max(1, whole + (rest > 0) + (rest > size));     // exact: 64 at most
        }
        const uint64_t fit = __ballot(count <= share), one = __ballot(count * a.Hkv <= 256);
        if (fit == 0) {
            p.keys = longest;
        } else {
            // or a larger one with which no CU has two workgroups, if that leaves the busiest less to do
            const int at = __builtin_ctzll(fit), last = one != 0 ? __builtin_ctzll(one) : at, first_keys = p.keys;
            const int rounds = (__builtin_amdgcn_readlane(count, at) * a.Hkv + 255) / 256;
            p.keys = first_keys + at * step;
            if ((first_keys + last * step) * 1.15f < (float)p.keys * rounds) p.keys = first_keys + last * step;
        }
    }
    p.first_slot = 0;
    for (int r0 = 0; r0 < a.R; r0 += 64) {
        if (a.R > 64) few_request(a, r0 + lane, tiles, span);
        const int splits = max(1, (span + p.keys - 1) / p.keys), mine = tiles * splits;
        int upto = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            if (a.R <= off) break;
            const int o = __shfl_up(upto, off);
            if (lane >= off) upto += o;
        }
        const uint64_t has = __ballot(slot < p.first_slot + upto && mine > 0);
        if (has != 0) {
            const int at = __builtin_ctzll(has);
            p.r = r0 + at;
            p.tiles = __builtin_amdgcn_readlane(tiles, at);
            p.splits = __builtin_amdgcn_readlane(splits, at);
            p.first_slot += __builtin_amdgcn_readlane(upto - mine, at);
            return true;
        }
        p.first_slot += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

#define PGN_CA_THREADS 256

// The kernel for single tokens and short requests: 16 rows of a request, four waves that take 64 keys in turn and join
// their maxima, sums and outputs at the end.
//
// What bounds it is the cache's bytes: a row has two operations for every byte of key or value, so nothing is staged and
// no lane waits for another one inside the loop; loads go to registers in the order in which the matrix instructions take
// them, one round ahead (75 us below, 88 without).  16 requests of 900 to 4096 keys, 32 heads by 128, one row each: 354 MB
// in 75 us, 4.7 TB/s; 4 requests of 60000 to 131072 keys of 8 KV heads: 738 MB in 138 us, 5.4 TB/s.  A kernel that only
// reads that much reaches 6.0.  One request of 257 keys: 8 us, a launch and a few trips to memory one behind the other.
template <int DT, int D>
__global__ __launch_bounds__(PGN_CA_THREADS) void pgn_cached_rows16_kernel(const CachedArgs a) {
    typedef typename Mat<DT>::v8 v8;
    constexpr int DB = D / 64, DTILES = D / 16;
    extern __shared__ float lds[];                           // [4][16][D] partial outputs
    __shared__ float lds_m[4][16], lds_l[4][16];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int g = lane >> 4, col = lane & 15;
    // heads fastest: 88 us against 101 with all heads of a stretch of keys on one XCD (before the loads went ahead)
    const int h = blockIdx.x % a.Hkv, slot = blockIdx.x / a.Hkv;
    TileRows t;
    FewPlan plan;
    int split = 0;
    if (a.few_split) {
        if (!few_plan<D>(a, slot, plan) || !request_rows(a, plan.r, t)) return;
        split = (slot - plan.first_slot) / plan.tiles;
        if (slot == plan.first_slot && h == 0 && tid == 0) a.plans[plan.r] = int4{plan.tiles, plan.splits, plan.first_slot, 0};
        t.first = (slot - plan.first_slot - split * plan.tiles) * 16;
        t.count = min(16, t.n * a.G - t.first);
    } else if (!few_rows_tile(a, slot, t)) {
        return;
    }
    int lo, hi;
    key_range(a, t, lo, hi);
    const int kb = (lo & ~63) + (a.few_split ? split * plan.keys : 0), kend = a.few_split ? min(hi, kb + plan.keys) : hi;

    const int row = t.first + min(col, t.count - 1);         // rows past the last repeat it and are not written
    const int token = t.begin + row / a.G, head = h * a.G + row % a.G;
    const int pos = t.len - t.n + row / a.G;
    const int vis_hi = a.causal ? min(t.len, pos + 1) : t.len;
    const int vis_lo = window_lo(a, pos);
    // keys that every row of the tile sees
    const int all_hi = a.causal ? min(t.len, t.len - t.n + t.first / a.G + 1) : t.len;
    const int all_lo = window_lo(a, t.len - t.n + (t.first + t.count - 1) / a.G);

    v8 qf[DB * 2];
    {
        const unsigned short* qp = a.q + token * a.q_st + head * a.q_sh + g * 16;
#pragma unroll
        for (int s = 0; s < DB * 2; ++s) qf[s] = *reinterpret_cast<const v8*>(qp + (s >> 1) * 64 + (s & 1) * 8);
    }
    f32x4_t o[DTILES];
#pragma unroll
    for (int d = 0; d < DTILES; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f, ref = 0.f;

    const int* table = a.table + t.r * a.table_stride;
    const int P = 1 << a.shift;
    // Bytes of 64 keys: asked for while the 64 before are worked on - keys when their scores are done, values when their
    // product is - and their pages, of the key rows that this lane loads and of the keys that it owns, one round earlier.
    uint4 kw[4][DB], vw[DTILES];
    float ks = 0.f, vs = 0.f;
    bool ogood = false;
    int kpage = 0, opage = 0;
    const auto look_up = [&](int base) {
        kpage = table[min((base + 16 * (col >> 2)) >> a.shift, a.W - 1)];
        opage = table[min((base + 16 * g) >> a.shift, a.W - 1)];
    };
    const auto load_keys = [&](int base, int page) {
        const int key = base + 16 * (col >> 2) + (col & 3);
        const bool good = key < t.len && (unsigned)page < (unsigned)a.N;
        const unsigned char* kp = a.k_pages + (((int64_t)(good ? page : 0) * a.Hkv + h) * P + (key & (P - 1))) * D + g * 16;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int s = 0; s < DB; ++s) kw[i][s] = *reinterpret_cast<const uint4*>(kp + i * 4 * D + s * 64);
    };
    const auto load_values = [&](int base, int page) {
        const int key = base + 16 * g;
        ogood = key < hi && key + 16 > lo && (unsigned)page < (unsigned)a.N;
        const int64_t at = (int64_t)(ogood ? page : 0) * a.Hkv + h;
        const unsigned char* vp = a.v_pages + (at * D + col) * P + (key & (P - 1));
#pragma unroll
        for (int d = 0; d < DTILES; ++d) vw[d] = *reinterpret_cast<const uint4*>(vp + (int64_t)d * 16 * P);
        ks = ogood ? a.k_scale[at] * a.c : 0.f;
        vs = ogood ? a.v_scale[at] : 0.f;
    };
    if (kb + wid * 64 < kend) {
        look_up(kb + wid * 64);
        load_keys(kb + wid * 64, kpage);
        load_values(kb + wid * 64, opage);
        look_up(kb + wid * 64 + 256);
    }
    for (int base = kb + wid * 64; base < kend; base += 256) {
        const int okey = base + 16 * g;
        const bool more = base + 256 < kend;
        const int next_page = opage;

        f32x4_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < DB; ++s) {
                x[i] = Mat<DT>::mfma16(widen8<DT>(kw[i][s].x, kw[i][s].y, 1.f), qf[2 * s], x[i]);
                x[i] = Mat<DT>::mfma16(widen8<DT>(kw[i][s].z, kw[i][s].w, 1.f), qf[2 * s + 1], x[i]);
            }
            x[i] *= ks;
        }
        if (more) {
            load_keys(base + 256, kpage);
            look_up(base + 512);
        }
        // (a conversion reads only its scale's exponent: a scale of 0 has to clear the bytes instead)
        const bool ogive = ogood && vs != 0.f;
        const bool whole = base >= all_lo && base + 64 <= all_hi && __all(ogive);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = okey + 4 * i + j;
                    x[i][j] = ogood && key >= vis_lo && key < vis_hi ? x[i][j] : -INFINITY;
                }
        }
        float mx = x[0][0];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) mx = fmaxf(mx, x[i][j]);
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = fmaxf(m, mx), base_m = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m - base_m);   // 0 while nothing has been seen
        m = m_new;

        // Scale of the values.  bf16 has fp32's range: the conversion multiplies it in.  fp16 does not: the accumulator
        // is kept in units of the largest scale seen (`ref`), values are scaled by ratio >= 2^-15 (exact: e4m3's
        // smallest step is 2^-9, fp16's 2^-24), what is left of the ratio goes into the probabilities, and those are
        // raised by 2^14 so that neither falls under fp16's range.  All of it powers of two.  Ratios end at 2^-60: a
        // page that far under another has only zeros, or nothing that an fp16 output could show beside it.
        float raise = 0.f, vmul = ogood ? vs : 1.f, pscale = 1.f, oalpha = alpha;
        if constexpr (DT == PGN_F16) {
            float top = fmaxf(vs, __shfl_xor(vs, 16));
            top = fmaxf(ref, fmaxf(top, __shfl_xor(top, 32)));
            const float ratio = ogood ? fmaxf(vs / top, 0x1p-60f) : 1.f;
            oalpha *= ref > 0.f ? ref / top : 1.f;
            ref = top;
            vmul = fmaxf(ratio, 0x1p-15f);
            pscale = 0x1p-14f * (vmul / ratio);              // undoes the raise in the sum of probabilities
            raise = (float)(127 - (int)(__float_as_uint(pscale) >> 23));
        }
        float sum = 0.f;
        const float off = base_m - raise;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i][j] = __builtin_amdgcn_exp2f(x[i][j] - off);
                sum += x[i][j];
            }
        l = l * alpha + sum * pscale;
#pragma unroll
        for (int d = 0; d < DTILES; ++d) o[d] *= oalpha;

        v8 p[2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) p[s][j] = Mat<DT>::one(x[2 * s + (j >> 2)][j & 3]);
        if (!whole) {
            // bytes that no row sees (behind the request, on a page that is not one) may hold anything: they count as 0
            const unsigned b0 = ogive ? key_bytes(okey, 0, lo, hi) : 0u, b1 = ogive ? key_bytes(okey, 1, lo, hi) : 0u;
            const unsigned b2 = ogive ? key_bytes(okey, 2, lo, hi) : 0u, b3 = ogive ? key_bytes(okey, 3, lo, hi) : 0u;
            unsigned bad = 0;
#pragma unroll
            for (int d = 0; d < DTILES; ++d) {
                vw[d].x &= b0;
                vw[d].y &= b1;
                vw[d].z &= b2;
                vw[d].w &= b3;
                bad |= nan_bytes(vw[d].x) | nan_bytes(vw[d].y) | nan_bytes(vw[d].z) | nan_bytes(vw[d].w);
            }
            if (__any(bad != 0)) {
                // A NaN value that some rows see and others do not: 0 * NaN would reach the others.  The NaN bytes go
                // through a product of their own, ones against ones, which says which outputs they belong to.
                v8 see[2];
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int key = okey + 8 * s + j;
                        see[s][j] = Mat<DT>::one(ogood && key >= vis_lo && key < vis_hi ? 1.f : 0.f);
                    }
#pragma unroll
                for (int d = 0; d < DTILES; ++d) {
                    unsigned* w = reinterpret_cast<unsigned*>(&vw[d]);
                    unsigned n[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const unsigned f = nan_bytes(w[j]) >> 7;      // 0x01 in the NaN bytes
                        n[j] = f * 0x38u;                             // e4m3 1.0
                        w[j] &= ~(f * 0xffu);
                    }
                    f32x4_t hit = {0.f, 0.f, 0.f, 0.f};
                    hit = Mat<DT>::mfma16(widen8<DT>(n[0], n[1], 1.f), see[0], hit);
                    hit = Mat<DT>::mfma16(widen8<DT>(n[2], n[3], 1.f), see[1], hit);
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[d][j] = hit[j] > 0.f ? NAN : o[d][j];
                }
            }
        }
#pragma unroll
        for (int d = 0; d < DTILES; ++d) {
            o[d] = Mat<DT>::mfma16(widen8<DT>(vw[d].x, vw[d].y, vmul), p[0], o[d]);
            o[d] = Mat<DT>::mfma16(widen8<DT>(vw[d].z, vw[d].w, vmul), p[1], o[d]);
        }
        if (more) load_values(base + 256, next_page);
    }

    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        lds_m[wid][col] = m;
        lds_l[wid][col] = l;
    }
    const float unit = DT == PGN_F16 ? ref * 0x1p-14f : 1.f;
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
        *reinterpret_cast<f32x4_t*>(lds + (wid * 16 + col) * D + d * 16 + g * 4) = o[d] * unit;
    __syncthreads();
    for (int e = tid; e < t.count * D; e += PGN_CA_THREADS) {
        const int rr = e / D, d = e - rr * D;
        float big = -INFINITY, den = 0.f, num = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) big = fmaxf(big, lds_m[w][rr]);
        const float at = big == -INFINITY ? 0.f : big;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(lds_m[w][rr] - at);
            den = fmaf(lds_l[w][rr], f, den);
            num = fmaf(lds[(w * 16 + rr) * D + d], f, num);
        }
        const int rw = t.first + rr, tok = t.begin + rw / a.G, hd = h * a.G + rw % a.G;
        if (!a.few_split || plan.splits == 1) {
            a.out[tok * a.o_st + hd * a.o_sh + d] = Cvt<DT>::from_f32(den == 0.f ? 0.f : num / den);
        } else {
            const int64_t at_row = ((int64_t)slot * 16 + rr) * a.Hkv + h;
            if (kb < kend) a.part_o[at_row * D + d] = num;
            if (d == 0) a.part_ml[at_row] = make_float2(big, den);
        }
    }
}

// The kernel for prompts: 128 rows of a request, 32 to a wave, 64 keys at a time.
//
// What bounds it is arithmetic: the matrix units are busy for 35 % of the time and the vector units for 49 %, mostly with
// the softmax (scaling, exp2, sum and rounding of 32 numbers a lane against 32 matrix instructions at head dim 128) and
// the widening of bytes, which is done ONCE per workgroup, on the way into LDS, not in every wave.  4 prompts of 2048
// tokens, 32 heads by 128: 520 to 535 us, 820 to 844 TFLOP/s (a library product of 16384^3 reaches 1346); in fp16 562.
// Taking 256 rows with 64 a wave (1234 us, one wave a SIMD), 256 rows with eight waves (515 against 517, but 147 against 80
// for a batch of short requests) or 32 keys at a time with three waves a SIMD (566) was not better.  Tiles of 16-bit keys
// [64][D] and transposed values [D][64] are double buffered; while one is used, the next one's bytes are in flight
// to registers.  Each wave fetches one 16-key chunk of a tile, which lies in one page.
//
// Keys are stored in the row order in which the 32x32 result hands its rows to lanes: row b + 4 h + 8 a of a half tile is
// key 16 h + 4 a + b, so a lane ends up with 16 consecutive keys of its query and the probabilities are, without any
// exchange, the second operand of O^T = V^T P^T.
// The reference that probabilities are taken against is not the running maximum: it stays as long as a lane's sum of
// probabilities says that none is above 2^8, so the common path takes no maximum and rescales nothing.
// The 16-byte units of a row are permuted by its number, so that 16 lanes that read one unit of 16 rows meet all 64 banks:
// rows of 128 bytes take two to go round them.
template <int ROW>
__device__ __forceinline__ int key_swizzle(int row) {
    return ROW == 64 ? (row >> 1) & 7 : row & 15;
}

template <int DT, int D>
struct BigTile {
    unsigned short k[64 * D];
    unsigned short v[D * 64];
};

template <int DT, int D>
struct BigLds {
    BigTile<DT, D> tile[2];
    float ks[2][4], raise[2][4], pscale[2][4], ref[2];
    int nan[2][4], live[2][4];
    unsigned short nans[2][4][D];                            // of each chunk and head dim: which of its 16 values are NaN
};

template <int DT, int D>
__global__ __launch_bounds__(256, (D == 256 ? 1 : 2)) void pgn_cached_rows128_kernel(const CachedArgs a) {
    typedef typename Mat<DT>::v8 v8;
    constexpr int L = D / 64, KS = D / 16, DTILES = D / 32;
    extern __shared__ unsigned char smem_big[];
    BigLds<DT, D>& s = *reinterpret_cast<BigLds<DT, D>*>(smem_big);
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int hf = lane >> 5, col = lane & 31;
    const int h = blockIdx.x % a.Hkv, split = blockIdx.y;    // heads fastest: a head's tiles share one XCD's L2
    TileRows t;
    if (!many_rows_tile<128>(a, a.big_tiles - 1 - (int)(blockIdx.x / a.Hkv), t)) return;     // a request's longest rows first
    int lo, hi;
    key_range(a, t, lo, hi);
    const int keys = split_keys(a, lo, hi, a.big_nsplit), kb = (lo & ~63) + split * keys, kend = min(hi, kb + keys);

    const int wrow = wid * 32;                               // first row of the wave in the tile
    const int mine = min(wrow + col, t.count - 1);           // rows past the last repeat it and are not written
    const int row = t.first + mine;
    const int token = t.begin + row / a.G, head = h * a.G + row % a.G;
    const int pos = t.len - t.n + row / a.G;
    const int vis_hi = a.causal ? min(t.len, pos + 1) : t.len;
    const int vis_lo = window_lo(a, pos);
    // keys that every row of the wave sees, and that any does
    const int pos0 = t.len - t.n + (t.first + min(wrow, t.count - 1)) / a.G;
    const int pos1 = t.len - t.n + (t.first + min(wrow + 31, t.count - 1)) / a.G;
    const int all_hi = a.causal ? min(t.len, pos0 + 1) : t.len, any_hi = a.causal ? min(t.len, pos1 + 1) : t.len;
    const int all_lo = window_lo(a, pos1), any_lo = window_lo(a, pos0);

    const bool flip = a.c < 0.f;                             // the maximum is taken before the scaling: c has to be positive
    const float c = fabsf(a.c);
    v8 qf[KS];
    {
        const unsigned short* qp = a.q + token * a.q_st + head * a.q_sh + hf * 8;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            uint4 w = *reinterpret_cast<const uint4*>(qp + i * 16);
            if (flip) {
                w.x ^= 0x80008000u;
                w.y ^= 0x80008000u;
                w.z ^= 0x80008000u;
                w.w ^= 0x80008000u;
            }
            qf[i] = __builtin_bit_cast(v8, w);
        }
    }
    f32x16_t o[DTILES];
#pragma unroll
    for (int d = 0; d < DTILES; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -INFINITY, l = 0.f, ref = 0.f;

    const int* table = a.table + t.r * a.table_stride;
    const int P = 1 << a.shift;
    const int chunk = wid;                                   // of 16 keys of a tile, which the wave fetches
    uint4 kw[L], vw[L];
    bool good = false;                                       // the wave's chunk lies on a page
    // Pages and scales of the tile's chunks, chunk lane % 4 in each lane: scalar loads would be waited for together with the
    // LDS reads of the tile that is worked on.  Pages are looked up one tile ahead.
    const auto page_at = [&](int base) { return table[min((base + 16 * (lane & 3)) >> a.shift, a.W - 1)]; };
    int page = page_at(kb);
    float ks = 0.f, vs = 0.f;
    bool on_page = false;
    const auto of_chunk = [&](float v, int w) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), w)); };

    // bytes of the wave's chunk of the tile at `base`, and the scales of the tile
    auto fetch = [&](int base) {
        const int key = base + 16 * chunk, lkey = base + 16 * (lane & 3);
        on_page = lkey < hi && lkey + 16 > lo && (unsigned)page < (unsigned)a.N;
        const int own = __builtin_amdgcn_readlane(on_page ? page : -1, chunk);
        good = own >= 0;
        const int64_t at = (int64_t)(good ? own : 0) * a.Hkv + h, lat = (int64_t)(on_page ? page : 0) * a.Hkv + h;
        const unsigned char* kp = a.k_pages + (at * P + (key & (P - 1)) + (lane >> 2)) * D + (lane & 3) * 16;
#pragma unroll
        for (int i = 0; i < L; ++i) kw[i] = *reinterpret_cast<const uint4*>(kp + i * 64);
        const unsigned char* vp = a.v_pages + (at * D + lane) * P + (key & (P - 1));
#pragma unroll
        for (int i = 0; i < L; ++i) vw[i] = *reinterpret_cast<const uint4*>(vp + (int64_t)i * 64 * P);
        ks = a.k_scale[lat];
        vs = a.v_scale[lat];
        page = page_at(base + 64);
    };
    float store_ref = 0.f;
    auto store = [&](int base, int buf) {
        BigTile<DT, D>& tile = s.tile[buf];
        const float kscale = of_chunk(ks, chunk), vlane = on_page ? vs : 0.f, vscale = of_chunk(vlane, chunk);
        const int key = lane >> 2, mrow = (key & 3) + 4 * (chunk & 1) + 8 * (key >> 2);
        unsigned short* kp = tile.k + (32 * (chunk >> 1) + mrow) * D;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int u = (lane & 3) * 2 + i * 8;
            *reinterpret_cast<v8*>(kp + ((u ^ key_swizzle<D>(mrow)) * 8)) = widen8<DT>(kw[i].x, kw[i].y, 1.f);
            *reinterpret_cast<v8*>(kp + (((u + 1) ^ key_swizzle<D>(mrow)) * 8)) = widen8<DT>(kw[i].z, kw[i].w, 1.f);
        }
        if (lane == 0) {
            s.ks[buf][chunk] = fmaxf(good ? kscale * c : c, 0x1p-126f);      // 0 would turn a masked -inf into NaN
            s.live[buf][chunk] = good;
        }
        float vmul = 1.f, raise = 0.f, pscale = 1.f;
        if constexpr (DT == PGN_F16) {                   // as in the 16-row kernel, raised by 2^7: probabilities reach 2^8
            store_ref = fmaxf(store_ref, fmaxf(fmaxf(of_chunk(vlane, 0), of_chunk(vlane, 1)),
                                               fmaxf(of_chunk(vlane, 2), of_chunk(vlane, 3))));
            const float ratio = good ? fmaxf(vscale / store_ref, 0x1p-60f) : 1.f;
            vmul = fmaxf(ratio, 0x1p-15f);
            pscale = 0x1p-7f * (vmul / ratio);
            raise = (float)(127 - (int)(__float_as_uint(pscale) >> 23));
        } else {
            vmul = good ? vscale : 1.f;
        }
        // bytes that no row sees may hold anything: they count as 0, as do those of a page whose scale is 0
        const int vkey = base + 16 * chunk;
        if (vkey < lo || vkey + 16 > hi || vscale == 0.f) {
            const bool give = good && vscale != 0.f;
            const unsigned b0 = give ? key_bytes(vkey, 0, lo, hi) : 0u, b1 = give ? key_bytes(vkey, 1, lo, hi) : 0u;
            const unsigned b2 = give ? key_bytes(vkey, 2, lo, hi) : 0u, b3 = give ? key_bytes(vkey, 3, lo, hi) : 0u;
#pragma unroll
            for (int i = 0; i < L; ++i) {
                vw[i].x &= b0;
                vw[i].y &= b1;
                vw[i].z &= b2;
                vw[i].w &= b3;
            }
        }
        unsigned bad = 0;
#pragma unroll
        for (int i = 0; i < L; ++i)
            bad |= nan_bytes(vw[i].x) | nan_bytes(vw[i].y) | nan_bytes(vw[i].z) | nan_bytes(vw[i].w);
        const bool any_nan = __any(bad != 0);
        if (any_nan) {
            // A NaN value must reach the rows that see it and no other, but 0 * NaN would reach all.  It is kept
            // apart as a bit, and counts as 0 in the product.
#pragma unroll
            for (int i = 0; i < L; ++i) {
                unsigned bits = 0;
                unsigned* w = reinterpret_cast<unsigned*>(&vw[i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned f = nan_bytes(w[j]) >> 7;      // 0x01 in the NaN bytes
                    w[j] &= ~(f * 0xffu);
                    bits |= (((f * 0x01020408u) >> 24) & 15u) << (4 * j);     // byte n -> bit n
                }
                s.nans[buf][chunk][lane + 64 * i] = (unsigned short)bits;
            }
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int d = lane + 64 * i;
            unsigned short* vp = tile.v + d * 64;
            *reinterpret_cast<v8*>(vp + (((2 * chunk) ^ key_swizzle<64>(d)) * 8)) = widen8<DT>(vw[i].x, vw[i].y, vmul);
            *reinterpret_cast<v8*>(vp + (((2 * chunk + 1) ^ key_swizzle<64>(d)) * 8)) = widen8<DT>(vw[i].z, vw[i].w, vmul);
        }
        if (lane == 0) {
            s.raise[buf][chunk] = raise;
            s.pscale[buf][chunk] = pscale;
            s.nan[buf][chunk] = any_nan;
            s.ref[buf] = store_ref;
        }
    };

    if (kb < kend) {
        fetch(kb);
        store(kb, 0);
    }
    __syncthreads();
    for (int base = kb, buf = 0; base < kend; base += 64, buf ^= 1) {
        const bool more = base + 64 < kend;
        if (more) fetch(base + 64);
        if (base < any_hi && base + 64 > any_lo) {
            const BigTile<DT, D>& tile = s.tile[buf];
            f32x16_t x[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
                for (int i = 0; i < 16; ++i) x[kt][i] = 0.f;
                const unsigned short* kp = tile.k + (32 * kt + col) * D;
#pragma unroll
                for (int i = 0; i < KS; ++i)
                    x[kt] = Mat<DT>::mfma32(*reinterpret_cast<const v8*>(kp + (((2 * i + hf) ^ key_swizzle<D>(col)) * 8)),
                                              qf[i], x[kt]);
            }
            const bool whole = base >= all_lo && base + 64 <= all_hi &&
                               (s.live[buf][0] & s.live[buf][1] & s.live[buf][2] & s.live[buf][3]);
            if (!whole) {
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) {
                    const bool live = s.live[buf][2 * kt + hf];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = base + 32 * kt + 16 * hf + i;
                        x[kt][i] = live && key >= vis_lo && key < vis_hi ? x[kt][i] : -INFINITY;
                    }
                }
            }
            if constexpr (DT == PGN_F16) {
                const float now = s.ref[buf];
                if (now != ref) {                            // another unit for the accumulator
                    const float f = ref > 0.f ? ref / now : 1.f;
                    ref = now;
#pragma unroll
                    for (int d = 0; d < DTILES; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] *= f;
                }
            }
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const float kc = s.ks[buf][2 * kt + hf];
                const float raise = DT == PGN_F16 ? s.raise[buf][2 * kt + hf] : 0.f;
                const float pscale = DT == PGN_F16 ? s.pscale[buf][2 * kt + hf] : 1.f;
                f32x16_t e;
                float off = (m == -INFINITY ? 0.f : m) - raise, sum = 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    e[i] = __builtin_amdgcn_exp2f(fmaf(x[kt][i], kc, -off));
                    sum += e[i];
                }
                sum *= pscale;
                // a sum up to 2^8 says that no probability is above; otherwise, and while a row has seen nothing, the
                // reference moves to the maximum
                if (__any(!(sum <= 256.f) || m == -INFINITY)) {
                    float mx = x[kt][0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[kt][i]);
                    mx *= kc;
                    mx = fmaxf(mx, __shfl_xor(mx, 32));
                    const float m_new = fmaxf(m, mx);
                    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
                    m = m_new;
                    l *= alpha;
#pragma unroll
                    for (int d = 0; d < DTILES; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
                    off = (m == -INFINITY ? 0.f : m) - raise;
                    sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        e[i] = __builtin_amdgcn_exp2f(fmaf(x[kt][i], kc, -off));
                        sum += e[i];
                    }
                    sum *= pscale;
                }
                l += sum;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    v8 p;
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[j] = Mat<DT>::one(e[8 * half + j]);
#pragma unroll
                    for (int d = 0; d < DTILES; ++d) {
                        const unsigned short* vp = tile.v + (32 * d + col) * 64;
                        o[d] = Mat<DT>::mfma32(
                            *reinterpret_cast<const v8*>(vp + (((4 * kt + 2 * hf + half) ^ key_swizzle<64>(col)) * 8)), p, o[d]);
                    }
                }
            }
            if (s.nan[buf][0] | s.nan[buf][1] | s.nan[buf][2] | s.nan[buf][3]) {
                for (int w = 0; w < 4; ++w) {
                    if (!s.nan[buf][w]) continue;
                    unsigned see = 0;                        // of the chunk's keys
                    for (int i = 0; i < 16; ++i) {
                        const int key = base + 16 * w + i;
                        see |= key >= vis_lo && key < vis_hi ? 1u << i : 0u;
                    }
#pragma unroll
                    for (int d = 0; d < DTILES; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            o[d][i] = see & s.nans[buf][w][32 * d + 8 * (i >> 2) + 4 * hf + (i & 3)] ? NAN : o[d][i];
                }
            }
        }
        if (more) store(base + 64, buf ^ 1);
        __syncthreads();
    }

    l += __shfl_xor(l, 32);
    const float unit = DT == PGN_F16 ? ref * 0x1p-7f : 1.f;
    if (wrow + col >= t.count) return;
    if (a.big_nsplit == 1) {
        const float inv = l == 0.f ? 0.f : unit / l;
        unsigned short* op = a.out + token * a.o_st + head * a.o_sh;
#pragma unroll
        for (int d = 0; d < DTILES; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                u16x4_t w;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = Cvt<DT>::from_f32(l == 0.f ? 0.f : o[d][4 * q + j] * inv);
                unsigned short* p = op + d * 32 + q * 8 + hf * 4;
                if (a.out_vec) {
                    *reinterpret_cast<u16x4_t*>(p) = w;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) p[j] = w[j];
                }
            }
    } else {
        const int64_t at_row = ((int64_t)split * a.T + token) * a.Hq + head;
        if (kb < kend) {
#pragma unroll
            for (int d = 0; d < DTILES; ++d)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x4_t w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = o[d][4 * q + j] * unit;
                    *reinterpret_cast<f32x4_t*>(a.big_part_o + at_row * D + d * 32 + q * 8 + hf * 4) = w;
                }
        }
        if (hf == 0) a.big_part_ml[at_row] = make_float2(m, l);
    }
}

// Joins the splits of the rows of one kernel's tiles, a wave a row, four rows a workgroup.  Each lane takes one split's
// maximum and sum (64 splits at most), so that every weight is known before the first partial output is read and the
// reads do not wait for one another.
template <int DT, int D, int ROWS>
__global__ __launch_bounds__(PGN_CA_THREADS) void pgn_cached_join_kernel(const CachedArgs a) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TileRows t;
    const int h = blockIdx.x % a.Hkv, tile = blockIdx.x / a.Hkv;
    if (!(ROWS > 16 ? many_rows_tile<ROWS>(a, tile, t) : few_rows_tile(a, tile, t))) return;
    const int rr = blockIdx.y * 4 + wid;
    if (rr >= t.count) return;
    int nsplit = a.big_nsplit;
    int64_t row = 0, step = 0;
    if constexpr (ROWS == 16) {
        const int4 plan = a.plans[t.r];
        nsplit = plan.y;
        if (nsplit == 1) return;                             // is in `out` already
        row = ((int64_t)(plan.z + t.first / 16) * 16 + rr) * a.Hkv + h;
        step = (int64_t)plan.x * 16 * a.Hkv;
    }
    const int rw = t.first + rr, tok = t.begin + rw / a.G, hd = h * a.G + rw % a.G;
    if constexpr (ROWS > 16) {
        row = (int64_t)tok * a.Hq + hd;
        step = (int64_t)a.T * a.Hq;
    }
    const float2* part_ml = ROWS > 16 ? a.big_part_ml : a.part_ml;
    const float2 ml = lane < nsplit ? part_ml[lane * step + row] : make_float2(-INFINITY, 0.f);
    float big = ml.x;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor(big, off));
    const float at = big == -INFINITY ? 0.f : big;
    const float f = __builtin_amdgcn_exp2f(ml.x - at);
    // a split that saw nothing has written no output
    uint64_t seen = __ballot(!(ml.x == -INFINITY && ml.y == 0.f));
    float den = ml.y * f;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) den += __shfl_xor(den, off);
    float num[E] = {};
    const float* part = (ROWS > 16 ? a.big_part_o : a.part_o) + row * D + lane;
    while (seen) {
        float w[8], v[8][E];
#pragma unroll
        for (int i = 0; i < 8; ++i) {                        // eight splits at a time; the last ones may repeat, weighing 0
            const int s = seen ? __builtin_ctzll(seen) : 0;
            w[i] = seen ? __shfl(f, s) : 0.f;
            const bool on = seen != 0;
            seen &= seen - 1;
#pragma unroll
            for (int e = 0; e < E; ++e) v[i][e] = on ? part[s * step * D + e * 64] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) num[e] = fmaf(v[i][e], w[i], num[e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        a.out[tok * a.o_st + hd * a.o_sh + e * 64 + lane] = Cvt<DT>::from_f32(den == 0.f ? 0.f : num[e] / den);
}

struct CachedPlan {
    int tiles, tiles_per_request, few_split, few_slots;      // 16-row kernel
    int big_tiles, big_nsplit;                               // 128-row kernel; no tiles: not launched
};

// Splits of the 128-row kernel's keys so that 512 workgroups are there, which is what the CUs hold at a time.
static int splits(int64_t wgs, int64_t max_keys) {
    const int64_t most = (max_keys + PGN_CA_LEAST_KEYS - 1) / PGN_CA_LEAST_KEYS;
    int64_t n = (512 + wgs - 1) / wgs;
    n = n < most ? n : most;
    return (int)(n < 1 ? 1 : (n > 64 ? 64 : n));
}

static CachedPlan cached_plan(int T, int R, bool packed, int G, int Hkv, int D, int64_t max_keys) {
    CachedPlan p;
    const int few = packed ? (PGN_CA_FEW_ROWS < (int64_t)T * G ? PGN_CA_FEW_ROWS : T * G) : G;
    p.tiles_per_request = (few + 15) / 16;
    p.tiles = R * p.tiles_per_request;
    // Enough tiles for all CUs are split only in wide tables, where one long request would go on alone (16 requests of 32
    // heads, one of 65519 keys, the others of 500: 102 us instead of 476; all of 4000: 79 instead of 77), and not where
    // there are so many that this matters little, or that adding them up would.
    const int64_t tiles = (int64_t)p.tiles * Hkv, share = Hkv < few_resident(D) ? few_resident(D) / Hkv : 1;
    p.few_split = max_keys > PGN_CA_LEAST_KEYS && (tiles < few_resident(D) || max_keys > 8192) && R <= 512 && tiles <= 4096;
    p.few_slots = !p.few_split ? p.tiles : (int)(R <= 64 && p.tiles < share ? share : p.tiles + share);
    p.big_tiles = packed && (int64_t)T * G > PGN_CA_FEW_ROWS ? (int)((int64_t)T * G / 128 + R) : 0;
    p.big_nsplit = p.big_tiles ? splits((int64_t)p.big_tiles * Hkv, max_keys) : 1;
    return p;
}

// Rows times splits of each kernel.  Splits end where there are 512 workgroups, so both are small (some 10^5) whatever
// the number of tokens is.
static int64_t few_parts(const CachedPlan& p, int Hkv) { return p.few_split ? (int64_t)p.few_slots * 16 * Hkv : 0; }
// behind them, room for the plans: 512 times 16 bytes in the outputs of two slots of one head of 64
static int64_t plan_parts(const CachedPlan& p, int Hkv) { return p.few_split ? 2 * 16 * (int64_t)Hkv : 0; }
static int64_t big_parts(const CachedPlan& p, int64_t rows) { return p.big_nsplit > 1 ? p.big_nsplit * rows : 0; }
static size_t cached_workspace(const CachedPlan& p, int64_t rows, int Hkv, int D) {
    return (size_t)(few_parts(p, Hkv) + plan_parts(p, Hkv) + big_parts(p, rows)) * (D * 4 + 8);
}

}  // namespace

static int cached_shift(int P) { return P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : -1; }

static bool cached_sizes(int T, int R, int Hq, int Hkv, int D, int W, int page_size) {
    return T > 0 && R > 0 && Hq > 0 && Hkv > 0 && D > 0 && W > 0 && page_size > 0 && Hq % Hkv == 0;
}

extern "C" size_t pgn_cached_attention_workspace_bytes(int num_tokens, int R, int packed, int Hq, int Hkv, int head_dim,
                                                       int W, int page_size) {
    if (!cached_sizes(num_tokens, R, Hq, Hkv, head_dim, W, page_size)) return 0;
    const CachedPlan p = cached_plan(num_tokens, R, packed != 0, Hq / Hkv, Hkv, head_dim, (int64_t)W * page_size);
    return cached_workspace(p, (int64_t)num_tokens * Hq, Hkv, head_dim);
}

extern "C" int pgn_cached_attention(const void* q, int dtype, const void* k_pages, const void* v_pages,
                                    const float* k_scale, const float* v_scale, const int32_t* table,
                                    int64_t table_stride, const int32_t* lens, const int32_t* starts, void* out,
                                    int num_tokens, int R, int Hq, int Hkv, int head_dim, int num_pages, int W,
                                    int page_size, int64_t q_st, int64_t q_sh, int64_t o_st, int64_t o_sh, float scale,
                                    int causal, int window, void* workspace, size_t workspace_bytes, void* stream) {
    if (q == nullptr || k_pages == nullptr || v_pages == nullptr || k_scale == nullptr || v_scale == nullptr ||
        table == nullptr || lens == nullptr || out == nullptr)
        return PGN_ERR_INVALID;
    if (!cached_sizes(num_tokens, R, Hq, Hkv, head_dim, W, page_size) || num_pages <= 0 || table_stride < W || window < 0 ||
        (window > 0 && !causal) || (starts == nullptr && num_tokens != R) || !(scale == scale))
        return PGN_ERR_INVALID;
    if (dtype != PGN_BF16 && dtype != PGN_F16) return PGN_ERR_UNSUPPORTED;
    const int shift = cached_shift(page_size);
    if (shift < 0 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return PGN_ERR_UNSUPPORTED;
    // positions are ints, and 64 splits of 512 keys more than there are may be counted
    if (((int64_t)W << shift) > PGN_CACHED_MAX_KEYS || Hkv > 65535 || R > (1 << 26) || (int64_t)num_tokens * (Hq / Hkv) > 0x7fffffff - 65536)
        return PGN_ERR_UNSUPPORTED;
    if (!pgn_aligned(q, 16) || q_st % 8 != 0 || q_sh % 8 != 0 || !pgn_aligned(k_pages, 16) || !pgn_aligned(v_pages, 16) ||
        !pgn_aligned(out, 2))
        return PGN_ERR_INVALID;
    const CachedPlan p = cached_plan(num_tokens, R, starts != nullptr, Hq / Hkv, Hkv, head_dim, (int64_t)W << shift);
    const int64_t widest = p.few_slots > p.tiles ? p.few_slots : p.tiles;
    if ((widest > p.big_tiles ? widest : p.big_tiles) * Hkv > PGN_MAX_GRID / PGN_CA_THREADS) return PGN_ERR_UNSUPPORTED;
    const size_t need = cached_workspace(p, (int64_t)num_tokens * Hq, Hkv, head_dim);
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !pgn_aligned(workspace, 16))) return PGN_ERR_INVALID;
    CachedArgs a;
    a.q = (const unsigned short*)q;
    a.k_pages = (const unsigned char*)k_pages;
    a.v_pages = (const unsigned char*)v_pages;
    a.k_scale = k_scale;
    a.v_scale = v_scale;
    a.table = table;
    a.lens = lens;
    a.starts = starts;
    a.out = (unsigned short*)out;
    const int64_t few = few_parts(p, Hkv), big = big_parts(p, (int64_t)num_tokens * Hq);
    a.part_o = (float*)workspace;
    a.plans = (int4*)(a.part_o + few * head_dim);
    a.big_part_o = a.part_o + (few + plan_parts(p, Hkv)) * head_dim;
    a.part_ml = (float2*)(a.big_part_o + big * head_dim);
    a.big_part_ml = a.part_ml + few;
    a.table_stride = table_stride;
    a.q_st = q_st;
    a.q_sh = q_sh;
    a.o_st = o_st;
    a.o_sh = o_sh;
    a.T = num_tokens;
    a.R = R;
    a.Hq = Hq;
    a.Hkv = Hkv;
    a.G = Hq / Hkv;
    a.W = W;
    a.shift = shift;
    a.N = num_pages;
    a.causal = causal != 0;
    a.window = window;
    a.few_split = p.few_split;
    a.few_slots = p.few_slots;
    a.tiles_per_request = p.tiles_per_request;
    a.big_nsplit = p.big_nsplit;
    a.big_tiles = p.big_tiles;
    a.out_vec = pgn_aligned(out, 8) && o_st % 4 == 0 && o_sh % 4 == 0;
    a.c = scale * 1.4426950408889634f;
    hipStream_t s = (hipStream_t)stream;
#define PGN_CA_KERNEL(kernel, lds, grid)                                                                               \
    do {                                                                                                               \
        if ((lds) > 64 * 1024 - 1024) {                                                                                \
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),                                  \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)(lds));                \
            if (e != hipSuccess) return (int)e;                                                                        \
        }                                                                                                              \
        hipLaunchKernelGGL(kernel, grid, dim3(PGN_CA_THREADS), lds, s, a);                                             \
        PGN_LAUNCH_CHECK();                                                                                            \
    } while (0)
#define PGN_CA_LAUNCH(DT, D)                                                                                           \
    do {                                                                                                               \
        if (p.big_tiles)                                                                                               \
            PGN_CA_KERNEL((pgn_cached_rows128_kernel<DT, D>), sizeof(BigLds<DT, D>),                                   \
                          dim3(Hkv * p.big_tiles, p.big_nsplit));                                                      \
        PGN_CA_KERNEL((pgn_cached_rows16_kernel<DT, D>), (size_t)4 * 16 * D * 4, dim3(Hkv * p.few_slots));       \
        if (p.few_split)                                                                                              \
            PGN_CA_KERNEL((pgn_cached_join_kernel<DT, D, 16>), 0, dim3(Hkv * p.tiles, 4));                             \
        if (p.big_nsplit > 1)                                                                                          \
            PGN_CA_KERNEL((pgn_cached_join_kernel<DT, D, 128>), 0, dim3(Hkv * p.big_tiles, 32));                       \
    } while (0)
#define PGN_CA_DIMS(DT)                                                                                                \
    do {                                                                                                               \
        if (head_dim == 64) PGN_CA_LAUNCH(DT, 64);                                                                     \
        else if (head_dim == 128) PGN_CA_LAUNCH(DT, 128);                                                              \
        else PGN_CA_LAUNCH(DT, 256);                                                                                   \
    } while (0)
    if (dtype == PGN_BF16) PGN_CA_DIMS(PGN_BF16);
    else PGN_CA_DIMS(PGN_F16);
#undef PGN_CA_DIMS
#undef PGN_CA_LAUNCH
#undef PGN_CA_KERNEL
    return PGN_OK;
}
