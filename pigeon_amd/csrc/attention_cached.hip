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
    float* part_o;
    float2* part_ml;
    int64_t table_stride, q_st, q_sh, o_st, o_sh;
    int T, R, Hq, Hkv, G, W, shift, N, causal, window, split_keys, nsplit, tiles_per_request;
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

// The rows of a workgroup: `rows` consecutive (token, head-in-group) pairs of one request, ROWS to a tile.  Tile numbers
// leave each request floor(start * G / ROWS) + r and up, which is room for its ceil(n * G / ROWS) tiles whatever the
// lengths are, so the launch needs to know only the number of tokens and requests.
struct TileRows {
    int r, first, count, begin, n, len;                      // first row of the tile in its request, its valid rows
};

template <int ROWS>
__device__ __forceinline__ bool find_tile(const CachedArgs& a, int tile, TileRows& t) {
    int local;
    if (a.starts == nullptr) {
        t.r = tile / a.tiles_per_request;
        local = tile - t.r * a.tiles_per_request;
        t.begin = t.r;
        t.n = 1;
    } else {
        int lo = 0, hi = a.R;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((int64_t)a.starts[mid] * a.G / ROWS + mid <= tile) lo = mid;
            else hi = mid;
        }
        t.r = lo;
        t.begin = a.starts[lo];
        const int end = a.starts[lo + 1];
        if (t.begin < 0 || end < t.begin || end > a.T) return false;
        t.n = end - t.begin;
        local = tile - (int)((int64_t)t.begin * a.G / ROWS + lo);
    }
    t.first = local * ROWS;
    t.count = min(ROWS, t.n * a.G - t.first);
    if (local < 0 || t.count <= 0) return false;
    const int64_t room = (int64_t)a.W << a.shift;
    const int len = a.lens[t.r];
    t.len = len < 0 ? 0 : (len > room ? (int)room : len);
    return true;
}

// Keys that any row of the tile sees: [lo, hi).
__device__ __forceinline__ void key_range(const CachedArgs& a, const TileRows& t, int& lo, int& hi) {
    const int pos0 = t.len - t.n + t.first / a.G, pos1 = t.len - t.n + (t.first + t.count - 1) / a.G;
    hi = a.causal ? max(0, min(t.len, pos1 + 1)) : t.len;
    lo = a.window ? max(0, pos0 - a.window + 1) : 0;
}

#define PGN_CA_THREADS 256

template <int DT, int D>
__global__ __launch_bounds__(PGN_CA_THREADS) void pgn_cached_rows16_kernel(const CachedArgs a) {
    typedef typename Mat<DT>::v8 v8;
    constexpr int DB = D / 64, DTILES = D / 16;
    extern __shared__ float lds[];                           // [4][16][D] partial outputs
    __shared__ float lds_m[4][16], lds_l[4][16];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int g = lane >> 4, col = lane & 15;
    const int h = blockIdx.y, split = blockIdx.z;
    TileRows t;
    if (!find_tile<16>(a, blockIdx.x, t)) return;
    int lo, hi;
    key_range(a, t, lo, hi);
    const int kb = (lo & ~63) + split * a.split_keys;
    const int kend = min(hi, kb + a.split_keys);

    const int row = t.first + min(col, t.count - 1);         // rows past the last repeat it and are not written
    const int token = t.begin + row / a.G, head = h * a.G + row % a.G;
    const int pos = t.len - t.n + row / a.G;
    const int vis_hi = a.causal ? min(t.len, pos + 1) : t.len;
    const int vis_lo = a.window ? max(0, pos - a.window + 1) : 0;
    // keys that every row of the tile sees
    const int all_hi = a.causal ? min(t.len, t.len - t.n + t.first / a.G + 1) : t.len;
    const int all_lo = a.window ? max(0, t.len - t.n + (t.first + t.count - 1) / a.G - a.window + 1) : 0;

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
    for (int base = kb + wid * 64; base < kend; base += 256) {
        // pages: of the key rows that this lane loads, and of the keys that it owns
        const int kkey = base + 16 * (col >> 2) + (col & 3), okey = base + 16 * g;
        const int kpage = table[min(kkey >> a.shift, a.W - 1)], opage = table[min(okey >> a.shift, a.W - 1)];
        const bool kgood = kkey < t.len && (unsigned)kpage < (unsigned)a.N;
        const bool ogood = okey < hi && okey + 16 > lo && (unsigned)opage < (unsigned)a.N;
        const unsigned char* kp = a.k_pages + (((int64_t)(kgood ? kpage : 0) * a.Hkv + h) * P + (kkey & (P - 1))) * D + g * 16;
        const unsigned char* vp = a.v_pages + (((int64_t)(ogood ? opage : 0) * a.Hkv + h) * D + col) * P + (okey & (P - 1));
        uint4 kw[4][DB], vw[DTILES];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int s = 0; s < DB; ++s) kw[i][s] = *reinterpret_cast<const uint4*>(kp + i * 4 * D + s * 64);
#pragma unroll
        for (int d = 0; d < DTILES; ++d) vw[d] = *reinterpret_cast<const uint4*>(vp + (int64_t)d * 16 * P);
        const float ks = ogood ? a.k_scale[(int64_t)opage * a.Hkv + h] * a.c : 0.f;
        const float vs = ogood ? a.v_scale[(int64_t)opage * a.Hkv + h] : 0.f;

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
        if (a.nsplit == 1) {
            a.out[tok * a.o_st + hd * a.o_sh + d] = Cvt<DT>::from_f32(den == 0.f ? 0.f : num / den);
        } else {
            const int64_t at_row = ((int64_t)split * a.T + tok) * a.Hq + hd;
            if (kb < kend) a.part_o[at_row * D + d] = num;
            if (d == 0) a.part_ml[at_row] = make_float2(big, den);
        }
    }
}

// Joins the splits of each row: the same tiles, one wave a row.
template <int DT, int D>
__global__ __launch_bounds__(PGN_CA_THREADS) void pgn_cached_join_kernel(const CachedArgs a) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, h = blockIdx.y;
    TileRows t;
    if (!find_tile<16>(a, blockIdx.x, t)) return;
    for (int rr = wid; rr < t.count; rr += 4) {
        const int rw = t.first + rr, tok = t.begin + rw / a.G, hd = h * a.G + rw % a.G;
        const int64_t row = (int64_t)tok * a.Hq + hd, step = (int64_t)a.T * a.Hq;
        float big = -INFINITY;
        for (int s = 0; s < a.nsplit; ++s) big = fmaxf(big, a.part_ml[s * step + row].x);
        const float at = big == -INFINITY ? 0.f : big;
        float den = 0.f, num[E] = {};
        for (int s = 0; s < a.nsplit; ++s) {
            const float2 ml = a.part_ml[s * step + row];
            if (ml.x == -INFINITY && ml.y == 0.f) continue;  // nothing seen: its output was not written
            const float f = __builtin_amdgcn_exp2f(ml.x - at);
            den = fmaf(ml.y, f, den);
#pragma unroll
            for (int e = 0; e < E; ++e) num[e] = fmaf(a.part_o[(s * step + row) * D + e * 64 + lane], f, num[e]);
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            a.out[tok * a.o_st + hd * a.o_sh + e * 64 + lane] = Cvt<DT>::from_f32(den == 0.f ? 0.f : num[e] / den);
    }
}

struct CachedPlan {
    int tiles, tiles_per_request, nsplit, split_keys;
};

// Tiles and splits of a call.  Enough workgroups for every CU to hold four are wanted; a split is 256 keys at least (one
// round of the workgroup's four waves).
static CachedPlan cached_plan(int T, int R, bool packed, int G, int Hkv, int64_t max_keys) {
    CachedPlan p;
    p.tiles_per_request = (G + 15) / 16;
    p.tiles = packed ? (int)(((int64_t)T * G) / 16 + R) : R * p.tiles_per_request;
    const int64_t wgs = (int64_t)p.tiles * Hkv, most = (max_keys + 255) / 256;
    int64_t n = (1024 + wgs - 1) / wgs;
    n = n < most ? n : most;
    n = n < 1 ? 1 : (n > 64 ? 64 : n);
    p.split_keys = (int)(((max_keys + 64 + n - 1) / n + 255) / 256 * 256);
    p.nsplit = (int)((max_keys + 64 + p.split_keys - 1) / p.split_keys);
    return p;
}

}  // namespace

static int cached_shift(int P) { return P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : -1; }

static bool cached_sizes(int T, int R, int Hq, int Hkv, int D, int W, int page_size) {
    return T > 0 && R > 0 && Hq > 0 && Hkv > 0 && D > 0 && W > 0 && page_size > 0 && Hq % Hkv == 0;
}

extern "C" size_t pgn_cached_attention_workspace_bytes(int num_tokens, int R, int packed, int Hq, int Hkv, int head_dim,
                                                       int W, int page_size) {
    if (!cached_sizes(num_tokens, R, Hq, Hkv, head_dim, W, page_size)) return 0;
    const CachedPlan p = cached_plan(num_tokens, R, packed != 0, Hq / Hkv, Hkv, (int64_t)W * page_size);
    return p.nsplit == 1 ? 0 : (size_t)p.nsplit * num_tokens * Hq * (head_dim * 4 + 8);
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
    if (((int64_t)W << shift) > 0x7fffff00 - 65536 || Hkv > 65535 || (int64_t)num_tokens * (Hq / Hkv) > 0x7fffffff - 65536)
        return PGN_ERR_UNSUPPORTED;
    if (!pgn_aligned(q, 16) || q_st % 8 != 0 || q_sh % 8 != 0 || !pgn_aligned(k_pages, 16) || !pgn_aligned(v_pages, 16) ||
        !pgn_aligned(out, 2))
        return PGN_ERR_INVALID;
    const CachedPlan p = cached_plan(num_tokens, R, starts != nullptr, Hq / Hkv, Hkv, (int64_t)W << shift);
    const size_t need = p.nsplit == 1 ? 0 : (size_t)p.nsplit * num_tokens * Hq * (head_dim * 4 + 8);
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
    a.part_o = (float*)workspace;
    a.part_ml = need ? (float2*)((char*)workspace + (size_t)p.nsplit * num_tokens * Hq * head_dim * 4) : nullptr;
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
    a.split_keys = p.split_keys;
    a.nsplit = p.nsplit;
    a.tiles_per_request = p.tiles_per_request;
    a.c = scale * 1.4426950408889634f;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(p.tiles, Hkv, p.nsplit), join(p.tiles, Hkv), block(PGN_CA_THREADS);
    const size_t lds = (size_t)4 * 16 * head_dim * 4;        // 64 KiB at head dim 256
#define PGN_CA_LAUNCH(DT, D)                                                                                           \
    do {                                                                                                               \
        if (D == 256) {                                      /* 64 KiB and the maxima beside it */                     \
            hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(pgn_cached_rows16_kernel<DT, D>),         \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, 72 * 1024);                 \
            if (e != hipSuccess) return (int)e;                                                                        \
        }                                                                                                              \
        hipLaunchKernelGGL((pgn_cached_rows16_kernel<DT, D>), grid, block, lds, s, a);                                 \
        PGN_LAUNCH_CHECK();                                                                                            \
        if (p.nsplit > 1) {                                                                                            \
            hipLaunchKernelGGL((pgn_cached_join_kernel<DT, D>), join, block, 0, s, a);                                 \
            PGN_LAUNCH_CHECK();                                                                                        \
        }                                                                                                              \
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
    return PGN_OK;
}
