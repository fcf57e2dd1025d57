// Block tables and the 8-bit paged key / value cache (see include/pigeon_hip.h: pgn_page_advance, pgn_cache_write).
//
// A page holds P tokens of one layer for every KV head: keys as [kv_heads][P][D] and values TRANSPOSED as
// [kv_heads][D][P], e4m3 bytes, each (page, head) with one fp32 scale for its keys and one for its values.  Values lie
// transposed because attention contracts them over tokens: a matrix instruction then takes 16 consecutive tokens of one
// head dim with a single 16-byte load, as it takes 16 consecutive head dims of one token's key.
// Scales are powers of two.  e4m3 is a floating-point type, so that costs no relative precision, and it makes every
// rescaling exact: a page whose scale has to grow when a larger token is appended is rewritten by an exponent shift
// that rounds only what falls under e4m3's subnormal step, however often it happens.
#include "pgn_common.h"

#include "pgn_fp8.h"

namespace {

// ------------------------------------------------------------------------------------------------ page_advance
// One workgroup does the bookkeeping: it is a chain of three prefix sums over the requests (pages given back, tokens
// added, pages wanted) whose results every later step needs, 4 bytes a request.  The pages themselves are then moved
// flat, four a thread at a time: a thread finds their requests by bisection in the prefix sums, which lie in LDS.
// A chain of short steps is bound by their latency, and a barrier of 16 waves is the longest of them, so a call takes no
// more waves than it has work for (us a call in a replayed graph, pages of 16, with 64, 256, 512 and 1024 threads):
//   64 requests and slots  4.2  4.8  5.5  6.5        512 requests and slots       21 8.5   5.7  6.8
//   64 and 512             8.1  5.6  5.3  6.6        512 and 4096                 55  19  11.6  9.8
//   256 and 256            12   5.1  5.4  6.7        512 and 16384, two launches  23  12  10.0 11.0
//   64 and 2048            23   10   7.8  7.6        16 and 8192, two launches   8.4 8.1   8.1  9.2
#define PGN_ADV_THREADS 1024
// Up to this many slots the bookkeeping workgroup fills the slot map itself (one launch); above it a second, wide launch
// does (512 requests, 4096 slots: 9.8 us against 11.0; 64 and 16384: 22 against 9.0).
#define PGN_ADV_FUSED_SLOTS 4096

__device__ __forceinline__ int64_t adv_pages(int64_t tokens, int shift) {
    return (tokens + ((int64_t)1 << shift) - 1) >> shift;
}

// inclusive prefix sum over the workgroup; `total` is the sum of all
template <int NT, typename I>
__device__ I adv_scan(I v, int64_t* wave_sums, I& total) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const I o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    if constexpr (NT == 64) {
        total = __shfl(v, 63);
        return v;
    } else {
        if (lane == 63) wave_sums[wid] = v;
        __syncthreads();
        I before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            const I x = (I)wave_sums[w];
            before += w < wid ? x : 0;
            all += x;
        }
        total = all;
        __syncthreads();
        return v + before;
    }
}

// last index i in [0, n) with at[i] <= x (at[] ascending, at[0] <= x)
__device__ __forceinline__ int adv_find(const int* at, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// the same of four numbers, in their places; n a power of two
__device__ __forceinline__ void adv_find4(const int* at, int n, int* x) {
    int lo[4] = {0, 0, 0, 0};
    for (int step = n >> 1; step > 0; step >>= 1) {
#pragma unroll
        for (int u = 0; u < 4; ++u) lo[u] += at[lo[u] + step] <= x[u] ? step : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = lo[u];
}

struct AdvRequest {
    int64_t held, keep, add;
    int have, kept;
};

__device__ __forceinline__ AdvRequest adv_request(const int* lens, const int* keep, const int* add, int r, int R, int W,
                                                  int shift) {
    AdvRequest q = {0, 0, 0, 0, 0};
    if (r < R) {
        const int64_t room = (int64_t)W << shift;
        const int64_t h = lens[r], k = keep ? keep[r] : h, a = add[r];
        q.held = h < 0 ? 0 : (h > room ? room : h);          // a length beyond the table names pages that do not exist
        q.keep = k < 0 ? 0 : (k > q.held ? q.held : k);
        q.add = a < 0 ? 0 : a;
        q.have = (int)adv_pages(q.held, shift);
        q.kept = (int)adv_pages(q.keep, shift);
    }
    return q;
}

template <int NT>
__global__ __launch_bounds__(NT) void pgn_page_advance_kernel(
    int* lens, const int* keep, const int* add, int* __restrict__ table, int64_t table_stride,
    int* __restrict__ free_pages, int* __restrict__ free_count, int N, int R, int W, int shift, int T, int fill_slots,
    int64_t* __restrict__ slots, int* __restrict__ starts, int* __restrict__ status) {
    __shared__ int64_t wave_sums[NT / 64];
    __shared__ int at[NT + 1];                               // prefix of what is being moved, within the chunk
    __shared__ int col[NT];                                  // first table column concerned (or the kept length)
    const int tid = threadIdx.x;
    AdvRequest q = adv_request(lens, keep, add, tid, R, W, shift);       // of the chunk at hand, here the first
    int64_t count = free_count[0];
    count = count < 0 ? 0 : (count > N ? N : count);

    // pages given back in all: the stack is filled so that popping returns them in request order
    int total, mine = q.have - q.kept, upto = adv_scan<NT>(mine, wave_sums, total);
    int64_t released = total;
    for (int r0 = NT; r0 < R; r0 += NT) {
        const AdvRequest o = adv_request(lens, keep, add, r0 + tid, R, W, shift);
        int more;
        adv_scan<NT>(o.have - o.kept, wave_sums, more);
        released += more;
    }
    if (released > 0) {
        int64_t done = 0;
        for (int r0 = 0;;) {
            at[tid] = upto - mine;
            col[tid] = q.kept;
            __syncthreads();
            for (int e0 = tid; e0 < total; e0 += 4 * NT) {
                int i[4], page[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) i[u] = min(e0 + u * NT, total - 1);
                adv_find4(at, NT, i);
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    page[u] = table[(r0 + i[u]) * table_stride + col[i[u]] + (min(e0 + u * NT, total - 1) - at[i[u]])];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t place = count + released - 1 - (done + e0 + u * NT);
                    if (e0 + u * NT < total && place < N)    // more pages back than the pool holds: a caller's mistake
                        free_pages[place] = page[u];
                }
            }
            done += total;
            __syncthreads();
            r0 += NT;
            if (r0 >= R) break;
            q = adv_request(lens, keep, add, r0 + tid, R, W, shift);
            mine = q.have - q.kept;
            upto = adv_scan<NT>(mine, wave_sums, total);
        }
        if (R > NT) q = adv_request(lens, keep, add, tid, R, W, shift);
    }
    int64_t top = count + released;
    top = top > N ? N : top;

    int64_t tokens = 0, wanted = 0, popped = 0;
    for (int r0 = 0; r0 < R; r0 += NT) {
        const int r = r0 + tid;
        if (r0 > 0) q = adv_request(lens, keep, add, r, R, W, shift);
        int64_t chunk_tokens;
        const int64_t end = tokens + adv_scan<NT>(q.add, wave_sums, chunk_tokens);
        const int64_t begin = end - q.add;
        tokens += chunk_tokens;
        const bool fits = r < R && q.keep + q.add <= ((int64_t)W << shift) && end <= T;
        int want = fits ? (int)adv_pages(q.keep + q.add, shift) - q.kept : 0;
        int first = adv_scan<NT>(want, wave_sums, total);
        bool ok = fits;
        if (wanted + total > top) {                          // not enough pages: nobody who needs some overtakes
            ok = fits && (want == 0 || wanted + first <= top);
            wanted += total;
            want = ok ? want : 0;
            first = adv_scan<NT>(want, wave_sums, total);
        } else {
            wanted += total;
        }
        first -= want;
        if (r < R) {
            lens[r] = (int)(ok ? q.keep + q.add : q.keep);
            status[r] = ok ? 0 : 1;
            starts[r + 1] = (int)(end < T ? end : T);
            if (r == 0) starts[0] = 0;
        }
        if (total > 0) {
            at[tid] = first;
            col[tid] = q.kept;
            __syncthreads();
            for (int e0 = tid; e0 < total; e0 += 4 * NT) {
                int i[4], page[4];                           // four at a time, so that their steps do not wait for one another
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = min(e0 + u * NT, total - 1);
                    page[u] = free_pages[top - 1 - popped - e];
                    i[u] = e;
                }
                adv_find4(at, NT, i);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = e0 + u * NT;
                    if (e < total) table[(r0 + i[u]) * table_stride + col[i[u]] + (e - at[i[u]])] = page[u];
                }
            }
            popped += total;
            __syncthreads();
        }
        if (fill_slots) {                                    // T <= PGN_ADV_FUSED_SLOTS here
            at[tid] = (int)(begin < T ? begin : T);
            if (tid == NT - 1) at[NT] = (int)(end < T ? end : T);
            col[tid] = ok ? (int)q.keep : -1;
            __syncthreads();
            for (int t = at[0] + tid; t < at[NT]; t += NT) {
                const int i = adv_find(at, NT, t);
                int64_t slot = -1;
                if (col[i] >= 0) {
                    const int pos = col[i] + (t - at[i]);
                    slot = ((int64_t)table[(r0 + i) * table_stride + (pos >> shift)] << shift) + (pos & ((1 << shift) - 1));
                }
                slots[t] = slot;
            }
            __syncthreads();
        }
    }
    if (fill_slots)
        for (int t = (int)(tokens < T ? tokens : T) + tid; t < T; t += NT) slots[t] = -1;
    if (tid == 0) free_count[0] = (int)(top - popped);
}

// The slot map of a large call: four consecutive tokens a thread, the request found by bisection in `starts`.
__global__ __launch_bounds__(256) void pgn_page_slots_kernel(const int* __restrict__ lens, const int* __restrict__ table,
                                                             int64_t table_stride, int R, int shift, int T,
                                                             int64_t* __restrict__ slots, const int* __restrict__ starts,
                                                             const int* __restrict__ status) {
    const int64_t t0 = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (t0 >= T) return;
    int r = adv_find(starts, R + 1, (int)t0);                // starts[R] <= t0: behind the last token
    int begin = 0, end = -1;
    int64_t base = -1;
    for (int j = 0; j < 4 && t0 + j < T; ++j) {
        const int t = (int)t0 + j;
        if (t >= end) {
            while (r < R && starts[r + 1] <= t) ++r;
            if (r < R) {
                begin = starts[r];
                end = starts[r + 1];
                base = status[r] ? -1 : (int64_t)lens[r] - (end - begin);
            } else {
                end = 0x7fffffff;
                base = -1;
            }
        }
        int64_t slot = -1;
        if (base >= 0) {
            const int pos = (int)base + (t - begin);
            slot = ((int64_t)table[r * table_stride + (pos >> shift)] << shift) + (pos & ((1 << shift) - 1));
        }
        slots[t] = slot;
    }
}

// ------------------------------------------------------------------------------------------------ cache_write
// A run is a stretch of consecutive tokens whose slots follow one another inside one page; the slot map makes at most
// one run of a page in a call.  One workgroup takes the runs that begin among its `chunk` tokens, for one head and one
// of the two halves, so it owns the (page, head) pairs that it writes: their scale is found, the older tokens of the
// page are rescaled if it grew, and the new ones are stored, with no exchange between workgroups.  Its four waves share
// a run of more than 16 tokens and take shorter ones each for itself.
//
// A wave keeps 16 rows in registers between finding the largest magnitude and storing, so a run of up to 64 tokens is
// read once.  Keys: 8 consecutive dims a lane, 16 bytes in and 8 out.  Values: the 16 page rows by D / 64 consecutive
// dims a lane, and they leave as they have to lie: the conversions pack four TOKENS of one dim, 16 tokens of a dim are
// one 16-byte store.

// The least power of two s >= 2^-100 with amax <= 448 s (448 = 1.75 * 2^8 is e4m3's largest value), from the bits.
__device__ __forceinline__ float cw_scale(float amax) {
    const unsigned u = __float_as_uint(amax);
    int k = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    k = k < PGN_CACHE_SCALE_FLOOR ? PGN_CACHE_SCALE_FLOOR : k;
    return __uint_as_float((unsigned)(k + 127) << 23);
}

// Magnitudes are compared as the 16-bit patterns that they are, two at a time (larger magnitude, larger pattern); from
// `CwInf` on they are not finite.
template <int DT>
struct CwInf {
    static constexpr unsigned bits = DT == PGN_BF16 ? 0x7f80u : 0x7c00u;
};
__device__ __forceinline__ unsigned cw_max2(unsigned amax, unsigned pair) {
    const u16x2_t m = __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, amax),
                                                __builtin_bit_cast(u16x2_t, pair & 0x7fff7fffu));
    return __builtin_bit_cast(unsigned, m);
}
// a pair with what is not finite left out
template <int DT>
__device__ __forceinline__ unsigned cw_finite2(unsigned pair) {
    const unsigned m = pair & 0x7fff7fffu;
    return ((m & 0xffffu) < CwInf<DT>::bits ? m & 0xffffu : 0) | ((m >> 16) < CwInf<DT>::bits ? m & 0xffff0000u : 0);
}

template <int DT>
__device__ __forceinline__ float cw_lo(unsigned pair) { return Cvt<DT>::to_f32((unsigned short)(pair & 0xffffu)); }
template <int DT>
__device__ __forceinline__ float cw_hi(unsigned pair) { return Cvt<DT>::to_f32((unsigned short)(pair >> 16)); }

// N consecutive elements in (N + 1) / 2 words
template <int N>
struct CwVec {
    unsigned w[(N + 1) / 2];
};

template <int N>
__device__ __forceinline__ CwVec<N> cw_load(const unsigned short* p, bool vec) {
    CwVec<N> v;
    if constexpr (N == 1) {
        v.w[0] = p[0];
    } else if (vec) {
        if constexpr (N == 8) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            v.w[0] = u.x, v.w[1] = u.y, v.w[2] = u.z, v.w[3] = u.w;
        } else if constexpr (N == 4) {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            v.w[0] = u.x, v.w[1] = u.y;
        } else {
            v.w[0] = *reinterpret_cast<const unsigned*>(p);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N / 2; ++j) v.w[j] = p[2 * j] | ((unsigned)p[2 * j + 1] << 16);
    }
    return v;
}

#define PGN_CW_WAVES 4

// The waves that work on a run together: all of the workgroup, or one.
struct CwTeam {
    int all, tid, threads;
    unsigned* wave_max;
};

// The largest pattern over the team.
__device__ __forceinline__ unsigned cw_team_max(unsigned amax, const CwTeam& g) {
    amax = max(amax & 0xffffu, amax >> 16);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) amax = max(amax, (unsigned)__shfl_xor((int)amax, off));
    if (g.all) {
        __syncthreads();                                     // what was there before has been read
        if ((g.tid & 63) == 0) g.wave_max[g.tid >> 6] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < PGN_CW_WAVES; ++w) amax = max(amax, g.wave_max[w]);
    }
    return amax;
}

// Tokens x[0 .. count) of one head, for rows row0 .. row0 + count of the page half at dst.
template <int DT, int D>
__device__ __forceinline__ void cw_keys(const unsigned short* x, int64_t x_st, bool vec, int row0, int count,
                                        unsigned char* dst, float* scale, const CwTeam& g) {
    constexpr int PER_ROW = D / 8, KEEP = PER_ROW / 4;       // 16 rows a wave in registers
    const int tid = g.tid, n = count * PER_ROW;
    const auto load = [&](int e) { return cw_load<8>(x + (int64_t)(e / PER_ROW) * x_st + (e % PER_ROW) * 8, vec); };
    CwVec<8> v[KEEP];
#pragma unroll
    for (int i = 0; i < KEEP; ++i) v[i] = load(min(tid + i * g.threads, n - 1));
    const float old = row0 > 0 ? *scale : 0.f;
    unsigned amax = 0;
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = cw_max2(amax, v[i].w[j]);
    for (int e = tid + KEEP * g.threads; e < n; e += g.threads) {            // a longer run: read again below
        const CwVec<8> u = load(e);
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = cw_max2(amax, u.w[j]);
    }
    unsigned top = cw_team_max(amax, g);
    const bool odd = top >= CwInf<DT>::bits;                 // infinities or NaN: they do not count
    if (odd) {
        amax = 0;
        for (int e = tid; e < n; e += g.threads) {
            const CwVec<8> u = load(e);
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = cw_max2(amax, cw_finite2<DT>(u.w[j]));
        }
        top = cw_team_max(amax, g);
    }
    const float s = fmaxf(cw_scale(cw_lo<DT>(top)), old), inv = 1.0f / s;        // exact: s is a power of two
    if (old < s && row0 > 0) {                               // older tokens of the page, under the larger scale
        const float f = old * inv;
        for (int e = tid; e < row0 * PER_ROW; e += g.threads) {
            uint2 w = *reinterpret_cast<const uint2*>(dst + e * 8);
            w.x = pgn_fp8_rescale4(w.x, f);
            w.y = pgn_fp8_rescale4(w.y, f);
            *reinterpret_cast<uint2*>(dst + e * 8) = w;
        }
    }
    const auto put = [&](int e, const CwVec<8>& u) {
        unsigned w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float f0 = cw_lo<DT>(u.w[2 * j]) * inv, f1 = cw_hi<DT>(u.w[2 * j]) * inv;
            const float f2 = cw_lo<DT>(u.w[2 * j + 1]) * inv, f3 = cw_hi<DT>(u.w[2 * j + 1]) * inv;
            w[j] = odd ? pgn_fp8_pack4_any(f0, f1, f2, f3) : pgn_fp8_pack4(f0, f1, f2, f3);
        }
        *reinterpret_cast<uint2*>(dst + (int64_t)row0 * D + e * 8) = uint2{w[0], w[1]};
    };
#pragma unroll
    for (int i = 0; i < KEEP; ++i)
        if (tid + i * g.threads < n) put(tid + i * g.threads, v[i]);
    for (int e = tid + KEEP * g.threads; e < n; e += g.threads) put(e, load(e));
    if (g.all) __syncthreads();                             // every thread has read the old scale
    if (tid == 0) *scale = s;
}

template <int DT, int D>
__device__ __forceinline__ void cw_values(const unsigned short* x, int64_t x_st, bool vec, int row0, int count, int P,
                                          unsigned char* dst, float* scale, const CwTeam& g) {
    constexpr int DV = D / 64, DW = (DV + 1) / 2;
    const int tid = g.tid, lane = tid & 63, wid = tid >> 6, waves = g.threads >> 6;
    const int slab0 = row0 >> 4, slabs = ((row0 + count + 15) >> 4) - slab0;     // slabs of 16 page rows that the run touches
    const auto row = [&](int slab, int j) { return (slab0 + slab) * 16 + j - row0; };    // token of the run, if in [0, count)
    const auto load = [&](int slab, CwVec<DV>* u) {
#pragma unroll
        for (int j = 0; j < 16; ++j)                         // rows outside the run repeat one of it: no branch, same maximum
            u[j] = cw_load<DV>(x + (int64_t)min(max(row(slab, j), 0), count - 1) * x_st + lane * DV, vec);
    };
    CwVec<DV> v[16];
    if (wid < slabs) {
        load(wid, v);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = CwVec<DV>{};
    }
    const float old = row0 > 0 ? *scale : 0.f;
    unsigned amax = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int d = 0; d < DW; ++d) amax = cw_max2(amax, v[j].w[d]);
    for (int slab = wid + waves; slab < slabs; slab += waves) {    // a longer run: read again below
        CwVec<DV> u[16];
        load(slab, u);
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int d = 0; d < DW; ++d) amax = cw_max2(amax, u[j].w[d]);
    }
    unsigned top = cw_team_max(amax, g);
    const bool odd = top >= CwInf<DT>::bits;
    if (odd) {
        amax = 0;
        for (int slab = wid; slab < slabs; slab += waves) {
            CwVec<DV> u[16];
            load(slab, u);
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
                for (int d = 0; d < DW; ++d) amax = cw_max2(amax, cw_finite2<DT>(u[j].w[d]));
        }
        top = cw_team_max(amax, g);
    }
    const float s = fmaxf(cw_scale(cw_lo<DT>(top)), old), inv = 1.0f / s;
    if (old < s && row0 > 0) {
        const float f = old * inv;
        const int words = (row0 + 3) >> 2;                   // the last word may hold tokens behind row0: bytes there
        for (int e = tid; e < D * words; e += g.threads) {
            const int d = e / words, w = e - d * words;
            unsigned char* p = dst + (int64_t)d * P + w * 4;
            const unsigned is = pgn_fp8_rescale4(*reinterpret_cast<const unsigned*>(p), f);
            if (w * 4 + 4 <= row0) {
                *reinterpret_cast<unsigned*>(p) = is;
            } else {
                for (int j = 0; w * 4 + j < row0; ++j) p[j] = (unsigned char)(is >> (8 * j));
            }
        }
    }
    const auto put = [&](int slab, const CwVec<DV>* u) {
        const bool whole = row(slab, 0) >= 0 && row(slab, 15) < count;
#pragma unroll
        for (int d = 0; d < DV; ++d) {
            unsigned char* p = dst + (int64_t)(lane * DV + d) * P + (slab0 + slab) * 16;
            unsigned w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = (d & 1 ? cw_hi<DT>(u[4 * j + i].w[d / 2]) : cw_lo<DT>(u[4 * j + i].w[d / 2])) * inv;
                w[j] = odd ? pgn_fp8_pack4_any(f[0], f[1], f[2], f[3]) : pgn_fp8_pack4(f[0], f[1], f[2], f[3]);
            }
            if (whole) {
                *reinterpret_cast<uint4*>(p) = uint4{w[0], w[1], w[2], w[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    if (row(slab, j) >= 0 && row(slab, j) < count) p[j] = (unsigned char)(w[j / 4] >> (8 * (j % 4)));
            }
        }
    };
    if (wid < slabs) put(wid, v);
    for (int slab = wid + waves; slab < slabs; slab += waves) {
        CwVec<DV> u[16];
        load(slab, u);
        put(slab, u);
    }
    if (g.all) __syncthreads();
    if (tid == 0) *scale = s;
}

template <int DT, int D>
__global__ __launch_bounds__(PGN_CW_WAVES * 64) void pgn_cache_write_kernel(
    const unsigned short* __restrict__ k, const unsigned short* __restrict__ v, const int64_t* __restrict__ slots, int T,
    int H, int shift, int64_t N, int chunk, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int k_vec, int v_vec,
    unsigned char* k_pages, unsigned char* v_pages, float* k_scale, float* v_scale) {
    __shared__ unsigned wave_max[PGN_CW_WAVES];
    // Workgroups go round the 8 XCDs.  One XCD takes all heads of a chunk, one after another: a token's heads lie side by
    // side, and an XCD that read only every eighth of them would use few of its L2's channels.
    const int lane = threadIdx.x & 63, xcd = blockIdx.x & 7, j = blockIdx.x >> 3, h = j % H;
    const int P = 1 << shift;
    const int64_t limit = N << shift;

    // which of the chunk's tokens begin a run: one lane a token, the same in every wave (chunk <= 64)
    const int t0 = (j / H * 8 + xcd) * chunk;                // may lie behind the last token: then nothing begins a run
    const int64_t my_slot = t0 + lane < T ? slots[t0 + lane] : -1;
    const int64_t next_slot = t0 + 64 + lane < T ? slots[t0 + 64 + lane] : -1;
    int64_t my_before = __shfl_up(my_slot, 1);
    if (lane == 0) my_before = t0 > 0 && t0 < T ? slots[t0 - 1] : -2;
    uint64_t runs = __ballot(lane < chunk && my_slot >= 0 && my_slot < limit &&
                             ((my_slot & (P - 1)) == 0 || my_before != my_slot - 1));
    int turn = threadIdx.x >> 6;                             // short runs until the wave's next
    for (; runs != 0; runs &= runs - 1) {                    // every bound here is the same for the whole workgroup
        const int first = __builtin_ctzll(runs), t = t0 + first;
        const int64_t slot = __shfl(my_slot, first);
        const int row0 = (int)(slot & (P - 1)), most = P - row0;
        // tokens of the run, up to the page's end: among the 128 that the lanes hold, then 64 at a time
        uint64_t on = ~__ballot(lane >= first && lane - first < most && my_slot == slot + (lane - first)) >> first;
        int count = on == 0 ? 64 - first : __builtin_ctzll(on);
        for (int c = 64 - first; count == c && c < most; c += 64) {
            const int64_t sl = c == 64 - first ? next_slot : t + c + lane < T ? slots[t + c + lane] : -1;
            on = ~__ballot(c + lane < most && sl == slot + (c + lane));
            count += on == 0 ? 64 : __builtin_ctzll(on);
        }
        const int64_t page = slot >> shift, half = (page * H + h) * (int64_t)P * D;
        CwTeam g = {1, (int)threadIdx.x, PGN_CW_WAVES * 64, wave_max};
        if (count <= 16) {
            if (turn-- != 0) continue;
            turn = PGN_CW_WAVES - 1;
            g.all = 0, g.tid = lane, g.threads = 64;
        }
        if (blockIdx.y == 0)
            cw_keys<DT, D>(k + (int64_t)t * k_st + h * k_sh, k_st, k_vec, row0, count, k_pages + half,
                           k_scale + page * H + h, g);
        else
            cw_values<DT, D>(v + (int64_t)t * v_st + h * v_sh, v_st, v_vec, row0, count, P, v_pages + half,
                             v_scale + page * H + h, g);
    }
}

}  // namespace

static int page_shift(int P) { return P == 16 ? 4 : P == 32 ? 5 : P == 64 ? 6 : P == 128 ? 7 : -1; }

extern "C" int pgn_page_advance(int32_t* lens, const int32_t* keep, const int32_t* add, int32_t* table,
                                int64_t table_stride, int32_t* free_pages, int32_t* free_count, int num_pages, int R,
                                int W, int page_size, int64_t num_slots, int64_t* slots, int32_t* starts,
                                int32_t* status, void* stream) {
    if (lens == nullptr || add == nullptr || table == nullptr || free_pages == nullptr || free_count == nullptr ||
        starts == nullptr || status == nullptr || (slots == nullptr && num_slots > 0))
        return PGN_ERR_INVALID;
    if (R <= 0 || W <= 0 || num_pages <= 0 || num_slots < 0 || table_stride < W) return PGN_ERR_INVALID;
    const int shift = page_shift(page_size);
    if (shift < 0 || num_slots > 0x7fffffff - 4 * 256) return PGN_ERR_UNSUPPORTED;
    if (((int64_t)W << shift) > 0x7fffffff || (int64_t)W * PGN_ADV_THREADS > 0x7fffffff) return PGN_ERR_UNSUPPORTED;
    hipStream_t s = (hipStream_t)stream;
    const int T = (int)num_slots, fused = T <= PGN_ADV_FUSED_SLOTS;
#define PGN_ADV_LAUNCH(NT)                                                                                             \
    hipLaunchKernelGGL((pgn_page_advance_kernel<NT>), dim3(1), dim3(NT), 0, s, lens, keep, add, table, table_stride,   \
                       free_pages, free_count, num_pages, R, W, shift, T, fused, slots, starts, status)
    // requests, rounds over the slots, or (a few slots each) pages to hand out
    const int per = fused ? T / 2 : T / 64, work = R > per ? R : per;
    if (work <= 64) PGN_ADV_LAUNCH(64);
    else if (work <= 256) PGN_ADV_LAUNCH(256);
    else if (work <= 512) PGN_ADV_LAUNCH(512);
    else PGN_ADV_LAUNCH(PGN_ADV_THREADS);
#undef PGN_ADV_LAUNCH
    PGN_LAUNCH_CHECK();
    if (!fused) {
        hipLaunchKernelGGL(pgn_page_slots_kernel, dim3((T + 1023) / 1024), dim3(256), 0, s, lens, table, table_stride, R,
                           shift, T, slots, starts, status);
        PGN_LAUNCH_CHECK();
    }
    return PGN_OK;
}

extern "C" int pgn_cache_write(const void* k, const void* v, int dtype, const int64_t* slots, int64_t num_tokens,
                               int kv_heads, int head_dim, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh,
                               void* k_pages, void* v_pages, float* k_scale, float* v_scale, int num_pages,
                               int page_size, void* stream) {
    if (k == nullptr || v == nullptr || slots == nullptr || k_pages == nullptr || v_pages == nullptr ||
        k_scale == nullptr || v_scale == nullptr)
        return PGN_ERR_INVALID;
    if (num_tokens <= 0 || kv_heads <= 0 || head_dim <= 0 || num_pages <= 0) return PGN_ERR_INVALID;
    if (dtype != PGN_BF16 && dtype != PGN_F16) return PGN_ERR_UNSUPPORTED;
    const int shift = page_shift(page_size);
    if (shift < 0 || (head_dim != 64 && head_dim != 128 && head_dim != 256) || kv_heads > 65535 ||
        num_tokens > 0x7fffffff - 1024)
        return PGN_ERR_UNSUPPORTED;
    if (!pgn_aligned(k, 2) || !pgn_aligned(v, 2) || !pgn_aligned(k_pages, 16) || !pgn_aligned(v_pages, 16))
        return PGN_ERR_INVALID;
    // keys are read 16 bytes at a time, values head_dim / 64 elements
    const int dv = head_dim / 64;
    const int k_vec = pgn_aligned(k, 16) && k_st % 8 == 0 && k_sh % 8 == 0;
    const int v_vec = pgn_aligned(v, 2 * dv) && v_st % dv == 0 && v_sh % dv == 0;
    const int T = (int)num_tokens;
    // Few tokens, for decoding: each a run of its own, one for each wave (64 tokens of 8 heads by 128: 5.9 us, 15.0 with
    // 16 tokens a workgroup, 51 with 64).  Many, for prompts: most lie inside a run that began before, and a workgroup
    // without a run costs its look at the slot map all the same (2048 tokens: 18.6, 10.8 and 5.1 us; as many runs of one
    // token: 42, 48 and 59 us).
    const int chunk = T <= 512 ? 4 : T <= 1024 ? 16 : 64;
    const int64_t wgs = (int64_t)(((T + chunk - 1) / chunk + 7) / 8 * 8) * kv_heads;
    if (wgs > PGN_MAX_GRID / (PGN_CW_WAVES * 64)) return PGN_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)wgs, 2);
    hipStream_t s = (hipStream_t)stream;
#define PGN_CW_LAUNCH(DT, D)                                                                                           \
    hipLaunchKernelGGL((pgn_cache_write_kernel<DT, D>), grid, dim3(PGN_CW_WAVES * 64), 0, s, (const unsigned short*)k, \
                       (const unsigned short*)v, slots, T, kv_heads, shift, (int64_t)num_pages, chunk, k_st, k_sh, v_st, \
                       v_sh, k_vec, v_vec, (unsigned char*)k_pages, (unsigned char*)v_pages, k_scale, v_scale)
#define PGN_CW_DIMS(DT)                                                                                                \
    do {                                                                                                               \
        if (head_dim == 64) PGN_CW_LAUNCH(DT, 64);                                                                     \
        else if (head_dim == 128) PGN_CW_LAUNCH(DT, 128);                                                              \
        else PGN_CW_LAUNCH(DT, 256);                                                                                   \
    } while (0)
    if (dtype == PGN_BF16) PGN_CW_DIMS(PGN_BF16);
    else PGN_CW_DIMS(PGN_F16);
#undef PGN_CW_DIMS
#undef PGN_CW_LAUNCH
    PGN_LAUNCH_CHECK();
    return PGN_OK;
}
