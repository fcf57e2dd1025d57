// Drawing token ids from logits (see include/pigeon_hip.h: pgn_sample_tokens).
//
// The weights w_i = exp((x_i - max) / temperature) are computed in 64 bits and rounded to whole multiples of 2^-45:
// sums of them are integers under 2^63 (2^18 ids), which are the same in any order, so atomics and any split of the row
// give the same ids every time.  The rounding is at most 2^-46 of the largest weight per id.
//
// One order ranks the ids: larger logit first, lower index first among equal ones.  As a 64-bit key - the logit's bits
// made monotone and complemented, then the index - "rank before" is "smaller key", and every filter keeps the ids up to
// some key: top-k the one where k ids, top-p the one where the wanted weight is reached.  That key is found without
// sorting the row: a histogram over the distance to the maximum (2048 bins, 32 to a factor of two of weight) says in
// which bin it lies, the few ids of that bin are gathered and sorted in LDS.
//
// One workgroup of 1024 threads takes a row and reads it two or three times: maximum, histogram (of ids for top-k, of
// weights for top-p), then either the gathering of the few ids that are left (top-k) or the sums of kept weights by
// stretches of the row, one of which holds the drawn id.  Only the first reading comes from HBM.
#include "pgn_common.h"

#define PGN_SAMPLE_THREADS 1024
#define PGN_SAMPLE_WAVES (PGN_SAMPLE_THREADS / 64)
#define PGN_SAMPLE_BINS 2048
#define PGN_SAMPLE_BINS_PER_OCTAVE 32.0f
#define PGN_SAMPLE_LIST 4096                                 // ids of one bin, or of a whole top-k, that are sorted in LDS
#define PGN_SAMPLE_TABLE 1024
#define PGN_SAMPLE_BITS 45

namespace {

typedef unsigned long long u64;

struct SampleArgs {
    const void* logits;
    const float* u;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int64_t* ids;
    int64_t stride;
    int V;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
};

struct SampleLds {
    u64 hist[PGN_SAMPLE_BINS];
    u64 key[PGN_SAMPLE_LIST];                                // the gathered ids
    u64 weight[PGN_SAMPLE_LIST];
    u64 seg[PGN_SAMPLE_MAX_IDS / 256 + PGN_SAMPLE_WAVES];    // kept weight of each 64 vectors (4 or 8 ids each) of the row
    double table[PGN_SAMPLE_TABLE];                          // 2^(-j / 1024)
    u64 part[PGN_SAMPLE_WAVES];
    u64 found, before;
    float fpart[PGN_SAMPLE_WAVES];
    int count, at;
};

// rank key of a logit: ascending keys are descending values
__device__ __forceinline__ unsigned rank_bits(float x) {
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}
__device__ __forceinline__ float rank_value(unsigned r) {
    return __uint_as_float((r & 0x80000000u) ? r : ~r & 0x7fffffffu);
}
__device__ __forceinline__ u64 rank_key(float x, int i) { return ((u64)rank_bits(x) << 24) | (unsigned)i; }

// NaN counts as a logit of -inf; -0 as 0, so that the two tie as they compare
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }

// A row in 16-byte vectors.  It may begin at any element: vector 0 is the aligned one that holds its first element, and
// vectors that reach over either end are put together from single loads.
template <int DT>
struct Row {
    typedef typename Cvt<DT>::storage S;
    static constexpr int E = 16 / (int)sizeof(S);
    const S* first;                                          // aligned, at most E - 1 elements before the row
    int lead, V, vectors;
    __device__ __forceinline__ Row(const void* p, int n) {
        lead = (int)(((uintptr_t)p & 15) / sizeof(S));
        first = reinterpret_cast<const S*>(p) - lead;
        V = n;
        vectors = (lead + n + E - 1) / E;
    }
    // elements of vector j; index of the first of them is j * E - lead
    __device__ __forceinline__ void load(int j, float* x) const {
        const int i0 = j * E - lead;
        S v[E];
        if (i0 >= 0 && i0 + E <= V) {
            *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(first + (int64_t)j * E);
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = clean(Cvt<DT>::to_f32(v[e]));
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                x[e] = i0 + e >= 0 && i0 + e < V ? clean(Cvt<DT>::to_f32(first[(int64_t)j * E + e])) : -INFINITY;
        }
    }
};

struct Weights {
    double max, c;                                           // c: 1024 log2(e) / temperature
    float fmax, fc;                                          // fc: bins per unit of distance
    bool infinite;                                           // the maximum is +inf: only its equals weigh anything
    const double* table;
    // w 2^45, nearest whole number.  2^-(t / 1024) with t = k + f, k whole, |f| <= 1/2: a table of 2^-(k % 1024 / 1024),
    // an exponent, and e^-(f ln2 / 1024) as its series up to the third power (the fourth is 2^-50).
    __device__ __forceinline__ u64 fixed(float x) const {
        if (infinite) return x == INFINITY ? 1ull << PGN_SAMPLE_BITS : 0;
        const double t = (max - (double)x) * c;
        if (!(t < 1024.0 * (PGN_SAMPLE_BITS + 2))) return x == fmax ? 1ull << PGN_SAMPLE_BITS : 0;
        const double d = t + 0x1.8p52;
        const int k = (int)(unsigned)(u64)__double_as_longlong(d);
        const double f = t - (d - 0x1.8p52);
        constexpr double c1 = -0.693147180559945309417 / 1024, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
        const double e = fma(fma(fma(c3, f, c2), f, c1), f, 1.0) * table[k & 1023];
        const double up = __hiloint2double((1023 + PGN_SAMPLE_BITS - (k >> 10)) << 20, 0);
        return (u64)__double_as_longlong(fma(e, up, 0x1p52)) & 0xfffffffffffffull;
    }
    // monotone in x: 32 bins to a factor of two, everything from 2^-64 on in the last
    __device__ __forceinline__ int bin(float x) const {
        const float y = x == fmax ? 0.f : (fmax - x) * fc;
        return (int)fminf(y, (float)(PGN_SAMPLE_BINS - 1));
    }
};

__device__ u64 block_sum(u64 v, u64* part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int w = 0; w < PGN_SAMPLE_WAVES; ++w) s += part[w];
    return s;
}

__device__ __forceinline__ u64 wave_scan(u64 v) {            // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const u64 o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    return v;
}

__device__ u64 block_scan(u64 v, u64* part, u64& total) {    // inclusive
    const int wid = threadIdx.x >> 6;
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) part[wid] = v;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PGN_SAMPLE_WAVES; ++w) {
        const u64 p = part[w];
        before += w < wid ? p : 0;
        all += p;
    }
    total = all;
    return v + before;
}

// hist[b] += v in one lane for the whole wave where all its lanes add to one bin (equal logits), else lane by lane
__device__ __forceinline__ void hist_add(u64* hist, int b, u64 v, bool on) {
    const uint64_t lanes = __ballot(on);
    if (lanes == 0) return;
    const int leader = __builtin_ctzll(lanes), b0 = __shfl(b, leader);
    if (__popcll(lanes) > 1 && __all(!on || b == b0)) {
        u64 s = on ? v : 0;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
        if ((int)(threadIdx.x & 63) == leader) atomicAdd(&hist[b0], s);
    } else if (on) {
        atomicAdd(&hist[b], v);
    }
}

// The key up to which the ids (of keys up to `limit`) hold `target` together, by eight bits of the key at a time over the
// whole row: for bins with more ids than the list takes.
template <int DT>
__device__ u64 select_key(SampleLds& s, const Row<DT>& row, const Weights& w, bool by_weight, u64 target, u64 limit) {
    u64 prefix = 0, before = 0;
    const int tid = threadIdx.x;
    for (int shift = 48; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int b = tid; b < 256; b += PGN_SAMPLE_THREADS) s.hist[b] = 0;
        __syncthreads();
        for (int j0 = 0; j0 < row.vectors; j0 += PGN_SAMPLE_THREADS) {
            float x[Row<DT>::E];
            const bool in = j0 + tid < row.vectors;
            if (in) row.load(j0 + tid, x);
#pragma unroll 1
            for (int e = 0; e < Row<DT>::E; ++e) {
                const float xe = in ? x[e] : -INFINITY;
                const u64 key = rank_key(xe, (j0 + tid) * Row<DT>::E - row.lead + e);
                const bool on = xe > -INFINITY && key <= limit && (key >> (shift + 8)) == prefix;
                const u64 v = !on ? 0 : by_weight ? w.fixed(xe) : 1;
                hist_add(s.hist, (int)(key >> shift) & 255, v, on && v > 0);
            }
        }
        __syncthreads();
        u64 total;
        const u64 v = tid < 256 ? s.hist[tid] : 0;
        const u64 c = before + block_scan(v, s.part, total);
        if (tid < 256 && v > 0 && c - v < target && c >= target) {
            s.found = (prefix << 8) | (unsigned)tid;
            s.before = c - v;
        }
        __syncthreads();
        prefix = s.found;
        before = s.before;
    }
    return prefix;
}

// Bin in which the running sum over the histogram reaches `target` (it does), and the sum before it.
__device__ int find_bin(SampleLds& s, u64 target, u64& before) {
    constexpr int PER = PGN_SAMPLE_BINS / PGN_SAMPLE_THREADS;
    u64 v[PER], sum = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        v[i] = s.hist[threadIdx.x * PER + i];
        sum += v[i];
    }
    u64 c = block_scan(sum, s.part, total) - sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (c < target && c + v[i] >= target) {
            s.at = threadIdx.x * PER + i;
            s.before = c;
        }
        c += v[i];
    }
    __syncthreads();
    before = s.before;
    const int b = s.at;
    __syncthreads();
    return b;
}

// Ascending sort of n keys (n a power of two, the list filled up to it), their weights with them.
__device__ void sort_list(SampleLds& s, int n) {
    for (int size = 2; size <= n; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < n / 2; i += PGN_SAMPLE_THREADS) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const u64 ka = s.key[a], kb = s.key[b];
                if ((ka > kb) == ((a & size) == 0)) {
                    s.key[a] = kb;
                    s.key[b] = ka;
                    const u64 wa = s.weight[a];
                    s.weight[a] = s.weight[b];
                    s.weight[b] = wa;
                }
            }
        }
    __syncthreads();
}

// Fills the list up to a power of two with what sorts last and weighs nothing.
__device__ int pad_list(SampleLds& s, int n) {
    int m = 2;
    while (m < n) m <<= 1;
    for (int i = n + threadIdx.x; i < m; i += PGN_SAMPLE_THREADS) {
        s.key[i] = ~0ull;
        s.weight[i] = 0;
    }
    return m;
}

// First place of the list at which the running sum of weights reaches `target`; n - 1 if none.  n <= 4 per thread.
__device__ int find_place(SampleLds& s, int n, u64 target, u64& total) {
    constexpr int PER = PGN_SAMPLE_LIST / PGN_SAMPLE_THREADS;
    u64 v[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = threadIdx.x * PER + i;
        v[i] = at < n ? s.weight[at] : 0;
        sum += v[i];
    }
    if (threadIdx.x == 0) s.at = n - 1;
    u64 c = block_scan(sum, s.part, total) - sum;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (v[i] > 0 && c < target && c + v[i] >= target) s.at = threadIdx.x * PER + i;
        c += v[i];
    }
    __syncthreads();
    const int at = s.at;
    __syncthreads();
    return at;
}

// what the sum has to exceed, as the least whole number that does: u times z, kept under z
__device__ __forceinline__ u64 draw_target(float u, u64 z) {
    const double r = u >= 0.f ? (double)u : 0.0;             // a NaN too
    const double cut = floor(r * (double)z);
    const u64 t = cut >= (double)z ? z - 1 : (u64)cut;
    return (t >= z ? z - 1 : t) + 1;
}

__device__ __forceinline__ u64 nucleus_target(float p, u64 z) {
    const double want = ceil((double)p * (double)z);
    const u64 t = want < 1.0 ? 1 : (u64)want;
    return t < z ? t : z;
}

template <int DT>
__global__ __launch_bounds__(PGN_SAMPLE_THREADS) void pgn_sample_tokens_kernel(const SampleArgs a) {
    extern __shared__ unsigned char smem[];
    SampleLds& s = *reinterpret_cast<SampleLds*>(smem);
    constexpr int E = Row<DT>::E;
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, b = blockIdx.x, V = a.V;
    const Row<DT> row(reinterpret_cast<const char*>(a.logits) + (int64_t)b * a.stride * sizeof(typename Cvt<DT>::storage), V);
    const float t = a.temperature ? a.temperature[b] : a.temperature_all;
    const int k = a.top_k ? a.top_k[b] : a.top_k_all;
    const float p = a.top_p ? a.top_p[b] : a.top_p_all;
    const float min_p = a.min_p ? a.min_p[b] : a.min_p_all;

    float m = -INFINITY;
    for (int j = tid; j < row.vectors; j += PGN_SAMPLE_THREADS) {
        float x[E];
        row.load(j, x);
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
    }
    for (int i = tid; i < PGN_SAMPLE_BINS; i += PGN_SAMPLE_THREADS) s.hist[i] = 0;
    s.table[tid] = exp2((double)tid * (-1.0 / PGN_SAMPLE_TABLE));
    if (tid == 0) s.count = 0;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    if (lane == 0) s.fpart[wid] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PGN_SAMPLE_WAVES; ++w) m = fmaxf(m, s.fpart[w]);
    if (m == -INFINITY) {                                    // nothing may be drawn
        if (tid == 0) a.ids[b] = -1;
        return;
    }
    if (!(t > 0.f) || p <= 0.f || k == 1) {                  // the first in rank: the lowest index of the largest logit
        int at = V;
        for (int j = tid; j < row.vectors; j += PGN_SAMPLE_THREADS) {
            float x[E];
            row.load(j, x);
#pragma unroll
            for (int e = E - 1; e >= 0; --e) at = x[e] == m ? min(at, j * E - row.lead + e) : at;
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) at = min(at, __shfl_xor(at, off));
        if (lane == 0) s.part[wid] = (u64)at;
        __syncthreads();
        if (tid == 0) {
            for (int w = 0; w < PGN_SAMPLE_WAVES; ++w) at = min(at, (int)s.part[w]);
            a.ids[b] = at;
        }
        return;
    }

    Weights w;
    w.max = m;
    w.fmax = m;
    w.infinite = m == INFINITY;
    w.c = PGN_SAMPLE_TABLE * 1.44269504088896340736 / (double)t;
    w.fc = (float)(PGN_SAMPLE_BINS_PER_OCTAVE * 1.44269504088896340736 / (double)t);
    w.table = s.table;
    u64 limit = ~0ull;                                       // keys up to it are kept

    if (k > 0 && k < V) {
        for (int j0 = 0; j0 < row.vectors; j0 += PGN_SAMPLE_THREADS) {
            float x[E];
            const bool in = j0 + tid < row.vectors;
            if (in) row.load(j0 + tid, x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xe = in ? x[e] : -INFINITY;
                hist_add(s.hist, w.bin(xe), 1, xe > -INFINITY);
            }
        }
        __syncthreads();
        u64 sum = 0;
        for (int i = tid; i < PGN_SAMPLE_BINS; i += PGN_SAMPLE_THREADS) sum += s.hist[i];
        if (block_sum(sum, s.part) > (u64)k) {
            u64 before;
            const int cut = find_bin(s, (u64)k, before);
            const u64 inside = s.hist[cut];
            const bool all = before + inside <= PGN_SAMPLE_LIST;
            if (all || inside <= PGN_SAMPLE_LIST) {          // all ids up to the bin's end, or those of the bin alone
                for (int j = tid; j < row.vectors; j += PGN_SAMPLE_THREADS) {
                    float x[E];
                    row.load(j, x);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int bin = w.bin(x[e]);
                        if (x[e] > -INFINITY && (bin == cut || (all && bin < cut))) {
                            const int at = atomicAdd(&s.count, 1);
                            s.key[at] = rank_key(x[e], j * E - row.lead + e);
                            s.weight[at] = 0;
                        }
                    }
                }
                __syncthreads();
                const int n = s.count;
                const int padded = pad_list(s, n);
                sort_list(s, padded);
                if (!all) {
                    limit = s.key[k - (int)before - 1];
                } else {                                     // the k ids are here: the rest is done in the list
                    for (int i = tid; i < k; i += PGN_SAMPLE_THREADS) s.weight[i] = w.fixed(rank_value((unsigned)(s.key[i] >> 24)));
                    __syncthreads();
                    int kept = k;
                    u64 z;
                    if (p < 1.f) {
                        u64 sum_k = 0;
                        for (int i = tid; i < k; i += PGN_SAMPLE_THREADS) sum_k += s.weight[i];
                        sum_k = block_sum(sum_k, s.part);
                        kept = find_place(s, k, nucleus_target(p, sum_k), z) + 1;
                    }
                    const int again = pad_list(s, kept);
                    const double least = (double)min_p * (double)(1ull << PGN_SAMPLE_BITS);
                    for (int i = tid; i < kept; i += PGN_SAMPLE_THREADS) {
                        const bool on = (double)s.weight[i] >= least || s.weight[i] == 1ull << PGN_SAMPLE_BITS;
                        s.weight[i] = on ? s.weight[i] : 0;
                        s.key[i] &= 0xffffff;                // by index now
                    }
                    sort_list(s, again);
                    u64 zero = 0;
                    for (int i = tid; i < kept; i += PGN_SAMPLE_THREADS) zero += s.weight[i];
                    z = block_sum(zero, s.part);
                    const int at = find_place(s, kept, draw_target(a.u[b], z), z);
                    if (tid == 0) a.ids[b] = (int64_t)s.key[at];
                    return;
                }
            } else {
                limit = select_key<DT>(s, row, w, false, (u64)k, limit);
            }
        }
        __syncthreads();
        for (int i = tid; i < PGN_SAMPLE_BINS; i += PGN_SAMPLE_THREADS) s.hist[i] = 0;
        if (tid == 0) s.count = 0;
        __syncthreads();
    }

    int cut = PGN_SAMPLE_BINS;                               // bins before it are kept whole (as far as `limit` goes)
    u64 target_p = 0, inside_target = 0;
    bool listed = false;
    if (p < 1.f) {
        for (int j0 = 0; j0 < row.vectors; j0 += PGN_SAMPLE_THREADS) {
            float x[E];
            const bool in = j0 + tid < row.vectors;
            if (in) row.load(j0 + tid, x);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float xe = in ? x[e] : -INFINITY;
                const u64 v = rank_key(xe, (j0 + tid) * E - row.lead + e) <= limit ? w.fixed(xe) : 0;
                hist_add(s.hist, w.bin(xe), v, v > 0);
            }
        }
        __syncthreads();
        u64 sum = 0, before;
        for (int i = tid; i < PGN_SAMPLE_BINS; i += PGN_SAMPLE_THREADS) sum += s.hist[i];
        target_p = nucleus_target(p, block_sum(sum, s.part));
        cut = find_bin(s, target_p, before);
        inside_target = target_p - before;
        listed = true;
    }

    // weights of what is kept, by stretches of 64 vectors; the ids of the bin with the border go to the list
    const double least = (double)min_p * (double)(1ull << PGN_SAMPLE_BITS);
    const int segs = (row.vectors + 63) >> 6;
    for (;;) {
        for (int g = wid; g < segs; g += PGN_SAMPLE_WAVES) {
            const int j = g * 64 + lane;
            u64 sum = 0;
            if (j < row.vectors) {
                float x[E];
                row.load(j, x);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const u64 key = rank_key(x[e], j * E - row.lead + e);
                    const int bin = w.bin(x[e]);
                    if (x[e] > -INFINITY && bin <= cut && key <= limit) {
                        const u64 v = w.fixed(x[e]);
                        if (listed && bin == cut) {
                            const int at = atomicAdd(&s.count, 1);
                            if (at < PGN_SAMPLE_LIST) {
                                s.key[at] = key;
                                s.weight[at] = v;
                            }
                        } else if ((double)v >= least || x[e] == m) {
                            sum += v;
                        }
                    }
                }
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
            if (lane == 0) s.seg[g] = sum;
        }
        __syncthreads();
        if (!listed || s.count <= PGN_SAMPLE_LIST) break;
        limit = select_key<DT>(s, row, w, true, target_p, limit);    // too many ids in the border's bin
        cut = PGN_SAMPLE_BINS;
        listed = false;
    }
    if (listed) {
        const int n = s.count, padded = pad_list(s, n);
        sort_list(s, padded);
        u64 total;
        const int last = find_place(s, n, inside_target, total);
        limit = min(limit, s.key[last]);
        for (int i = tid; i <= last; i += PGN_SAMPLE_THREADS) {
            const u64 v = s.weight[i];
            if ((double)v >= least || v == 1ull << PGN_SAMPLE_BITS)
                atomicAdd(&s.seg[((int)(s.key[i] & 0xffffff) + row.lead) / (64 * E)], v);
        }
        __syncthreads();
    }
    if (wid != 0) return;

    u64 z = 0;
    for (int g = lane; g < segs; g += 64) z += s.seg[g];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) z += __shfl_xor(z, off);
    const u64 target = draw_target(a.u[b], z);
    u64 before = 0;
    int g0 = 0;
    for (; g0 < segs; g0 += 64) {
        const u64 v = g0 + lane < segs ? s.seg[g0 + lane] : 0, c = wave_scan(v);
        const uint64_t over = __ballot(before + c >= target);
        if (over) {
            const int at = __builtin_ctzll(over);
            before += __shfl(c, at) - __shfl(v, at);
            g0 += at;
            break;
        }
        before += __shfl(c, 63);
    }
    const int j = g0 * 64 + lane;
    u64 v[E], sum = 0;
    float x[E];
    if (j < row.vectors) row.load(j, x);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        v[e] = 0;
        if (j < row.vectors && x[e] > -INFINITY && rank_key(x[e], j * E - row.lead + e) <= limit) {
            const u64 f = w.fixed(x[e]);
            if ((double)f >= least || x[e] == m) v[e] = f;
        }
        sum += v[e];
    }
    u64 c = before + wave_scan(sum) - sum;
    int hit = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (hit < 0 && c < target && c + v[e] >= target) hit = j * E - row.lead + e;
        c += v[e];
    }
    const uint64_t any = __ballot(hit >= 0);
    if (any && lane == __builtin_ctzll(any)) a.ids[b] = hit;
}

}  // namespace

extern "C" int pgn_sample_tokens(const void* logits, int dtype, int64_t stride, int B, int V, const float* u,
                                 const float* temperature, float temperature_all, const int32_t* top_k, int top_k_all,
                                 const float* top_p, float top_p_all, const float* min_p, float min_p_all, int64_t* ids,
                                 void* stream) {
    if (logits == nullptr || u == nullptr || ids == nullptr || B <= 0 || V <= 0 || stride < 0) return PGN_ERR_INVALID;
    if (dtype != PGN_F32 && dtype != PGN_BF16 && dtype != PGN_F16) return PGN_ERR_UNSUPPORTED;
    if (V > PGN_SAMPLE_MAX_IDS) return PGN_ERR_UNSUPPORTED;
    if (!pgn_aligned(logits, pgn_dtype_size(dtype))) return PGN_ERR_INVALID;
    SampleArgs a;
    a.logits = logits;
    a.u = u;
    a.temperature = temperature;
    a.top_k = top_k;
    a.top_p = top_p;
    a.min_p = min_p;
    a.ids = ids;
    a.stride = stride;
    a.V = V;
    a.temperature_all = temperature_all;
    a.top_k_all = top_k_all;
    a.top_p_all = top_p_all;
    a.min_p_all = min_p_all;
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(B), block(PGN_SAMPLE_THREADS);
#define PGN_SAMPLE_LAUNCH(DT)                                                                                         \
    do {                                                                                                              \
        hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(pgn_sample_tokens_kernel<DT>),               \
                                           hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(SampleLds));            \
        if (e != hipSuccess) return (int)e;                                                                           \
        hipLaunchKernelGGL((pgn_sample_tokens_kernel<DT>), grid, block, sizeof(SampleLds), s, a);                     \
    } while (0)
    if (dtype == PGN_F32) PGN_SAMPLE_LAUNCH(PGN_F32);
    else if (dtype == PGN_BF16) PGN_SAMPLE_LAUNCH(PGN_BF16);
    else PGN_SAMPLE_LAUNCH(PGN_F16);
#undef PGN_SAMPLE_LAUNCH
    PGN_LAUNCH_CHECK();
    return PGN_OK;
}
