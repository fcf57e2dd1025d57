// Drawing token ids from logits (see include/pigeon_hip.h: pgn_sample_tokens).
//
// The weights w_i = exp((x_i - max) / temperature) are computed in 64 bits and rounded to whole multiples of 2^-45:
// sums of them are integers under 2^63 (2^18 ids), which are the same in any order, so atomics and any split of the row
// give the same ids every time.  The rounding is at most 2^-46 of the largest weight per id.
//
// One order ranks the ids: larger logit first, lower index first among equal ones.  As a 64-bit key - the logit's bits
// made monotone and complemented, then the index - "rank before" is "smaller key", and every filter keeps the ids up to
// some key: top-k the one where k ids, top-p the one where the wanted weight is reached.  That key is found without
// sorting the row, by bins over the distance to the maximum (2048 bins, 32 to a factor of two of weight).
//
// One workgroup of 1024 threads takes a row.  It is bound by what each id costs in the passes over the row, in
// instructions and in LDS, whose loads only the first time come from HBM, and for short rows by the steps between them, each
// with its barriers (some 20 of 0.3 us).  256 bf16 rows of 131072 with top-p take 91 us, 14 of them for the first pass (67 MB at
// 4.8 TB/s), 33 for the bins and 11 to 21 for the stretches; 64 rows of 48386 with a top-k of 50 19 us; one fp32 row 27 us.
//   top-k   the k-th largest of the 1024 threads' own maxima, known after the first pass, is at most the k-th largest
//           logit: one more pass gathers the ids up to its bin, some 1.1 k, and the rest (k, p, min-p, draw) is done
//           among those in LDS;
//   top-p   a pass adds the weights to the bins (whole numbers: an fp32 addition in LDS takes seven times as long), which
//           says in which bin the border is; the next pass gathers the ids of that bin, where the border is found by a
//           sort, and sums what is kept by stretches of the row.  A bin with more ids than the list takes (thousands of
//           equal logits) has its key searched for by digits;
//   draw    the stretch that the random number falls into is summed again by one wave.
#include "pgn_common.h"

#define PGN_SAMPLE_THREADS 1024
#define PGN_SAMPLE_WAVES (PGN_SAMPLE_THREADS / 64)
#define PGN_SAMPLE_BINS 2048
#define PGN_SAMPLE_BINS_PER_OCTAVE 32.0f
#define PGN_SAMPLE_LIST 4096                                 // ids that are sorted in LDS
#define PGN_SAMPLE_FEW 256                                   // ids that are compared each with each instead
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
    union {
        u64 mass[PGN_SAMPLE_BINS];
        unsigned ids[PGN_SAMPLE_BINS];
        u64 digit[256];
    } hist;
    u64 key[PGN_SAMPLE_LIST];                                // the gathered ids
    u64 weight[PGN_SAMPLE_LIST];
    u64 seg[PGN_SAMPLE_MAX_IDS / 256 + PGN_SAMPLE_WAVES];    // kept weight of each 64 vectors (4 or 8 ids each) of the row
    double table[PGN_SAMPLE_TABLE];                          // 2^(-j / 1024)
    u64 pile[PGN_SAMPLE_WAVES][128];                         // of each wave: kept logits and their indexes, 64 at a time
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
__device__ __forceinline__ float clean(float x) { return fmaxf(x + 0.f, -INFINITY); }

// A row in 16-byte vectors.  It may begin at any element: vector 0 is the aligned one that holds its first element.  The
// vectors that reach over an end are put together from single loads, with -inf where there is no id.
template <int DT>
struct Row {
    typedef typename Cvt<DT>::storage S;
    static constexpr int E = 16 / (int)sizeof(S);
    const S* first;                                          // aligned, at most E - 1 elements before the row
    int lead, V, vectors, whole_lo, whole_hi;                // vectors [whole_lo, whole_hi) lie inside the row
    __device__ __forceinline__ Row(const void* p, int n) {
        lead = (int)(((uintptr_t)p & 15) / sizeof(S));
        first = reinterpret_cast<const S*>(p) - lead;
        V = n;
        vectors = (lead + n + E - 1) / E;
        whole_lo = lead > 0;
        whole_hi = (lead + n) / E;
    }
    __device__ __forceinline__ float one(int i) const { return clean(Cvt<DT>::to_f32(first[lead + i])); }
    // index of element e of vector j
    __device__ __forceinline__ int index(int j, int e) const { return j * E - lead + e; }
    static __device__ __forceinline__ void unpack(const uint4& r, float* x) {
        const unsigned w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < E; ++e) {
            if constexpr (DT == PGN_F32)
                x[e] = clean(__uint_as_float(w[e]));
            else
                x[e] = clean(Cvt<DT>::to_f32((unsigned short)(e & 1 ? w[e / 2] >> 16 : w[e / 2] & 0xffffu)));
        }
    }
    // any vector, one element at a time
    __device__ __forceinline__ void pick(int j, float* x) const {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = index(j, e);
            x[e] = j < vectors && i >= 0 && i < V ? one(i) : -INFINITY;
        }
    }
    // f(j, x[E]) for every vector of the row, in all threads equally often, some with vectors that hold nothing.  Vector j
    // is thread j % 1024's.  The loads are free of branches and AHEAD of them are in flight: four where the work on a vector
    // is short, one where it hides the next load (every copy of the body is instructions to fetch, once a launch).
    template <int AHEAD, typename F>
    __device__ __forceinline__ void each(F f) const {
        const int tid = threadIdx.x;
        const auto load = [&](int j) {
            return *reinterpret_cast<const uint4*>(first + (int64_t)min(max(j, whole_lo), whole_hi - 1) * E);
        };
        uint4 r[AHEAD];
        if (whole_hi > whole_lo) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) r[u] = load(u * PGN_SAMPLE_THREADS + tid);
        }
        const int rounds = whole_hi > whole_lo ? (whole_hi + PGN_SAMPLE_THREADS - 1) / PGN_SAMPLE_THREADS : 0;
        const int all = rounds + (whole_lo > 0 || whole_hi < vectors);       // one more for the ends, two vectors at most
        const int last = vectors - 1;
        const int end = tid == 0 && whole_lo > 0 ? 0 : tid == 1 && whole_hi < vectors && (last > 0 || whole_lo == 0) ? last : vectors;
#pragma unroll 1
        for (int i0 = 0; i0 < all; i0 += AHEAD) {
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int i = i0 + u;
                if (i >= all) break;
                float x[E];
                int j = i * PGN_SAMPLE_THREADS + tid;
                if (i < rounds) {
                    unpack(r[u], x);
                    r[u] = load(j + AHEAD * PGN_SAMPLE_THREADS);
                    if (j < whole_lo || j >= whole_hi) {
#pragma unroll
                        for (int e = 0; e < E; ++e) x[e] = -INFINITY;
                    }
                } else {
                    j = end;
                    pick(j, x);
                }
                f(j, x);
            }
        }
    }
};

// The ids that a filter keeps: those above a logit, and those of that logit up to an index.
struct Kept {
    float x;
    int i;
    __device__ __forceinline__ bool operator()(float y, int j) const { return y > x || (y == x && j <= i); }
    __device__ __forceinline__ void upto(u64 k) {
        x = rank_value((unsigned)(k >> 24));
        i = (int)(k & 0xffffff);
    }
};

struct Weights {
    double max, c;                                           // c: 1024 log2(e) / temperature, not 0
    double least;                                            // min-p as a weight
    float fmax, fc;                                          // fc: bins per unit of distance
    const double* table;
    // w 2^45, nearest whole number.  2^-(t / 1024) with t = k + f, k whole, |f| <= 1/2: a table of 2^-(k % 1024 / 1024),
    // an exponent, and e^-(f ln2 / 1024) as its series up to the third power (the fourth is 2^-50).  Beyond 2^-47 the
    // result is 0 by itself; an infinite maximum leaves only its equals (inf - inf is a NaN, and fmax takes 0 for it).
    __device__ __forceinline__ u64 fixed(float x) const {
        const double t = fmin(::fmax((max - (double)x) * c, 0.0), 1024.0 * (PGN_SAMPLE_BITS + 2));
        const double d = t + 0x1.8p52;
        const int k = (int)(unsigned)(u64)__double_as_longlong(d);
        const double f = t - (d - 0x1.8p52);
        constexpr double c1 = -0.693147180559945309417 / 1024, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
        const double e = fma(fma(fma(c3, f, c2), f, c1), f, 1.0) * table[k & 1023];
        const double up = __hiloint2double((1023 + PGN_SAMPLE_BITS - (k >> 10)) << 20, 0);
        return (u64)__double_as_longlong(fma(e, up, 0x1p52)) & 0xfffffffffffffull;
    }
    // min-p's rule, the same wherever weights are summed or drawn from: the largest logits stay whatever min-p is, above 1 or
    // NaN, and of others only the weight counts.  (A weight of 1 need not be theirs: at a high temperature others round to it.)
    __device__ __forceinline__ bool leaves(u64 v, float x) const { return (double)v >= least || x == fmax; }
    // monotone in x > -inf: 32 bins to a factor of two, everything from 2^-64 on in the last; a NaN (inf - inf, 0 inf) is 0
    __device__ __forceinline__ int bin(float x) const {
        return (int)fminf(fmaxf((fmax - x) * fc, 0.f), (float)(PGN_SAMPLE_BINS - 1));
    }
};

// inclusive prefix sum over the wave, by lane shifts within rows of 16 and two broadcasts across them
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp0(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp0(u64 v) {
    const unsigned lo = (unsigned)dpp0<CTRL, ROWS>((int)(unsigned)v), hi = (unsigned)dpp0<CTRL, ROWS>((int)(unsigned)(v >> 32));
    return ((u64)hi << 32) | lo;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned dpp0(unsigned v) { return (unsigned)dpp0<CTRL, ROWS>((int)v); }
__device__ __forceinline__ unsigned of_lane(unsigned v, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ u64 of_lane(u64 v, int lane) {
    return ((u64)of_lane((unsigned)(v >> 32), lane) << 32) | of_lane((unsigned)v, lane);
}
template <typename T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp0<0x111, 0xf>(v);
    v += dpp0<0x112, 0xf>(v);
    v += dpp0<0x114, 0xf>(v);
    v += dpp0<0x118, 0xf>(v);
    v += dpp0<0x142, 0xa>(v);
    v += dpp0<0x143, 0xc>(v);
    return v;
}

// inclusive prefix sum over the workgroup, and the sum of all
template <typename T>
__device__ __forceinline__ T block_scan(T v, void* scratch, T& total) {
    T* part = reinterpret_cast<T*>(scratch);
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) part[wid] = v;
    __syncthreads();
    static_assert(PGN_SAMPLE_WAVES == 16, "a row of 16 lanes scans the sums of the waves");
    T p = part[threadIdx.x & 15];
    p += dpp0<0x111, 0xf>(p);
    p += dpp0<0x112, 0xf>(p);
    p += dpp0<0x114, 0xf>(p);
    p += dpp0<0x118, 0xf>(p);
    total = of_lane(p, 15);
    return v + (wid > 0 ? of_lane(p, wid - 1) : 0);
}
__device__ __forceinline__ u64 block_sum(u64 v, u64* part) {
    u64 total;
    block_scan(v, part, total);
    return total;
}

// hist[b] += v in one lane for the whole wave where all its lanes add to one place (equal logits), else lane by lane
__device__ __forceinline__ void digit_add(u64* hist, int b, u64 v) {
    const uint64_t lanes = __ballot(v > 0);
    if (lanes == 0) return;
    const int leader = __builtin_ctzll(lanes), b0 = __shfl(b, leader);
    if (__popcll(lanes) > 1 && __all(v == 0 || b == b0)) {
        const u64 s = wave_scan(v);
        if ((threadIdx.x & 63) == 63) atomicAdd(&hist[b0], s);
    } else if (v > 0) {
        atomicAdd(&hist[b], v);
    }
}

// The key up to which the kept ids hold `target` together, ids counted or weights summed, by eight bits
// of the key at a time over the whole row.
template <int DT>
__device__ __forceinline__ u64 select_key(SampleLds& s, const Row<DT>& row, const Weights& w, bool by_weight, u64 target,
                                          const Kept& kept) {
    u64 prefix = 0, before = 0;
    const int tid = threadIdx.x;
    for (int shift = 48; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int b = tid; b < 256; b += PGN_SAMPLE_THREADS) s.hist.digit[b] = 0;
        __syncthreads();
        for (int i0 = 0; i0 < row.V; i0 += PGN_SAMPLE_THREADS) {
            const float x = i0 + tid < row.V ? row.one(i0 + tid) : -INFINITY;
            const u64 key = rank_key(x, i0 + tid);
            const bool on = kept(x, i0 + tid) && (key >> (shift + 8)) == prefix;
            digit_add(s.hist.digit, (int)(key >> shift) & 255, !on ? 0 : by_weight ? w.fixed(x) : 1);
        }
        __syncthreads();
        u64 total;
        const u64 v = tid < 256 ? s.hist.digit[tid] : 0;
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

// Bin in which the running sum over the histogram reaches target(sum of all), and the sum before it; the last bin if none
// does.
template <typename T, typename F>
__device__ __forceinline__ int find_bin(SampleLds& s, const T* hist, F target_of, T& before) {
    constexpr int PER = PGN_SAMPLE_BINS / PGN_SAMPLE_THREADS;
    T v[PER], sum = 0, total;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        v[i] = hist[threadIdx.x * PER + i];
        sum += v[i];
    }
    if (threadIdx.x == 0) s.at = PGN_SAMPLE_BINS - 1;
    T c = block_scan(sum, s.part, total) - sum;
    const T target = target_of(total);
    T* out = reinterpret_cast<T*>(&s.before);
    if (threadIdx.x == 0) *out = total - hist[PGN_SAMPLE_BINS - 1];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (c < target && c + v[i] >= target) {
            s.at = threadIdx.x * PER + i;
            *out = c;
        }
        c += v[i];
    }
    __syncthreads();
    before = *out;
    const int b = s.at;
    __syncthreads();
    return b;
}

// Ascending sort of n keys (n a power of two, the list filled up to it), their weights with them.
__device__ __forceinline__ void sort_list(SampleLds& s, int n) {
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
__device__ __forceinline__ int pad_list(SampleLds& s, int n) {
    int m = 2;
    while (m < n) m <<= 1;
    for (int i = n + threadIdx.x; i < m; i += PGN_SAMPLE_THREADS) {
        s.key[i] = ~0ull;
        s.weight[i] = 0;
    }
    return m;
}

// First place of the list at which the running sum of weights reaches `target`; n - 1 if none.
__device__ __forceinline__ int find_place(SampleLds& s, int n, u64 target, u64& total) {
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

// The rest of a top-k among the n ids of the list, the first k in rank among them: top-p, min-p and the draw.  A few ids
// compare each with each (ranks and running sums without a sort, three rounds); more are sorted by rank, then by index.
__device__ __forceinline__ void finish_list(SampleLds& s, const Weights& w, int n, int k, float p, float u, int64_t* id) {
    const int tid = threadIdx.x;
    u64 z;
    if (n <= PGN_SAMPLE_FEW) {
        u64 key = 0, v = 0;
        if (tid < n) {
            key = s.key[tid];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) rank += s.key[j] < key;
            v = rank < k ? w.fixed(rank_value((unsigned)(key >> 24))) : 0;
            s.weight[tid] = v;
        }
        const u64 all = block_sum(v, s.part);
        if (p < 1.f) {
            const u64 target = nucleus_target(p, all);
            if (tid < n) {
                u64 before = 0;
#pragma unroll 8
                for (int j = 0; j < n; ++j) {
                    const u64 other = s.key[j], weight = s.weight[j];        // both loads at once, not the one for the other
                    before += other < key ? weight : 0;
                }
                v = before < target ? v : 0;
            }
        }
        if (!w.leaves(v, rank_value((unsigned)(key >> 24)))) v = 0;
        __syncthreads();
        if (tid < n) s.weight[tid] = v;
        if (tid == 0) s.found = ~0ull;
        z = block_sum(v, s.part);
        if (tid < n && v > 0) {
            const unsigned i = (unsigned)key & 0xffffff;
            u64 upto = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) {
                const u64 other = s.key[j], weight = s.weight[j];
                upto += ((unsigned)other & 0xffffff) <= i ? weight : 0;
            }
            if (upto >= draw_target(u, z)) atomicMin(&s.found, (u64)i);
        }
        __syncthreads();
        if (tid == 0) *id = (int64_t)s.found;
        return;
    }
    sort_list(s, pad_list(s, n));
    int kept = k < n ? k : n;
    u64 all = 0;
    for (int i = tid; i < kept; i += PGN_SAMPLE_THREADS) all += s.weight[i] = w.fixed(rank_value((unsigned)(s.key[i] >> 24)));
    all = block_sum(all, s.part);
    if (p < 1.f) kept = find_place(s, kept, nucleus_target(p, all), z) + 1;
    const int padded = pad_list(s, kept);
    u64 sum = 0;
    for (int i = tid; i < kept; i += PGN_SAMPLE_THREADS) {
        const u64 v = s.weight[i];
        const bool on = w.leaves(v, rank_value((unsigned)(s.key[i] >> 24)));
        s.weight[i] = on ? v : 0;
        s.key[i] &= 0xffffff;                                // by index now
        sum += on ? v : 0;
    }
    z = block_sum(sum, s.part);
    sort_list(s, padded);
    const int at = find_place(s, kept, draw_target(u, z), z);
    if (tid == 0) *id = (int64_t)s.key[at];
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
    const float u = a.u[b];

    float mine = -INFINITY;                                  // the thread's own maximum
    row.template each<4>([&](int, const float* x) {
#pragma unroll
        for (int e = 0; e < E; ++e) mine = fmaxf(mine, x[e]);
    });
    for (int i = tid; i < PGN_SAMPLE_BINS; i += PGN_SAMPLE_THREADS) s.hist.ids[i] = 0;
    s.table[tid] = exp2((double)tid * (-1.0 / PGN_SAMPLE_TABLE));
    if (tid == 0) s.count = 0;
    float m = mine;
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
        row.template each<1>([&](int j, const float* x) {
#pragma unroll
            for (int e = E - 1; e >= 0; --e) at = x[e] == m ? min(at, row.index(j, e)) : at;
        });
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
    w.c = fmax(PGN_SAMPLE_TABLE * 1.44269504088896340736 / (double)t, 1e-300);        // t may be infinite
    w.fc = (float)(PGN_SAMPLE_BINS_PER_OCTAVE * 1.44269504088896340736 / (double)t);
    w.table = s.table;
    w.least = (double)min_p * (double)(1ull << PGN_SAMPLE_BITS);
    Kept kept = {-INFINITY, -1};                             // everything that can be drawn

    // a logit that no id of a bin up to `bin` is under (1 % of a bin and an ulp cover the rounding of the places)
    const auto lowest = [&](int bin) {
        const float x = (float)(w.max - (bin + 1.01) / (double)w.fc);
        if (bin >= PGN_SAMPLE_BINS - 1 || x != x) return -INFINITY;      // the last bin has no end; inf - inf
        return fabsf(x) < INFINITY ? x - fabsf(x) * 0x1p-23f : x;
    };
    // gathers the ids of the bins from `first` to `last`; how many there are (the list takes PGN_SAMPLE_LIST of them).  lowest()
    // only keeps most of the others from being looked at: it has slack, so it must not be what decides.
    const auto gather = [&](int first, int last) {
        const float low = lowest(last);
        __syncthreads();
        if (tid == 0) s.count = 0;
        __syncthreads();
        row.template each<4>([&](int j, const float* x) {
            unsigned in = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) in |= x[e] >= low ? 1u << e : 0u;
#pragma unroll 1
            for (; __any(in != 0); in &= in - 1) {           // one id a lane at a time
                const int e = in ? __builtin_ctz(in) : 0;
                float xe = x[0];
#pragma unroll
                for (int n = 1; n < E; ++n) xe = e == n ? x[n] : xe;
                const int bin = w.bin(xe);
                if (in && xe > -INFINITY && bin >= first && bin <= last) {
                    const int at = atomicAdd(&s.count, 1);
                    if (at < PGN_SAMPLE_LIST) s.key[at] = rank_key(xe, row.index(j, e));
                }
            }
        });
        __syncthreads();
        return s.count;
    };

    if (k > 0 && k < V) {
        for (bool full = k > PGN_SAMPLE_THREADS;; full = true) {             // a full pass is the last
            unsigned total = 0, before;
            if (!full) {
                if (mine > -INFINITY) atomicAdd(&s.hist.ids[w.bin(mine)], 1u);
            } else {                                         // the last bin may hold most of a row: counted in registers
                unsigned last = 0;
                row.template each<1>([&](int, const float* x) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        const int bin = w.bin(x[e]);
                        const bool is = x[e] > -INFINITY;
                        if (is && bin < PGN_SAMPLE_BINS - 1) atomicAdd(&s.hist.ids[bin], 1u);
                        last += is && bin == PGN_SAMPLE_BINS - 1;
                    }
                });
                block_scan(last, s.part, total);
                if (tid == 0) s.hist.ids[PGN_SAMPLE_BINS - 1] = total;
            }
            __syncthreads();
            const int cut = find_bin(s, s.hist.ids, [&](unsigned z) { total = z; return (unsigned)k; }, before);
            if (full && total <= (unsigned)k) break;         // everything is among the first k
            const unsigned inside = s.hist.ids[cut];
            const bool alone = full && before + inside > PGN_SAMPLE_LIST;        // only the border is looked for in the list
            if (alone && inside > PGN_SAMPLE_LIST) {
                kept.upto(select_key<DT>(s, row, w, false, (u64)k, kept));
                break;
            }
            if (full || cut < PGN_SAMPLE_BINS - 1) {         // else there are fewer maxima than k
                const int n = gather(alone ? cut : 0, cut);
                if (alone) {
                    sort_list(s, pad_list(s, n));
                    kept.upto(s.key[k - (int)before - 1]);
                    break;
                }
                if (full || n <= PGN_SAMPLE_LIST) {          // full: n is before + inside
                    finish_list(s, w, n, k, p, u, a.ids + b);
                    return;
                }
            }
            __syncthreads();
            for (int i = tid; i < PGN_SAMPLE_BINS; i += PGN_SAMPLE_THREADS) s.hist.ids[i] = 0;
            __syncthreads();
        }
        __syncthreads();
    }

    int cut = PGN_SAMPLE_BINS;                               // bins before it are kept whole (as far as `kept` goes)
    u64 target_p = 0, inside_target = 0;
    if (p < 1.f) {
        for (int i = tid; i < PGN_SAMPLE_BINS; i += PGN_SAMPLE_THREADS) s.hist.mass[i] = 0;
        if (tid == 0) s.count = 0;
        __syncthreads();
        const bool filtered = kept.x > -INFINITY;
        row.template each<1>([&](int j, const float* x) {
            u64 v[E];                                        // all of them before the first addition: chains side by side
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = w.fixed(x[e]);
            if (filtered) {
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = kept(x[e], row.index(j, e)) ? v[e] : 0;
            }
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (v[e] > 0) atomicAdd(&s.hist.mass[w.bin(x[e])], v[e]);
        });
        __syncthreads();
        u64 before;
        cut = find_bin(s, s.hist.mass, [&](u64 z) { return target_p = nucleus_target(p, z); }, before);
        inside_target = target_p - before;
    }

    // weights of what is kept, by stretches of 64 vectors; the ids of the bin with the border go to the list
    const int segs = (row.vectors + 63) >> 6;
    bool listed = p < 1.f;
    for (;;) {
        for (int i = tid; i < segs; i += PGN_SAMPLE_THREADS) s.seg[i] = 0;
        __syncthreads();
        // Few ids may be kept, and a weight is dear: every wave collects kept logits until it has 64 to weigh.
        u64* pile = s.pile[wid];
        int held = 0;
        const auto weigh = [&](bool on, u64 entry) {
            const float xe = __uint_as_float((unsigned)entry);
            u64 v = on ? w.fixed(xe) : 0;
            if (!w.leaves(v, xe)) v = 0;
            const int at = on ? ((int)(entry >> 32) + row.lead) / (64 * E) : 0;
            if (__all(at == __builtin_amdgcn_readfirstlane(at))) {           // one stretch: summed here, not by 64 turns in LDS
                v = wave_scan(v);
                if (lane == 63) atomicAdd(&s.seg[at], v);
            } else if (v > 0) {
                atomicAdd(&s.seg[at], v);
            }
        };
        const float low = cut < PGN_SAMPLE_BINS ? lowest(cut) : -INFINITY;
        row.template each<1>([&](int j, const float* x) {
            unsigned in = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) in |= x[e] >= low ? 1u << e : 0u;
#pragma unroll 1
            for (; __any(in != 0); in &= in - 1) {           // one id a lane at a time
                const int e = in ? __builtin_ctz(in) : 0, i = row.index(j, e);
                float xe = x[0];
#pragma unroll
                for (int n = 1; n < E; ++n) xe = e == n ? x[n] : xe;
                const int bin = in && kept(xe, i) ? w.bin(xe) : PGN_SAMPLE_BINS + 1;
                if (bin == cut) {
                    const int at = atomicAdd(&s.count, 1);
                    if (at < PGN_SAMPLE_LIST) s.key[at] = rank_key(xe, i);
                }
                const uint64_t lanes = __ballot(bin < cut);
                if (bin < cut) pile[held + __popcll(lanes & ((1ull << lane) - 1))] = ((u64)(unsigned)i << 32) | __float_as_uint(xe);
                held += __popcll(lanes);
                if (held >= 64) {
                    __builtin_amdgcn_wave_barrier();
                    weigh(true, pile[lane]);
                    held -= 64;
                    const u64 rest = pile[64 + lane];
                    __builtin_amdgcn_wave_barrier();
                    if (lane < held) pile[lane] = rest;
                }
            }
        });
        __builtin_amdgcn_wave_barrier();
        weigh(lane < held, pile[lane]);
        __syncthreads();
        if (!listed) break;
        const int n = s.count;
        if (n <= PGN_SAMPLE_FEW) {                           // compared each with each
            u64 key = 0, v = 0;
            float xe = -INFINITY;
            if (tid < n) s.weight[tid] = v = w.fixed(xe = rank_value((unsigned)((key = s.key[tid]) >> 24)));
            if (tid == 0) s.found = 0;
            __syncthreads();
            if (tid < n) {
                u64 before = 0;
#pragma unroll 8
                for (int j = 0; j < n; ++j) {
                    const u64 other = s.key[j], weight = s.weight[j];
                    before += other < key ? weight : 0;
                }
                if (before < inside_target) {
                    atomicMax(&s.found, key);
                    if (w.leaves(v, xe))
                        atomicAdd(&s.seg[((int)(key & 0xffffff) + row.lead) / (64 * E)], v);
                }
            }
            __syncthreads();
            kept.upto(s.found);                              // under the top-k's border, if there is one
            break;
        }
        if (n <= PGN_SAMPLE_LIST) {
            u64 total;
            for (int i = tid; i < n; i += PGN_SAMPLE_THREADS) s.weight[i] = w.fixed(rank_value((unsigned)(s.key[i] >> 24)));
            sort_list(s, pad_list(s, n));
            const int last = find_place(s, n, inside_target, total);
            kept.upto(s.key[last]);
            for (int i = tid; i <= last; i += PGN_SAMPLE_THREADS) {
                const u64 v = s.weight[i];
                if (w.leaves(v, rank_value((unsigned)(s.key[i] >> 24))))
                    atomicAdd(&s.seg[((int)(s.key[i] & 0xffffff) + row.lead) / (64 * E)], v);
            }
            __syncthreads();
            break;
        }
        kept.upto(select_key<DT>(s, row, w, true, target_p, kept));
        cut = PGN_SAMPLE_BINS;
        listed = false;
        __syncthreads();
    }
    if (wid != 0) return;

    u64 z = 0;
    for (int g = lane; g < segs; g += 64) z += s.seg[g];
    z = __shfl(wave_scan(z), 63);
    const u64 target = draw_target(u, z);
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
    row.pick(j, x);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const u64 f = kept(x[e], row.index(j, e)) ? w.fixed(x[e]) : 0;
        v[e] = w.leaves(f, x[e]) ? f : 0;
        sum += v[e];
    }
    u64 c = before + wave_scan(sum) - sum;
    int hit = -1;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (hit < 0 && c < target && c + v[e] >= target) hit = row.index(j, e);
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
    if (V > PGN_SAMPLE_MAX_IDS || B > PGN_MAX_GRID / PGN_SAMPLE_THREADS) return PGN_ERR_UNSUPPORTED;
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
