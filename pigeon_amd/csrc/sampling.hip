// Drawing token ids from logits (see include/pigeon_hip.h: pgn_sample_tokens).
//
// The weights w_i = exp((x_i - max) / temperature) are computed in 64 bits and rounded to whole multiples of 2^-bits
// (bits = 45 for up to 2^18 ids): sums of them are then integers, which are the same in any order, so atomics and any
// split of the row give the same ids every time.  The rounding is at most 2^-46 of the largest weight per id.
//
// One order ranks the ids: larger logit first, lower index first among equal ones.  As a 64-bit key - the logit's bits
// made monotone and complemented, then the index - "rank before" is "smaller key", and every filter keeps the ids up to
// some key: top-k the one where k ids, top-p the one where the wanted weight is reached.
#include "pgn_common.h"

#define PGN_SAMPLE_THREADS 1024
#define PGN_SAMPLE_WAVES (PGN_SAMPLE_THREADS / 64)

namespace {

struct SampleArgs {
    const void* logits;
    const float* u;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    int64_t* ids;
    int64_t stride;
    int V, bits;
    float temperature_all, top_p_all, min_p_all;
    int top_k_all;
};

// rank key of a logit: ascending keys are descending values
__device__ __forceinline__ unsigned rank_bits(float x) {
    const unsigned u = __float_as_uint(x);
    return (u & 0x80000000u) ? u : ~(u | 0x80000000u);
}

// NaN counts as a logit of -inf; -0 as 0, so that the two tie as they compare
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }

template <int DT>
__device__ __forceinline__ float logit(const void* row, int i) {
    return clean(Cvt<DT>::to_f32(reinterpret_cast<const typename Cvt<DT>::storage*>(row)[i]));
}

struct Weights {
    double max, inv_t, one;
    bool infinite;                                           // the maximum is +inf: only its equals weigh anything
    __device__ __forceinline__ double real(float x) const {
        if (infinite) return x == INFINITY ? 1.0 : 0.0;
        return x == -INFINITY ? 0.0 : exp(((double)x - max) * inv_t);
    }
    __device__ __forceinline__ unsigned long long fixed(double w) const {
        // w <= 1 times 2^bits, rounded by an addition that leaves it in the low mantissa bits
        const double y = fma(w, one, 0x1p52);
        return (unsigned long long)__double_as_longlong(y) & 0xfffffffffffffull;
    }
};

__device__ unsigned long long block_sum(unsigned long long v, unsigned long long* part) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long s = 0;
#pragma unroll
    for (int w = 0; w < PGN_SAMPLE_WAVES; ++w) s += part[w];
    return s;
}

// The smallest key up to which the ids hold `target` together: ids counted, or weights summed.  Eight bits of the key at
// a time, 32 of the logit and 24 of the index, by a histogram of the ids that agree with the bits found so far.
// Needs target <= the total.  `limit`: only ids with keys up to it take part.
template <int DT>
__device__ unsigned long long select_key(const void* row, int V, const Weights& w, bool by_weight,
                                         unsigned long long target, unsigned long long limit, unsigned long long* hist) {
    __shared__ unsigned long long found_prefix, found_before;
    unsigned long long prefix = 0, before = 0;
    const int tid = threadIdx.x;
    for (int shift = 48; shift >= 0; shift -= 8) {
        for (int b = tid; b < 256; b += PGN_SAMPLE_THREADS) hist[b] = 0;
        __syncthreads();
        for (int i = tid; i < V; i += PGN_SAMPLE_THREADS) {
            const float x = logit<DT>(row, i);
            const unsigned long long key = ((unsigned long long)rank_bits(x) << 24) | (unsigned)i;
            if (key <= limit && x > -INFINITY && (key >> (shift + 8)) == prefix) {
                const unsigned long long v = by_weight ? w.fixed(w.real(x)) : 1ull;
                if (v) atomicAdd(&hist[(key >> shift) & 255], v);
            }
        }
        __syncthreads();
        if (tid == 0) {
            unsigned long long sum = before;
            int b = 0;
            for (; b < 255 && sum + hist[b] < target; ++b) sum += hist[b];
            found_prefix = (prefix << 8) | (unsigned)b;
            found_before = sum;
        }
        __syncthreads();
        prefix = found_prefix;
        before = found_before;
        __syncthreads();
    }
    return prefix;
}

template <int DT>
__global__ __launch_bounds__(PGN_SAMPLE_THREADS) void pgn_sample_tokens_kernel(const SampleArgs a) {
    __shared__ unsigned long long hist[256];
    __shared__ unsigned long long part[PGN_SAMPLE_WAVES];
    __shared__ float fpart[PGN_SAMPLE_WAVES];
    extern __shared__ unsigned long long seg[];              // weight of each 64 consecutive ids
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, b = blockIdx.x, V = a.V;
    const void* row = reinterpret_cast<const char*>(a.logits) + (int64_t)b * a.stride * sizeof(typename Cvt<DT>::storage);
    const float t = a.temperature ? a.temperature[b] : a.temperature_all;
    const int k = a.top_k ? a.top_k[b] : a.top_k_all;
    const float p = a.top_p ? a.top_p[b] : a.top_p_all;
    const float min_p = a.min_p ? a.min_p[b] : a.min_p_all;

    float m = -INFINITY;
    for (int i = tid; i < V; i += PGN_SAMPLE_THREADS) m = fmaxf(m, logit<DT>(row, i));
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    if (lane == 0) fpart[wid] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < PGN_SAMPLE_WAVES; ++w) m = fmaxf(m, fpart[w]);
    if (m == -INFINITY) {                                    // nothing may be drawn
        if (tid == 0) a.ids[b] = -1;
        return;
    }

    Weights w;
    w.max = m;
    w.infinite = m == INFINITY;
    w.inv_t = 1.0 / (double)t;
    w.one = ldexp(1.0, a.bits);
    unsigned long long limit = ~0ull;
    if (!(t > 0.f) || p <= 0.f || k == 1) {                  // the first in rank: the largest logit, the lowest index
        limit = select_key<DT>(row, V, w, false, 1, limit, hist);
        if (tid == 0) a.ids[b] = (int64_t)(limit & 0xffffff);
        return;
    }
    if (k > 0 && k < V) {
        unsigned long long n = 0;
        for (int i = tid; i < V; i += PGN_SAMPLE_THREADS) n += logit<DT>(row, i) > -INFINITY;
        if ((unsigned long long)k < block_sum(n, part)) limit = select_key<DT>(row, V, w, false, k, limit, hist);
    }
    if (p < 1.f) {
        unsigned long long z = 0;
        for (int i = tid; i < V; i += PGN_SAMPLE_THREADS) {
            const float x = logit<DT>(row, i);
            if ((((unsigned long long)rank_bits(x) << 24) | (unsigned)i) <= limit) z += w.fixed(w.real(x));
        }
        z = block_sum(z, part);
        const double want = ceil((double)p * (double)z);
        const unsigned long long target = want < 1.0 ? 1ull : (unsigned long long)want;
        limit = select_key<DT>(row, V, w, true, target < z ? target : z, limit, hist);
    }

    // weights of what is kept, in index order
    const int segs = (V + 63) >> 6;
    for (int s = wid; s < segs; s += PGN_SAMPLE_WAVES) {
        const int i = s * 64 + lane;
        unsigned long long v = 0;
        if (i < V) {
            const float x = logit<DT>(row, i);
            if ((((unsigned long long)rank_bits(x) << 24) | (unsigned)i) <= limit) {
                const double r = w.real(x);
                v = r >= (double)min_p || x == m ? w.fixed(r) : 0;
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
        if (lane == 0) seg[s] = v;
    }
    __syncthreads();
    if (wid != 0) return;
    unsigned long long z = 0;
    for (int s = lane; s < segs; s += 64) z += seg[s];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) z += __shfl_xor(z, off);
    double u = a.u[b];
    u = u >= 0.0 ? u : 0.0;                                  // a NaN too
    const double cut = floor(u * (double)z);
    unsigned long long target = cut >= (double)z ? z - 1 : (unsigned long long)cut;    // the first id with a sum above it
    if (target >= z) target = z - 1;
    int s0 = 0;
    unsigned long long before = 0;
    for (; s0 < segs; s0 += 64) {
        unsigned long long v = s0 + lane < segs ? seg[s0 + lane] : 0, c = v;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const unsigned long long o = __shfl_up(c, off);
            if (lane >= off) c += o;
        }
        const uint64_t over = __ballot(before + c > target);
        if (over) {
            const int at = __builtin_ctzll(over);
            before += __shfl(c, at) - __shfl(v, at);
            s0 += at;
            break;
        }
        before += __shfl(c, 63);
    }
    const int i = s0 * 64 + lane;
    unsigned long long c = 0;
    if (i < V) {
        const float x = logit<DT>(row, i);
        if ((((unsigned long long)rank_bits(x) << 24) | (unsigned)i) <= limit) {
            const double r = w.real(x);
            c = r >= (double)min_p || x == m ? w.fixed(r) : 0;
        }
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const unsigned long long o = __shfl_up(c, off);
        if (lane >= off) c += o;
    }
    const uint64_t over = __ballot(before + c > target);
    if (lane == 0) a.ids[b] = over ? (int64_t)s0 * 64 + __builtin_ctzll(over) : -1;
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
    a.bits = 45;                                             // V * 2^45 stays under 2^63
    a.temperature_all = temperature_all;
    a.top_k_all = top_k_all;
    a.top_p_all = top_p_all;
    a.min_p_all = min_p_all;
    hipStream_t s = (hipStream_t)stream;
    const size_t lds = (size_t)((V + 63) / 64) * 8;
    const dim3 grid(B), block(PGN_SAMPLE_THREADS);
    if (dtype == PGN_F32) hipLaunchKernelGGL((pgn_sample_tokens_kernel<PGN_F32>), grid, block, lds, s, a);
    else if (dtype == PGN_BF16) hipLaunchKernelGGL((pgn_sample_tokens_kernel<PGN_BF16>), grid, block, lds, s, a);
    else hipLaunchKernelGGL((pgn_sample_tokens_kernel<PGN_F16>), grid, block, lds, s, a);
    PGN_LAUNCH_CHECK();
    return PGN_OK;
}
