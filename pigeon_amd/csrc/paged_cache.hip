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
// flat, one thread a page: a thread finds its request by bisection in the prefix sums, which lie in LDS.
#define PGN_ADV_THREADS 1024
// Up to this many slots the bookkeeping workgroup fills the slot map itself (one launch); above it a second, wide launch
// does.  At 8192 slots the workgroup's 8 rounds cost what the second launch would.
#define PGN_ADV_FUSED_SLOTS 8192

__device__ __forceinline__ int64_t adv_pages(int64_t tokens, int shift) {
    return (tokens + ((int64_t)1 << shift) - 1) >> shift;
}

// inclusive prefix sum over the workgroup; `total` is the sum of all
__device__ int64_t adv_scan(int64_t v, int64_t* wave_sums, int64_t& total) {
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t o = __shfl_up(v, off);
        if (lane >= off) v += o;
    }
    if (lane == 63) wave_sums[wid] = v;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PGN_ADV_THREADS / 64; ++w) {
        const int64_t x = wave_sums[w];
        before += w < wid ? x : 0;
        all += x;
    }
    total = all;
    __syncthreads();
    return v + before;
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

struct AdvRequest {
    int64_t held, keep, add, have, kept;
};

__device__ __forceinline__ AdvRequest adv_request(const int* lens, const int* keep, const int* add, int r, int R, int W,
                                                  int shift) {
    AdvRequest q = {0, 0, 0, 0, 0};
    if (r < R) {
        const int64_t room = (int64_t)W << shift;
        const int64_t h = lens[r];
        q.held = h < 0 ? 0 : (h > room ? room : h);          // a length beyond the table names pages that do not exist
        const int64_t k = keep ? (int64_t)keep[r] : q.held;
        q.keep = k < 0 ? 0 : (k > q.held ? q.held : k);
        const int64_t a = add[r];
        q.add = a < 0 ? 0 : a;
        q.have = adv_pages(q.held, shift);
        q.kept = adv_pages(q.keep, shift);
    }
    return q;
}

__global__ __launch_bounds__(PGN_ADV_THREADS) void pgn_page_advance_kernel(
    int* lens, const int* keep, const int* add, int* __restrict__ table,
    int64_t table_stride, int* __restrict__ free_pages, int* __restrict__ free_count, int N, int R, int W, int shift,
    int T, int fill_slots, int64_t* __restrict__ slots, int* __restrict__ starts, int* __restrict__ status) {
    __shared__ int64_t wave_sums[PGN_ADV_THREADS / 64];
    __shared__ int at[PGN_ADV_THREADS + 1];                  // prefix of what is being moved, within the chunk
    __shared__ int col[PGN_ADV_THREADS];                     // first table column concerned (or the kept length)
    const int tid = threadIdx.x;
    int64_t count = free_count[0];
    count = count < 0 ? 0 : (count > N ? N : count);

    // pages given back in all: the stack is filled so that popping returns them in request order
    int64_t released = 0;
    for (int r0 = 0; r0 < R; r0 += PGN_ADV_THREADS) {
        const AdvRequest q = adv_request(lens, keep, add, r0 + tid, R, W, shift);
        int64_t total;
        adv_scan(q.have - q.kept, wave_sums, total);
        released += total;
    }
    int64_t done = 0;
    if (released > 0) {
        for (int r0 = 0; r0 < R; r0 += PGN_ADV_THREADS) {
            const AdvRequest q = adv_request(lens, keep, add, r0 + tid, R, W, shift);
            int64_t total;
            const int64_t mine = q.have - q.kept;
            at[tid] = (int)(adv_scan(mine, wave_sums, total) - mine);
            col[tid] = (int)q.kept;
            __syncthreads();
            for (int64_t e = tid; e < total; e += PGN_ADV_THREADS) {
                const int i = adv_find(at, PGN_ADV_THREADS, (int)e);
                const int64_t place = count + released - 1 - (done + e);
                if (place < N)                               // more pages back than the pool holds: a caller's mistake
                    free_pages[place] = table[(r0 + i) * table_stride + col[i] + ((int)e - at[i])];
            }
            done += total;
            __syncthreads();
        }
    }
    int64_t top = count + released;
    top = top > N ? N : top;

    int64_t tokens = 0, wanted = 0, popped = 0;
    for (int r0 = 0; r0 < R; r0 += PGN_ADV_THREADS) {
        const int r = r0 + tid;
        const AdvRequest q = adv_request(lens, keep, add, r, R, W, shift);
        int64_t total;
        const int64_t end = tokens + adv_scan(q.add, wave_sums, total);
        const int64_t begin = end - q.add;
        tokens += total;
        const bool fits = r < R && q.keep + q.add <= ((int64_t)W << shift) && end <= T;
        int64_t want = fits ? adv_pages(q.keep + q.add, shift) - q.kept : 0;
        const int64_t taken = wanted + adv_scan(want, wave_sums, total);
        wanted += total;
        const bool ok = fits && (want == 0 || taken <= top);
        want = ok ? want : 0;
        const int64_t first = adv_scan(want, wave_sums, total) - want;
        if (r < R) {
            lens[r] = (int)(ok ? q.keep + q.add : q.keep);
            status[r] = ok ? 0 : 1;
            starts[r + 1] = (int)(end < T ? end : T);
            if (r == 0) starts[0] = 0;
        }
        at[tid] = (int)first;
        col[tid] = (int)q.kept;
        __syncthreads();
        for (int64_t e = tid; e < total; e += PGN_ADV_THREADS) {
            const int i = adv_find(at, PGN_ADV_THREADS, (int)e);
            table[(r0 + i) * table_stride + col[i] + ((int)e - at[i])] = free_pages[top - 1 - popped - e];
        }
        popped += total;
        __syncthreads();
        if (fill_slots) {                                    // T <= PGN_ADV_FUSED_SLOTS here
            const int64_t b = begin < T ? begin : T;
            at[tid] = (int)b;
            if (tid == PGN_ADV_THREADS - 1) at[PGN_ADV_THREADS] = (int)(end < T ? end : T);
            col[tid] = ok ? (int)q.keep : -1;
            __syncthreads();
            for (int64_t t = at[0] + tid; t < at[PGN_ADV_THREADS]; t += PGN_ADV_THREADS) {
                const int i = adv_find(at, PGN_ADV_THREADS, (int)t);
                int64_t slot = -1;
                if (col[i] >= 0) {
                    const int pos = col[i] + ((int)t - at[i]);
                    slot = ((int64_t)table[(r0 + i) * table_stride + (pos >> shift)] << shift) + (pos & ((1 << shift) - 1));
                }
                slots[t] = slot;
            }
            __syncthreads();
        }
    }
    if (fill_slots)
        for (int64_t t = (tokens < T ? tokens : T) + tid; t < T; t += PGN_ADV_THREADS) slots[t] = -1;
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
// page are rescaled if it grew, and the new ones are stored, with no exchange between workgroups.  The tokens are read
// twice (the scale needs their largest magnitude first); the second read hits the caches.
#define PGN_CW_THREADS 256

// 8 consecutive elements of a token's row as fp32
template <int DT>
__device__ __forceinline__ void cw_load8(const unsigned short* p, bool vec, float* f) {
    u16x8_t v;
    if (vec) {
        v = *reinterpret_cast<const u16x8_t*>(p);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p[j];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = Cvt<DT>::to_f32(v[j]);
}

// The least power of two s >= 2^-100 with amax <= 448 s (448 = 1.75 * 2^8 is e4m3's largest value), from the bits.
__device__ __forceinline__ float cw_scale(float amax) {
    const unsigned u = __float_as_uint(amax);
    int k = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    k = k < PGN_CACHE_SCALE_FLOOR ? PGN_CACHE_SCALE_FLOOR : k;
    return __uint_as_float((unsigned)(k + 127) << 23);
}

template <int DT>
__global__ __launch_bounds__(PGN_CW_THREADS) void pgn_cache_write_kernel(
    const unsigned short* __restrict__ k, const unsigned short* __restrict__ v, const int64_t* __restrict__ slots, int T,
    int H, int D, int shift, int64_t N, int chunk, int64_t k_st, int64_t k_sh, int64_t v_st, int64_t v_sh, int k_vec,
    int v_vec, unsigned char* __restrict__ k_pages, unsigned char* __restrict__ v_pages, float* __restrict__ k_scale,
    float* __restrict__ v_scale) {
    extern __shared__ unsigned char tile[];                  // values: [tokens of the run][D + 4] bytes
    __shared__ float wave_max[PGN_CW_THREADS / 64];
    const int tid = threadIdx.x, h = blockIdx.y;
    const bool values = blockIdx.z != 0;
    const int P = 1 << shift;
    const int64_t limit = N << shift;
    const unsigned short* x = (values ? v + h * v_sh : k + h * k_sh);
    const int64_t x_st = values ? v_st : k_st;
    const bool vec = values ? v_vec : k_vec;
    unsigned char* pages = values ? v_pages : k_pages;
    float* scales = values ? v_scale : k_scale;
    const int per_row = D >> 3;

    // which of the chunk's tokens begin a run: one lane a token, the same in every wave (chunk <= 64)
    const int lane = tid & 63, t0 = blockIdx.x * chunk;
    const bool mine = lane < chunk && t0 + lane < T;
    const int64_t my_slot = mine ? slots[t0 + lane] : -1;
    const int64_t my_before = mine && t0 + lane > 0 ? slots[t0 + lane - 1] : -2;
    uint64_t runs = __ballot(my_slot >= 0 && my_slot < limit && ((my_slot & (P - 1)) == 0 || my_before != my_slot - 1));
    for (; runs != 0; runs &= runs - 1) {                    // every bound here is the same for the whole workgroup
        const int first = __builtin_ctzll(runs), t = t0 + first;
        const int64_t slot = __shfl(my_slot, first);
        const int row0 = (int)(slot & (P - 1));
        int count = 0;                                       // tokens of the run: up to the page's end, 64 at a time
        for (int c = 0; c < P - row0; c += 64) {
            const int i = c + lane;
            const uint64_t on = __ballot(i < P - row0 && t + i < T && slots[t + i] == slot + i);
            const int n = ~on == 0 ? 64 : __builtin_ctzll(~on);
            count += n;
            if (n < 64) break;
        }
        const int64_t page = slot >> shift;
        unsigned char* dst = pages + (page * H + h) * (int64_t)P * D;

        float amax = 0.f;
        for (int e = tid; e < count * per_row; e += PGN_CW_THREADS) {
            const int i = e / per_row, c = (e - i * per_row) * 8;
            float f[8];
            cw_load8<DT>(x + (int64_t)(t + i) * x_st + c, vec, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float a = fabsf(f[j]);
                amax = a < INFINITY ? fmaxf(amax, a) : amax;  // infinities and NaN do not count
            }
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
        if ((tid & 63) == 0) wave_max[tid >> 6] = amax;
        const float old = row0 > 0 ? scales[page * H + h] : 0.f;
        __syncthreads();
        amax = fmaxf(fmaxf(wave_max[0], wave_max[1]), fmaxf(wave_max[2], wave_max[3]));
        const float s = fmaxf(cw_scale(amax), old);          // a stored NaN loses against the new scale
        const float inv = 1.0f / s;                          // exact: s is a power of two

        if (row0 > 0 && old < s) {                           // older tokens of the page, under the larger scale
            const float f = old * inv;
            if (!values) {
                for (int e = tid; e < row0 * per_row; e += PGN_CW_THREADS) {
                    uint2 w = *reinterpret_cast<const uint2*>(dst + e * 8);
                    w.x = pgn_fp8_rescale4(w.x, f);
                    w.y = pgn_fp8_rescale4(w.y, f);
                    *reinterpret_cast<uint2*>(dst + e * 8) = w;
                }
            } else {
                const int words = (row0 + 3) >> 2;           // the last word may hold tokens behind row0: bytes there
                for (int e = tid; e < D * words; e += PGN_CW_THREADS) {
                    const int d = e / words, w = e - d * words;
                    unsigned char* p = dst + (int64_t)d * P + w * 4;
                    const unsigned was = *reinterpret_cast<const unsigned*>(p), is = pgn_fp8_rescale4(was, f);
                    if (w * 4 + 4 <= row0) {
                        *reinterpret_cast<unsigned*>(p) = is;
                    } else {
                        for (int j = 0; w * 4 + j < row0; ++j) p[j] = (unsigned char)(is >> (8 * j));
                    }
                }
            }
        }

        for (int e = tid; e < count * per_row; e += PGN_CW_THREADS) {
            const int i = e / per_row, c = (e - i * per_row) * 8;
            float f[8];
            cw_load8<DT>(x + (int64_t)(t + i) * x_st + c, vec, f);
            uint2 w;
            w.x = pgn_fp8_pack4(f[0] * inv, f[1] * inv, f[2] * inv, f[3] * inv);
            w.y = pgn_fp8_pack4(f[4] * inv, f[5] * inv, f[6] * inv, f[7] * inv);
            if (!values) {
                *reinterpret_cast<uint2*>(dst + (int64_t)(row0 + i) * D + c) = w;
            } else {
                *reinterpret_cast<unsigned*>(tile + i * (D + 4) + c) = w.x;
                *reinterpret_cast<unsigned*>(tile + i * (D + 4) + c + 4) = w.y;
            }
        }
        __syncthreads();                                     // the tile is whole; every thread has read the old scale
        if (values) {
            const int w0 = row0 >> 2, words = ((row0 + count + 3) >> 2) - w0;
            for (int e = tid; e < D * words; e += PGN_CW_THREADS) {
                const int w = e / D, d = e - w * D;
                const int r = (w0 + w) * 4;                  // tokens r .. r + 3 of the page, one word
                unsigned char* p = dst + (int64_t)d * P + r;
                if (r >= row0 && r + 4 <= row0 + count) {
                    unsigned word = 0;
#pragma unroll
                    for (int j = 0; j < 4; ++j) word |= (unsigned)tile[(r - row0 + j) * (D + 4) + d] << (8 * j);
                    *reinterpret_cast<unsigned*>(p) = word;
                } else {
                    for (int j = 0; j < 4; ++j)
                        if (r + j >= row0 && r + j < row0 + count) p[j] = tile[(r - row0 + j) * (D + 4) + d];
                }
            }
        }
        if (tid == 0) scales[page * H + h] = s;
        __syncthreads();                                     // the tile and wave_max are used again
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
    hipLaunchKernelGGL(pgn_page_advance_kernel, dim3(1), dim3(PGN_ADV_THREADS), 0, s, lens, keep, add, table,
                       table_stride, free_pages, free_count, num_pages, R, W, shift, T, fused, slots, starts, status);
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
    const int k_vec = pgn_aligned(k, 16) && k_st % 8 == 0 && k_sh % 8 == 0;
    const int v_vec = pgn_aligned(v, 16) && v_st % 8 == 0 && v_sh % 8 == 0;
    const int T = (int)num_tokens, D = head_dim;
    // One token a workgroup while the launch is small (a decoding step: every token is a run of its own and latency
    // counts), 16 above: most tokens then lie inside a run and only cost a look at the slot map.
    const int chunk = T <= 2048 ? 1 : 16;
    const dim3 grid((T + chunk - 1) / chunk, kv_heads, 2), block(PGN_CW_THREADS);
    const size_t lds = (size_t)page_size * (D + 4);          // <= 128 * 260 bytes
    hipStream_t s = (hipStream_t)stream;
#define PGN_CW_LAUNCH(DT)                                                                                              \
    hipLaunchKernelGGL((pgn_cache_write_kernel<DT>), grid, block, lds, s, (const unsigned short*)k,                    \
                       (const unsigned short*)v, slots, T, kv_heads, D, shift, (int64_t)num_pages, chunk, k_st, k_sh,  \
                       v_st, v_sh, k_vec, v_vec, (unsigned char*)k_pages, (unsigned char*)v_pages, k_scale, v_scale)
    if (dtype == PGN_BF16) PGN_CW_LAUNCH(PGN_BF16);
    else PGN_CW_LAUNCH(PGN_F16);
#undef PGN_CW_LAUNCH
    PGN_LAUNCH_CHECK();
    return PGN_OK;
}
