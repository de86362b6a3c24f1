// Routing of agents to modalities on gfx950: the k most probable modalities of each agent, the (agent, modality) pairs sorted
// by modality, the agents' rows copied to their pairs and the pairs' answers summed back with their weights; and the gradients.
//
// Everything here moves data: each kernel reads its inputs and writes its outputs once (the sort reads the ids twice).
// No result depends on the order in which workgroups run: sums go over a token's own pairs in their order, and the sort is
// stable.  Types float, bfloat16, half; softmax statistics, weights and sums are float.
#include <type_traits>

#include "mtp_internal.h"

namespace {

constexpr int ROUTE_MAX_E = 4096;  // index bits of a sort key; registers of a lane
constexpr int ROUTE_MAX_K = 128;

template <typename T>
__device__ __forceinline__ float up(T v) {
    return (float)v;
}

// ---- top k ----
// A key orders like (score, -index), so that a maximum finds value and index at once and equal scores go to the lower index.
// 16-bit scores: the bits made monotonous in the upper half of 32, 65535 - index in the lower.  float: 32 + 12 bits in the mantissa
// of a double with a fixed exponent, which v_max_f64 / v_min_f64 compare.  NONE is below every key, that of -inf included.
template <typename T>
struct RouteKey {
    typedef uint32_t type;
    static constexpr type NONE = 0;
    static constexpr uint32_t INF = std::is_same<T, _Float16>::value ? 0x7c00u : 0x7f80u;
    // nothing: NONE, or an index without a score (a place beyond the row; -inf's bits are 0x7f or 0x3ff)
    static __device__ __forceinline__ bool nothing(type k) { return k < 0x10000u; }
    // the keys of v[0 .. V), pieces of W with the indexes from[q] on, of which those in [first[q], end[q]) count.  Two scores at a
    // time; NaN (to become -inf) and -0 (to equal +0) are looked for at the end and put right only where a wave has one.
    template <int V, int W>
    static __device__ __forceinline__ void keys(const T (&v)[V], const int (&from)[V / W], const int (&first)[V / W],
                                                const int (&end)[V / W], type (&key)[V], bool *bad) {
        typedef short s2 __attribute__((ext_vector_type(2)));
        typedef unsigned short u2 __attribute__((ext_vector_type(2)));
        u2 o[(V + 1) / 2], odd = {0xffff, 0xffff}, big = {0, 0};
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            u2 x = {__builtin_bit_cast(unsigned short, v[j]), __builtin_bit_cast(unsigned short, v[j + 1 < V ? j + 1 : j])};
            const u2 neg = (u2)((s2)x >> 15);
            o[j / 2] = x ^ (neg | (u2){0x8000, 0x8000});
            odd = __builtin_elementwise_min(odd, (u2)(o[j / 2] - (u2){0x7fff, 0x7fff}));  // -0: 0
            big = __builtin_elementwise_max(big, (u2)(x & (u2){0x7fff, 0x7fff}));          // NaN: above INF
        }
        const bool special = odd[0] == 0 || odd[1] == 0 || big[0] > INF || big[1] > INF;
        if (__ballot(special) != 0) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                uint32_t b = __builtin_bit_cast(uint16_t, v[j]);
                const bool nan = (b & 0x7fffu) > INF;
                const int i = from[j / W] + j % W;
                *bad |= nan && i >= first[j / W] && i < end[j / W];
                b = nan ? 0x8000u | INF : b == 0x8000u ? 0u : b;
                o[j / 2][j & 1] = (unsigned short)((b & 0x8000u) ? (b ^ 0xffffu) : (b | 0x8000u));
            }
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = from[j / W] + j % W;
            const uint32_t w = __builtin_bit_cast(uint32_t, o[j / 2]);
            const uint32_t k = ((j & 1) ? (w & 0xffff0000u) : (w << 16)) | (0xffffu - i);
            key[j] = i >= first[j / W] && i < end[j / W] ? k : NONE;
        }
    }
    static __device__ __forceinline__ float score(type k) {
        uint32_t b = k >> 16;
        b = (b & 0x8000u) ? (b ^ 0x8000u) : (b ^ 0xffffu);
        return (float)__builtin_bit_cast(T, (uint16_t)b);
    }
    static __device__ __forceinline__ int index(type k) { return 0xffff - (int)(k & 0xffffu); }
    static __device__ __forceinline__ type more(type a, type b) { return a > b ? a : b; }
    static __device__ __forceinline__ type less(type a, type b) { return a > b ? b : a; }
    template <int CTRL>
    static __device__ __forceinline__ type turn(type v) {
        return (type)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true);
    }
    // the larger of a lane's and that of the lane 16 (32) away: the swap puts the two halves side by side
    static __device__ __forceinline__ type across16(type v) {
        const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return more(s[0], s[1]);
    }
    static __device__ __forceinline__ type across32(type v) {
        const auto s = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return more(s[0], s[1]);
    }
};
template <>
struct RouteKey<float> {
    typedef double type;
    static constexpr type NONE = 2.0;
    static __device__ __forceinline__ bool nothing(type k) { return k == NONE; }
    template <int V, int W>
    static __device__ __forceinline__ void keys(const float (&v)[V], const int (&from)[V / W], const int (&first)[V / W],
                                                const int (&end)[V / W], type (&key)[V], bool *bad) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int i = from[j / W] + j % W;
            const bool counts = i >= first[j / W] && i < end[j / W];
            const bool nan = v[j] != v[j];
            *bad |= nan && counts;
            uint32_t b = __float_as_uint((nan ? -__builtin_inff() : v[j]) + 0.0f);  // -0 equals +0
            b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
            const type k = __longlong_as_double(
                (long long)(0x4000000000000000ull | ((uint64_t)b << 12) | (uint32_t)(ROUTE_MAX_E - 1 - i)));
            key[j] = counts ? k : NONE;
        }
    }
    static __device__ __forceinline__ float score(type k) {
        const uint32_t b = (uint32_t)((uint64_t)__double_as_longlong(k) >> 12);
        return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
    }
    static __device__ __forceinline__ int index(type k) {
        return ROUTE_MAX_E - 1 - (int)((uint64_t)__double_as_longlong(k) & (ROUTE_MAX_E - 1));
    }
    static __device__ __forceinline__ type more(type a, type b) { return fmax(a, b); }
    static __device__ __forceinline__ type less(type a, type b) { return fmin(a, b); }
    template <int CTRL>
    static __device__ __forceinline__ type turn(type v) {
        const uint64_t b = (uint64_t)__double_as_longlong(v);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)b, CTRL, 0xf, 0xf, true);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, true);
        return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
    }
    static __device__ __forceinline__ type from_words(uint32_t lo, uint32_t hi) {
        return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
    }
    static __device__ __forceinline__ type across16(type v) {
        const uint64_t b = (uint64_t)__double_as_longlong(v);
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
        return more(from_words(lo[0], hi[0]), from_words(lo[1], hi[1]));
    }
    static __device__ __forceinline__ type across32(type v) {
        const uint64_t b = (uint64_t)__double_as_longlong(v);
        const auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
        const auto hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
        return more(from_words(lo[0], hi[0]), from_words(lo[1], hi[1]));
    }
};

constexpr int ROW_ROR = 0x120;  // rotation within 16 lanes
constexpr int HALF_MIRROR = 0x141, QUAD_XOR1 = 0xb1, QUAD_XOR2 = 0x4e;  // lane 7 - i of eight; the neighbour, the next but one of four

// over the L lanes (8, 16, 32 or 64) that share a row, the same result in each
template <typename T, int L>
__device__ __forceinline__ typename RouteKey<T>::type group_max(typename RouteKey<T>::type v) {
    typedef RouteKey<T> R;
    if constexpr (L == 8) {
        v = R::more(v, R::template turn<HALF_MIRROR>(v));
        v = R::more(v, R::template turn<QUAD_XOR1>(v));
        return R::more(v, R::template turn<QUAD_XOR2>(v));
    }
    v = R::more(v, R::template turn<ROW_ROR + 8>(v));
    v = R::more(v, R::template turn<ROW_ROR + 4>(v));
    v = R::more(v, R::template turn<ROW_ROR + 2>(v));
    v = R::more(v, R::template turn<ROW_ROR + 1>(v));
    if constexpr (L >= 32) v = R::across16(v);
    if constexpr (L == 64) v = R::across32(v);
    return v;
}
template <int CTRL>
__device__ __forceinline__ float turn_f32(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int L>
__device__ __forceinline__ float group_sum(float v) {
    if constexpr (L == 8) {
        v += turn_f32<HALF_MIRROR>(v);
        v += turn_f32<QUAD_XOR1>(v);
        return v + turn_f32<QUAD_XOR2>(v);
    }
    v += turn_f32<ROW_ROR + 8>(v);
    v += turn_f32<ROW_ROR + 4>(v);
    v += turn_f32<ROW_ROR + 2>(v);
    v += turn_f32<ROW_ROR + 1>(v);
    if constexpr (L >= 32) v += __shfl_xor(v, 16);
    if constexpr (L == 64) v += __shfl_xor(v, 32);
    return v;
}

// Batcher's odd-even merge sort of V registers, largest first
template <typename T, int V>
__device__ __forceinline__ void sort_registers(typename RouteKey<T>::type (&a)[V]) {
#pragma unroll
    for (int p = 1; p < V; p *= 2) {
#pragma unroll
        for (int q = p; q >= 1; q /= 2) {
#pragma unroll
            for (int j = q % p; j + q < V; j += 2 * q) {
#pragma unroll
                for (int i = 0; i < q; ++i) {
                    if (i + j + q < V && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
                        const typename RouteKey<T>::type x = a[i + j], y = a[i + j + q];
                        a[i + j] = RouteKey<T>::more(x, y);
                        a[i + j + q] = RouteKey<T>::less(x, y);
                    }
                }
            }
        }
    }
}

// p = exp(s - max) / sum exp(s - max) over all scores or the chosen ones, and the k largest.  L lanes share a row, lane `sub` holds
// the scores sub * V to sub * V + V - 1.  Each lane sorts its keys and lays them into LDS, as many as could be chosen; k times the
// largest head is taken (a maximum over the L lanes), and the lane it came from moves on to its next key.  Scores are read once.
// Bound by its vector instructions: for 16 keys a lane 63 pairs of the sort, then some twelve for each of the k.  1 M rows of
// 200 bfloat16, top 20: 230 us for 0.57 GB (2.5 TB/s, half the rate of a copy); 17 970 rows of 400, top 8: 13 us.
template <typename T, int L, int V, int KB>
__global__ __launch_bounds__(256) void k_route_topk(const T *__restrict__ scores, int64_t n, int e, int64_t ld, int k, int normalize,
                                                    int32_t *__restrict__ ids, float *__restrict__ weights,
                                                    float *__restrict__ stats) {
    typedef RouteKey<T> R;
    typedef typename R::type key_t;
    extern __shared__ __attribute__((aligned(16))) char route_lds[];  // key_t [min(V, k) + 1][256]
    key_t *lists = reinterpret_cast<key_t *>(route_lds);
    constexpr int W = V * (int)sizeof(T) < 16 ? V : 16 / (int)sizeof(T);  // elements of a piece
    const int tid = threadIdx.x, sub = tid % L;
    const int64_t row = (int64_t)blockIdx.x * (256 / L) + tid / L;
    const bool live = row < n;
    const T *s = scores + (live ? row : n - 1) * ld;

    // pieces of W elements at any address; the one that would reach beyond the row moves back, and what it says again is left out
    T v[V];
    int from[V / W];
#pragma unroll
    for (int q = 0; q < V / W; ++q) {
        const int i = sub * V + q * W;
        from[q] = i + W <= e ? i : e - W;
        if (i >= e) from[q] = 0;
        typedef T piece_t __attribute__((ext_vector_type(W), aligned(sizeof(T))));
        if (e >= W) {
            const piece_t p = *reinterpret_cast<const piece_t *>(s + from[q]);
#pragma unroll
            for (int j = 0; j < W; ++j) v[q * W + j] = p[j];
        } else {  // a row shorter than one piece
            from[q] = 0;
#pragma unroll
            for (int j = 0; j < W; ++j) v[q * W + j] = s[j < e ? j : 0];
        }
    }
    key_t key[V];
    bool bad = false;
    // element j of the lane is score from[j / W] + j % W, and counts where no other piece has it
    int first[V / W], end[V / W];
#pragma unroll
    for (int q = 0; q < V / W; ++q) {
        first[q] = sub * V + q * W;
        end[q] = first[q] + W < e ? first[q] + W : e;
    }
    R::template keys<V, W>(v, from, first, end, key, &bad);
    float total = 0.f, top = 0.f;
    if (!normalize) {  // the softmax over all modalities
        key_t m = key[0];
#pragma unroll
        for (int j = 1; j < V; ++j) m = R::more(m, key[j]);
        top = R::score(group_max<T, L>(m));
        if (top == -__builtin_inff()) top = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) total += !R::nothing(key[j]) ? expf(R::score(key[j]) - top) : 0.f;
        total = group_sum<L>(total);
    }
    const uint64_t any_bad = __ballot(bad);
    const bool row_bad = ((any_bad >> ((tid & 63) / L * L)) & (L == 64 ? ~0ull : (1ull << (L & 63)) - 1)) != 0;

    sort_registers<T, V>(key);
    const int depth = V < k ? V : k;
    key_t *next = lists + tid;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (j < depth) next[j * 256] = key[j];
    next[depth * 256] = R::NONE;
    key_t head = key[0];
    key_t chosen[KB];
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        chosen[b] = R::NONE;
        const int most = k - b * L < L ? k - b * L : L;
        auto take = [&](int i) {
            const key_t best = group_max<T, L>(head);
            if (sub == i) chosen[b] = best;
            // keys differ by their index, so one lane moves on; there are k keys at least, so the largest is never NONE
            next += head == best ? 256 : 0;
            head = *next;
        };
        int i = 0;
        for (; i + 4 <= most; i += 4) {
            take(i);
            take(i + 1);
            take(i + 2);
            take(i + 3);
        }
        for (; i < most; ++i) take(i);
    }
    float w[KB];
    if (normalize) {
        // lane 0 of the first batch has the largest score
        const key_t first = __shfl(chosen[0], (tid & 63) / L * L);
        top = R::nothing(first) ? 0.f : R::score(first);
        if (top == -__builtin_inff()) top = 0.f;
    }
    float sum = 0.f;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        const float x = R::score(chosen[b]);
        const bool none = R::nothing(chosen[b]) || x == -__builtin_inff();
        if (none) chosen[b] = R::NONE;
        w[b] = none ? 0.f : expf(x - top);
        sum += w[b];
    }
    if (normalize) total = group_sum<L>(sum);
    const float scale = total != 0.f ? 1.f / total : (total != total ? total : 0.f);
    if (!live) return;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
        const int i = b * L + sub;
        if (i < k) {
            const bool none = chosen[b] == R::NONE;
            ids[row * k + i] = none ? -1 : R::index(chosen[b]);
            weights[row * k + i] = row_bad ? __builtin_nanf("") : w[b] * scale;
        }
    }
    if (stats != nullptr && sub == 0) {
        stats[row * 2] = top;
        stats[row * 2 + 1] = row_bad ? __builtin_nanf("") : scale;
    }
}

// Gradient towards the scores, a few rows per workgroup, put together in LDS and written in whole 16-byte pieces:
//   w_j (g_j - sum g w) at the chosen;  elsewhere zero (normalised) or -p_j sum g w, p the softmax over all
// Bound by memory; normalised, the scores are not read.  1 M rows of 200 bfloat16, top 20: 167 us for 640 MB, 3.8 TB/s; over all 238.
template <typename T>
__global__ __launch_bounds__(256) void k_route_grad(const T *__restrict__ scores, int64_t n, int e, int64_t ld, int k, int normalize,
                                                    const int32_t *__restrict__ ids, const float *__restrict__ weights,
                                                    const float *__restrict__ stats, const float *__restrict__ g,
                                                    T *__restrict__ out, int rows_per, int pieces) {
    extern __shared__ __attribute__((aligned(16))) char grad_lds[];  // float dots[rows_per], then T tile[rows_per][e]
    float *dots = reinterpret_cast<float *>(grad_lds);
    char *tile_at = grad_lds + (rows_per * 4 + 15) / 16 * 16;
    T *tile = reinterpret_cast<T *>(tile_at);
    const int tid = threadIdx.x, sub = tid & 15;
    const int64_t row0 = (int64_t)blockIdx.x * rows_per;
    const int rows = (int)(n - row0 < rows_per ? n - row0 : rows_per);
    for (int r = tid >> 4; r < rows; r += 16) {
        const int64_t at = (row0 + r) * k;
        float dot = 0.f;
        for (int j = sub; j < k; j += 16) {
            const float w = weights[at + j];
            float x = g[at + j];
            asm volatile("" : "+v"(x));     // loaded with w, not behind it (173 us, 208)
            dot += w != 0.f ? w * x : 0.f;  // where there is no choice (weight 0) g may be anything
        }
        dot = group_sum<16>(dot);
        if (sub == 0) dots[r] = dot;
    }
    const int held = rows * e, whole = (held * (int)sizeof(T) + 15) / 16;
    if (normalize) {
        for (int i = tid; i < whole; i += 256) reinterpret_cast<float4 *>(tile_at)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        __syncthreads();
    } else {
        __syncthreads();
        constexpr int N = 16 / (int)sizeof(T);
        if (e % N == 0) {
            typedef T loose __attribute__((ext_vector_type(N), aligned(sizeof(T))));
            typedef T whole_t __attribute__((ext_vector_type(N)));
            const uint32_t per = e / N;
            for (uint32_t i = tid; i < (uint32_t)rows * per; i += 256) {
                const uint32_t r = i / per;
                const float top = stats[(row0 + r) * 2], scale = stats[(row0 + r) * 2 + 1] * -dots[r];
                const loose v = *reinterpret_cast<const loose *>(scores + (row0 + r) * ld + (i - r * per) * N);
                whole_t w;
#pragma unroll
                for (int j = 0; j < N; ++j) w[j] = (T)(expf(up(v[j]) - top) * scale);
                reinterpret_cast<whole_t *>(tile)[i] = w;
            }
        } else for (int r = tid >> 6; r < rows; r += 4) {
            const float top = stats[(row0 + r) * 2], scale = stats[(row0 + r) * 2 + 1] * -dots[r];
            const T *s = scores + (row0 + r) * ld;
            for (int c = tid & 63; c < e; c += 64) tile[r * e + c] = (T)(expf(up(s[c]) - top) * scale);
        }
        __syncthreads();
    }
    for (int r = tid >> 4; r < rows; r += 16) {
        const int64_t at = (row0 + r) * k;
        const float dot = dots[r];
        for (int j = sub; j < k; j += 16) {
            const int id = ids[at + j];
            if (id >= 0 && id < e) tile[r * e + id] = (T)(weights[at + j] * (g[at + j] - dot));
        }
    }
    __syncthreads();
    T *o = out + row0 * e;
    if (pieces) {  // every workgroup's rows start on 16 bytes
        const int full = held * (int)sizeof(T) / 16;
        for (int i = tid; i < full; i += 256) reinterpret_cast<float4 *>(o)[i] = reinterpret_cast<const float4 *>(tile_at)[i];
        for (int i = full * 16 / (int)sizeof(T) + tid; i < held; i += 256) o[i] = tile[i];
    } else {
        for (int i = tid; i < held; i += 256) o[i] = tile[i];
    }
}

// ---- pairs sorted by modality ----
// Stable counting sort in three launches, or in one where a single workgroup has all pairs: pairs of each modality per run, prefix
// over the runs, places.  The ids are read twice, order and position written once (1.47 M pairs over 200: 24 MB, 5 + 9 + 16 us;
// bound by the way of the counts through LDS, not by bytes).  A wave owns a run of pairs and goes through it 64 at a time; lanes
// with the same modality find each other by ballots over the modality's bits, so a pair's place is (pairs of its modality before
// these 64) + (lanes below).
__device__ __forceinline__ int pair_key(int id, int e) { return id >= 0 && id < e ? id : e; }

__device__ __forceinline__ uint64_t same_key_lanes(int key, int bits, bool valid) {
    uint64_t mask = __ballot(valid);
    for (int b = 0; b < bits; ++b) {
        const uint64_t ones = __ballot((key >> b) & 1);
        mask &= ((key >> b) & 1) ? ones : ~ones;
    }
    return mask;
}

// counts[b * (e + 1) + x] = pairs of modality x in workgroup b's run
__global__ __launch_bounds__(256) void k_pairs_count(const int32_t *__restrict__ ids, int64_t pairs, int e, int run,
                                                     int32_t *__restrict__ counts) {
    extern __shared__ int hist[];
    for (int i = threadIdx.x; i <= e; i += 256) hist[i] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * run, hi = lo + run < pairs ? lo + run : pairs;
    for (int64_t i = lo + threadIdx.x; i < hi; i += 256) atomicAdd(&hist[pair_key(ids[i], e)], 1);
    __syncthreads();
    for (int i = threadIdx.x; i <= e; i += 256) counts[(int64_t)blockIdx.x * (e + 1) + i] = hist[i];
}

// counts -> the exclusive prefix over the workgroups, and the modality's total.  16 modalities and 64 parts a workgroup.
__global__ __launch_bounds__(1024) void k_pairs_scan(int32_t *__restrict__ counts, int blocks, int e, int32_t *__restrict__ totals) {
    __shared__ int part[64][16];
    const int m = threadIdx.x & 15, x = blockIdx.x * 16 + m, p = threadIdx.x >> 4;
    const int per = (blocks + 63) / 64;
    const int lo = p * per < blocks ? p * per : blocks, hi = lo + per < blocks ? lo + per : blocks;
    int sum = 0;
    if (x <= e)
        for (int b = lo; b < hi; ++b) sum += counts[(int64_t)b * (e + 1) + x];
    part[p][m] = sum;
    __syncthreads();
    int before = 0, all = 0;
    for (int i = 0; i < 64; ++i) {
        const int v = part[i][m];
        if (i < p) before += v;
        all += v;
    }
    if (x <= e) {
        for (int b = lo; b < hi; ++b) {
            const int v = counts[(int64_t)b * (e + 1) + x];
            counts[(int64_t)b * (e + 1) + x] = before;
            before += v;
        }
        if (p == 0) totals[x] = all;
    }
}

// exclusive prefix sum of v[0 .. m) in LDS, by the whole workgroup of W waves; scratch: W ints
template <int W>
__device__ __forceinline__ void scan_lds(int *v, int m, int *scratch) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int base = 0;
    for (int i0 = 0; i0 < m; i0 += W * 64) {
        const int i = i0 + tid;
        const int mine = i < m ? v[i] : 0;
        int sum = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int u = __shfl_up(sum, d);
            if (lane >= d) sum += u;
        }
        if (lane == 63) scratch[wave] = sum;
        __syncthreads();
        int before = base, all = 0;
        for (int w = 0; w < W; ++w) {
            if (w < wave) before += scratch[w];
            all += scratch[w];
        }
        if (i < m) v[i] = before + sum - mine;
        base += all;
        __syncthreads();
    }
}

// W waves; run: pairs per workgroup, a multiple of 64 * W.  counts / totals NULL: one workgroup has all the pairs.
template <int W>
__global__ __launch_bounds__(64 * W) void k_pairs_place(const int32_t *__restrict__ ids, int64_t pairs, int e, int bits, int run,
                                                        const int32_t *__restrict__ counts, const int32_t *__restrict__ totals,
                                                        int32_t *__restrict__ offsets, int32_t *__restrict__ order,
                                                        int32_t *__restrict__ position) {
    extern __shared__ int lds[];  // start[e + 1], next[W][e + 1], scratch[W]
    int *start = lds, *next = lds + (e + 1), *scratch = next + W * (e + 1);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t lo = (int64_t)blockIdx.x * run + (int64_t)wave * (run / W);
    const int64_t end = lo + run / W < pairs ? lo + run / W : pairs;
    for (int i = tid; i < W * (e + 1); i += 64 * W) next[i] = 0;
    __syncthreads();
    int *here = next + wave * (e + 1);
    for (int64_t i = lo + lane; i < end; i += 64) atomicAdd(&here[pair_key(ids[i], e)], 1);
    __syncthreads();
    for (int x = tid; x <= e; x += 64 * W) {
        int all = 0;
        for (int w = 0; w < W; ++w) {  // the waves' shares of this modality, one behind the other
            const int v = next[w * (e + 1) + x];
            next[w * (e + 1) + x] = all;
            all += v;
        }
        start[x] = totals != nullptr ? totals[x] : all;
    }
    __syncthreads();
    scan_lds<W>(start, e + 1, scratch);
    if (blockIdx.x == 0)
        for (int x = tid; x <= e; x += 64 * W) offsets[x] = start[x];
    for (int x = tid; x <= e; x += 64 * W) {
        const int at = start[x] + (counts != nullptr ? counts[(int64_t)blockIdx.x * (e + 1) + x] : 0);
        for (int w = 0; w < W; ++w) next[w * (e + 1) + x] += at;
    }
    __syncthreads();
    volatile int *mine = here;
    for (int64_t i0 = lo; i0 < end; i0 += 64) {
        const int64_t i = i0 + lane;
        const bool valid = i < end;
        const int key = valid ? pair_key(ids[i], e) : e;
        const uint64_t peers = same_key_lanes(key, bits, valid);
        const uint64_t below = peers & ((1ull << lane) - 1);
        const int at = valid ? mine[key] + __popcll(below) : 0;
        __builtin_amdgcn_wave_barrier();
        if (valid && below == 0) mine[key] = at + __popcll(peers);
        __builtin_amdgcn_wave_barrier();
        if (valid) {
            position[i] = at;
            order[at] = (int32_t)i;
        }
    }
}

// ---- rows to their pairs and back ----
// N elements at any address an element can have (the card reads and writes 16 bytes wherever they start)
template <typename T, int N>
struct Pack {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T>
struct Pack<T, 1> {
    typedef T type;
};
template <typename T, int N>
__device__ __forceinline__ void unpack(const typename Pack<T, N>::type &v, float *f) {
    if constexpr (N == 1) f[0] = up(v);
    else {
#pragma unroll
        for (int e = 0; e < N; ++e) f[e] = up(v[e]);
    }
}
template <typename T, int N>
__device__ __forceinline__ typename Pack<T, N>::type pack(const float *f) {
    typename Pack<T, N>::type v;
    if constexpr (N == 1) v = (T)f[0];
    else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = (T)f[e];
    }
    return v;
}
// A row of d >= N elements as ceil(d / N) pieces of N: the last one starts at d - N and says some of the one before it again
__device__ __forceinline__ int piece_at(int c, int d, int n) { return c * n + n <= d ? c * n : d - n; }

// Rows of pairs are read and written once.  More of them than the 256 MB memory-side cache holds go past the caches (ONCE: there
// and back with gradients over 1.47 M rows of 384 bytes 637 us, 745 us without); fewer are likely still there for the next kernel
// (143 760 rows of 192 bytes: the two sums 13 us, 17 us past the caches).
template <bool ONCE, typename T, int N>
__device__ __forceinline__ typename Pack<T, N>::type load_row(const T *p) {
    const auto *v = reinterpret_cast<const typename Pack<T, N>::type *>(p);
    if constexpr (ONCE) return __builtin_nontemporal_load(v);
    else return *v;
}
template <bool ONCE, typename T, int N>
__device__ __forceinline__ void store_row(T *p, const typename Pack<T, N>::type &v) {
    auto *to = reinterpret_cast<typename Pack<T, N>::type *>(p);
    if constexpr (ONCE) __builtin_nontemporal_store(v, to);
    else *to = v;
}

// Places come from the caller, and a plan may be another's: one that is none of the n * k rows (below 2^31) is left out, neither read
// nor written.
__device__ __forceinline__ bool is_place(int32_t p, uint32_t rows) { return (uint32_t)p < rows; }

// rows[position[t][j]] = x[t], zero where the pair has no modality; one thread per N elements of a token, which it reads once and
// writes k times.  I: an index that holds the number of threads (divisions of 64 bits cost more than the copy).  HBM-bound: 73 568
// rows of 96 floats to 1.47 M places 112 us, 5.3 TB/s.
template <typename T, int N, bool ONCE, typename I>
__global__ __launch_bounds__(256) void k_dispatch(const T *__restrict__ x, int64_t n, int d, int64_t ld, int k,
                                                  const int32_t *__restrict__ position, const int32_t *__restrict__ held_at,
                                                  T *__restrict__ rows) {
    typedef typename Pack<T, N>::type vec;
    const int per = (d + N - 1) / N;
    const I total = (I)n * per;
    const int held = *held_at;
    const uint32_t places = (uint32_t)n * (uint32_t)k;
    for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += (I)gridDim.x * 256) {
        const int64_t t = i / per;
        const int c = piece_at((int)(i - (I)t * per), d, N);
        const vec v = *reinterpret_cast<const vec *>(x + t * ld + c);
        const vec zero = {};
        for (int j = 0; j < k; ++j) {
            const int32_t p = position[t * k + j];
            if (is_place(p, places)) store_row<ONCE, T, N>(rows + (int64_t)p * d + c, p < held ? v : zero);
        }
    }
}

// y[t] = sum_j weights[t][j] rows[position[t][j]] (weights NULL: all one), pairs without a modality left out.  One thread per N
// elements of a token; four rows are in flight at a time (what does not count is dropped after the load).  HBM-bound: the same sizes
// back 100 us, 5.9 TB/s.
template <typename T, int N, bool ONCE, typename I>
__global__ __launch_bounds__(256) void k_combine(const T *__restrict__ rows, int64_t n, int d, int k,
                                                 const int32_t *__restrict__ position, const int32_t *__restrict__ held_at,
                                                 const float *__restrict__ weights, T *__restrict__ y) {
    typedef typename Pack<T, N>::type vec;
    const int per = (d + N - 1) / N;
    const I total = (I)n * per;
    const int held = *held_at;
    const uint32_t places = (uint32_t)n * (uint32_t)k;
    for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += (I)gridDim.x * 256) {
        const int64_t t = i / per;
        const int c = piece_at((int)(i - (I)t * per), d, N);
        const int32_t *at = position + t * k;
        const float *wt = weights + t * k;
        float sum[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = 0.f;
        for (int j0 = 0; j0 < k; j0 += 4) {
            vec v[4];
            float w[4];
            bool in[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int j = j0 + q < k ? j0 + q : k - 1;
                const int32_t p = at[j];
                const bool there = is_place(p, places);
                in[q] = there && p < held && j0 + q < k;
                v[q] = load_row<ONCE, T, N>(rows + (int64_t)(there ? p : 0) * d + c);
                w[q] = weights != nullptr ? wt[j] : 1.f;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float f[N];
                unpack<T, N>(v[q], f);
                if (in[q]) {
#pragma unroll
                    for (int e = 0; e < N; ++e) sum[e] = fmaf(w[q], f[e], sum[e]);
                }
            }
        }
        store_row<ONCE, T, N>(y + t * d + c, pack<T, N>(sum));
    }
}

// the sum over L neighbouring lanes, the same in each
template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
    v += turn_f32<0xB1>(v);                          // lane ^ 1
    v += turn_f32<0x4E>(v);                          // lane ^ 2
    v += turn_f32<0x141>(v);                         // the other four of eight
    if constexpr (L >= 16) v += turn_f32<0x140>(v);  // the other eight of sixteen
    if constexpr (L >= 32) v += __shfl_xor(v, 16);
    if constexpr (L >= 64) v += __shfl_xor(v, 32);
    return v;
}

// grad_rows[position[t][j]] = weights[t][j] g[t] (zero behind the last modality); grad_weights[t][j] = <rows[...], g[t]>.
// L lanes share a token and hold C pieces of N elements of its gradient each; four rows are in flight at a time.  HBM-bound, as
// much read as written: the same sizes 288 us, 4.0 TB/s (a copy 4.8).
template <typename T, int N, int L, int C, bool ONCE>
__global__ __launch_bounds__(256) void k_combine_grad(const T *__restrict__ rows, const T *__restrict__ g, int64_t n, int d, int k,
                                                      const int32_t *__restrict__ position, const int32_t *__restrict__ held_at,
                                                      const float *__restrict__ weights, T *__restrict__ grad_rows,
                                                      float *__restrict__ grad_weights) {
    typedef typename Pack<T, N>::type vec;
    constexpr int Q = C == 1 ? 4 : 1;
    const int per = (d + N - 1) / N, sub = threadIdx.x % L;
    const int held = *held_at;
    const uint32_t places = (uint32_t)n * (uint32_t)k, live = held < 0 ? 0 : min((uint32_t)held, places);
    for (int64_t t = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L; t < n; t += (int64_t)gridDim.x * (256 / L)) {
        const int32_t *at = position + t * k;
        for (int c0 = 0; c0 < per; c0 += L * C) {
            float gv[C][N];
            int from[C], again[C];  // where the lane's pieces start, and how many of their elements another piece has too
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int x = c0 + c * L + sub;
                from[c] = x < per ? piece_at(x, d, N) : 0;
                again[c] = x < per ? x * N - from[c] : N;
                unpack<T, N>(*reinterpret_cast<const vec *>(g + t * d + from[c]), gv[c]);
            }
            for (int j0 = 0; j0 < k; j0 += Q) {
                int32_t p[Q];
                vec v[Q][C];
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    p[q] = at[j0 + q < k ? j0 + q : k - 1];
                    if (grad_weights != nullptr) {
#pragma unroll
                        for (int c = 0; c < C; ++c)
                            v[q][c] = load_row<ONCE, T, N>(rows + (int64_t)(is_place(p[q], places) ? p[q] : 0) * d + from[c]);
                    }
                }
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    const int j = j0 + q;
                    if (j >= k) break;
                    const bool in = is_place(p[q], live);
                    if (grad_rows != nullptr) {
                        const float w = in ? weights[t * k + j] : 0.f;
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            float o[N];
#pragma unroll
                            for (int e = 0; e < N; ++e) o[e] = in ? w * gv[c][e] : 0.f;
                            if (c0 + c * L + sub < per && is_place(p[q], places))
                                store_row<ONCE, T, N>(grad_rows + (int64_t)p[q] * d + from[c], pack<T, N>(o));
                        }
                    }
                    if (grad_weights != nullptr) {
                        float dot = 0.f;
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            float rv[N];
                            unpack<T, N>(v[q][c], rv);
                            if (in) {
#pragma unroll
                                for (int e = 0; e < N; ++e) dot = e >= again[c] ? fmaf(rv[e], gv[c][e], dot) : dot;
                            }
                        }
                        dot = lanes_sum<L>(dot);
                        // a row longer than L * C pieces comes in parts, added in their order
                        if (sub == 0) grad_weights[t * k + j] = c0 == 0 ? dot : grad_weights[t * k + j] + dot;
                    }
                }
            }
        }
    }
}

unsigned blocks_of(int64_t items, int per_block) {
    const int64_t b = (items + per_block - 1) / per_block;
    return (unsigned)(b < 1 ? 1 : (b > 256 * 32 ? 256 * 32 : b));
}

template <typename T, int L, int V, int KB>
int launch_topk(const void *scores, int64_t n, int e, int64_t ld, int k, int normalize, int32_t *ids, float *weights, float *stats,
                hipStream_t s) {
    constexpr int KEY = (int)sizeof(typename RouteKey<T>::type);
    const int lds = ((V < k ? V : k) + 1) * 256 * KEY;
    constexpr int64_t ROWS = (int64_t)(256 / L) << 22;  // rows of a launch: a grid holds less than 2^32 threads
    MTP_SET_MAX_LDS_ONCE((k_route_topk<T, L, V, KB>), (V + 1) * 256 * KEY);
    for (int64_t r = 0; r < n; r += ROWS) {
        const int64_t m = n - r < ROWS ? n - r : ROWS;
        hipLaunchKernelGGL((k_route_topk<T, L, V, KB>), dim3((unsigned)((m + 256 / L - 1) / (256 / L))), dim3(256), lds, s,
                           reinterpret_cast<const T *>(scores) + r * ld, m, e, ld, k, normalize, ids + r * k, weights + r * k,
                           stats == nullptr ? nullptr : stats + r * 2);
        MTP_LAUNCH_CHECK();
    }
    return MTP_OK;
}

template <typename T, int L, int V>
int route_by_k(const void *scores, int64_t n, int e, int64_t ld, int k, int normalize, int32_t *ids, float *weights, float *stats,
               hipStream_t s) {
    if (k <= L) return launch_topk<T, L, V, 1>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    if (k <= 2 * L) return launch_topk<T, L, V, 2>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    if constexpr (L == 32) return launch_topk<T, L, V, 4>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    if constexpr (L == 16) return launch_topk<T, L, V, 8>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    if constexpr (L == 8) {
        if (k <= 4 * L) return launch_topk<T, L, V, 4>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        return launch_topk<T, L, V, 16>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    }
    mtp_set_error("mtp_route_topk: k=%d", k);
    return MTP_E_ARG;
}

template <typename T>
int route(const void *scores, int64_t n, int e, int64_t ld, int k, int normalize, int32_t *ids, float *weights, float *stats,
          hipStream_t s) {
    // More lanes a row: shorter sorts and longer maxima, k of them.  100 000 rows, microseconds for k = 1 / 7 / 20 / 64:
    //   400 float     16 lanes 67 / 73 / 86 / 160, 32 lanes 51 / 64 / 94 / 189, 64 lanes 51 / 84 / 152 / 415
    //   900 bfloat16  16 lanes 92 / 100 / 110 / 154, 32 lanes 66 / 75 / 91 / 143, 64 lanes 60 / 77 / 112 / 225
    // 400 000 rows, k = 4 / 20 / 40 / 100:
    //   50 bfloat16   8 lanes 22 / 39 / 71, 16 lanes 29 / 57 / 103;  float 30 / 56 / 101, 39 / 90 / 176
    //   100 bfloat16  8 lanes 35 / 52 / 83 / 130, 16 lanes 65 / 92 / 136 / 227;  float 54 / 81 / 129 / 217, 101 / 152 / 228 / 409
    //   200 bfloat16  8 lanes 67 / 89 / 123 / 172, 16 lanes 63 / 92 / 139 / 226;  float 127 / 157 / 260 / 377, 107 / 159 / 233 / 419
    // Few rows: one wave a row, since the card is not full anyway.
    if (n >= 1024 && e <= 1024) {
        if (e <= 32) return route_by_k<T, 8, 4>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        if (e <= 64) return route_by_k<T, 8, 8>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        if (e <= 128) return route_by_k<T, 8, 16>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        if (e <= 256 && sizeof(T) == 2 && k > 32) return route_by_k<T, 8, 32>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        if (e <= 256) return route_by_k<T, 16, 16>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        if (e <= 512 && k > 8) return route_by_k<T, 16, 32>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        if (e <= 512) return route_by_k<T, 32, 16>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
        return route_by_k<T, 32, 32>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    }
    if (e <= 256) return route_by_k<T, 64, 4>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    if (e <= 1024) return route_by_k<T, 64, 16>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
    return route_by_k<T, 64, 64>(scores, n, e, ld, k, normalize, ids, weights, stats, s);
}

// Up to here one workgroup sorts them all, in one launch (8192 pairs over 200: 13.6 us, 11.6 in three launches; 4096: 9.4 / 11.5).
constexpr int PAIRS_ALONE = 8192;
bool pairs_alone(int64_t pairs, int e) { return pairs <= PAIRS_ALONE && (int64_t)17 * (e + 1) * 4 + 64 <= 128 * 1024; }
// Pairs of a workgroup: short runs end sooner, long ones have fewer counts to add (143 760 pairs over 200: 15.2 us with runs of 512,
// 18.4 of 2048; 600 000: 21.3 of 1024, 25.9 of 512; 1 471 360: 30.3 of 2048, 37.6 of 1024).
// The runs' counts take no more room than the ids, or than COUNTS_BYTES: longer ones where there are many modalities.
constexpr int64_t COUNTS_BYTES = 64ll << 20;
int64_t pairs_blocks(int64_t pairs, int run) { return (pairs + run - 1) / run; }
int pairs_run(int64_t pairs, int e) {
    int run = pairs < 256 * 1024 ? 512 : pairs < 1024 * 1024 ? 1024 : 2048;
    const int64_t most = pairs * 4 > COUNTS_BYTES ? pairs * 4 : COUNTS_BYTES;
    while ((pairs_blocks(pairs, run) + 1) * (int64_t)(e + 1) * 4 > most) run *= 2;
    return run;
}

constexpr int64_t CACHE_BYTES = 256ll << 20;

template <typename T, int N, bool ONCE>
int launch_dispatch(const void *x, int64_t n, int d, int64_t ld, int k, const int32_t *position, const int32_t *held, void *rows,
                    hipStream_t s) {
    const int64_t threads = n * ((d + N - 1) / N);
    const dim3 grid(blocks_of(threads, 256));
    if (threads < 1ll << 31)
        hipLaunchKernelGGL((k_dispatch<T, N, ONCE, uint32_t>), grid, dim3(256), 0, s, reinterpret_cast<const T *>(x), n, d, ld, k,
                           position, held, reinterpret_cast<T *>(rows));
    else
        hipLaunchKernelGGL((k_dispatch<T, N, ONCE, int64_t>), grid, dim3(256), 0, s, reinterpret_cast<const T *>(x), n, d, ld, k,
                           position, held, reinterpret_cast<T *>(rows));
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

template <typename T>
int dispatch(const void *x, int64_t n, int d, int64_t ld, int k, const int32_t *position, const int32_t *held, void *rows,
             hipStream_t s) {
    constexpr int N = 16 / (int)sizeof(T);
    if (d < N) return launch_dispatch<T, 1, false>(x, n, d, ld, k, position, held, rows, s);
    if (n * k * d * (int64_t)sizeof(T) > CACHE_BYTES) return launch_dispatch<T, N, true>(x, n, d, ld, k, position, held, rows, s);
    return launch_dispatch<T, N, false>(x, n, d, ld, k, position, held, rows, s);
}

template <typename T, int N, bool ONCE>
int launch_combine(const void *rows, int64_t n, int d, int k, const int32_t *position, const int32_t *held, const float *weights,
                   void *y, hipStream_t s) {
    const int64_t threads = n * ((d + N - 1) / N);
    const dim3 grid(blocks_of(threads, 256));
    if (threads < 1ll << 31)
        hipLaunchKernelGGL((k_combine<T, N, ONCE, uint32_t>), grid, dim3(256), 0, s, reinterpret_cast<const T *>(rows), n, d, k,
                           position, held, weights, reinterpret_cast<T *>(y));
    else
        hipLaunchKernelGGL((k_combine<T, N, ONCE, int64_t>), grid, dim3(256), 0, s, reinterpret_cast<const T *>(rows), n, d, k,
                           position, held, weights, reinterpret_cast<T *>(y));
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

template <typename T>
int combine(const void *rows, int64_t n, int d, int k, const int32_t *position, const int32_t *held, const float *weights, void *y,
            hipStream_t s) {
    constexpr int N = 16 / (int)sizeof(T);
    if (d < N) return launch_combine<T, 1, false>(rows, n, d, k, position, held, weights, y, s);
    if (n * k * d * (int64_t)sizeof(T) > CACHE_BYTES) return launch_combine<T, N, true>(rows, n, d, k, position, held, weights, y, s);
    return launch_combine<T, N, false>(rows, n, d, k, position, held, weights, y, s);
}

template <typename T, int N, int L, int C, bool ONCE = false>
int launch_combine_grad(const void *rows, const void *g, int64_t n, int d, int k, const int32_t *position, const int32_t *held,
                        const float *weights, void *grad_rows, float *grad_weights, hipStream_t s) {
    hipLaunchKernelGGL((k_combine_grad<T, N, L, C, ONCE>), dim3(blocks_of(n, 256 / L)), dim3(256), 0, s,
                       reinterpret_cast<const T *>(rows), reinterpret_cast<const T *>(g), n, d, k, position, held, weights,
                       reinterpret_cast<T *>(grad_rows), grad_weights);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

template <typename T>
int combine_grad(const void *rows, const void *g, int64_t n, int d, int k, const int32_t *position, const int32_t *held,
                 const float *weights, void *grad_rows, float *grad_weights, hipStream_t s) {
    constexpr int N = 16 / (int)sizeof(T);
    const int per = (d + N - 1) / N;
    const bool once = n * k * d * (int64_t)sizeof(T) > CACHE_BYTES;
    if (d < N) return launch_combine_grad<T, 1, 8, 1>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
    if (per <= 8) return launch_combine_grad<T, N, 8, 1>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
    if (per <= 16) {
        if (once) return launch_combine_grad<T, N, 16, 1, true>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
        return launch_combine_grad<T, N, 16, 1>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
    }
    if (per <= 32) {
        if (once) return launch_combine_grad<T, N, 32, 1, true>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
        return launch_combine_grad<T, N, 32, 1>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
    }
    if (once) return launch_combine_grad<T, N, 64, 2, true>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
    return launch_combine_grad<T, N, 64, 2>(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights, s);
}

bool known_type(int dtype) { return dtype == MTP_FLOAT || dtype == MTP_BFLOAT16 || dtype == MTP_HALF; }

}  // namespace

#define ROUTE_BY_TYPE(dtype, call) ((dtype) == MTP_FLOAT ? call<float> : (dtype) == MTP_BFLOAT16 ? call<__bf16> : call<_Float16>)

extern "C" int mtp_route_topk(int dtype, const void *scores, int64_t n, int e, int64_t ld, int k, int normalize, int32_t *ids,
                              float *weights, float *stats, void *stream) {
    MTP_REQUIRE(known_type(dtype), "mtp_route_topk: unknown type %d", dtype);
    MTP_REQUIRE(n >= 0 && n <= 0x7fffffff && e >= 1 && e <= ROUTE_MAX_E && k >= 1 && k <= e && k <= ROUTE_MAX_K && ld >= e,
                "mtp_route_topk: bad shape n=%lld e=%d k=%d ld=%lld", (long long)n, e, k, (long long)ld);
    if (n == 0) return MTP_OK;
    MTP_REQUIRE(scores && ids && weights, "mtp_route_topk: null pointer");
    return ROUTE_BY_TYPE(dtype, route)(scores, n, e, ld, k, normalize != 0, ids, weights, stats, mtp_stream(stream));
}

extern "C" int mtp_route_topk_grad(int dtype, const void *scores, int64_t n, int e, int64_t ld, int k, int normalize,
                                   const int32_t *ids, const float *weights, const float *stats, const float *g, void *out,
                                   void *stream) {
    MTP_REQUIRE(known_type(dtype), "mtp_route_topk_grad: unknown type %d", dtype);
    MTP_REQUIRE(n >= 0 && n <= 0x7fffffff && e >= 1 && e <= ROUTE_MAX_E && k >= 1 && k <= e && k <= ROUTE_MAX_K && ld >= e,
                "mtp_route_topk_grad: bad shape n=%lld e=%d k=%d ld=%lld", (long long)n, e, k, (long long)ld);
    if (n == 0) return MTP_OK;
    MTP_REQUIRE(scores && ids && weights && stats && g && out, "mtp_route_topk_grad: null pointer");
    // 16 KB of rows; eight rows of any length start on 16 bytes
    const int sz = dtype == MTP_FLOAT ? 4 : 2;
    int rows_per = 16384 / (e * sz) / 8 * 8;
    if (rows_per == 0) rows_per = 8 * e * sz <= 56 * 1024 ? 8 : 1;
    if (rows_per > 64) rows_per = 64;
    const int pieces = (uintptr_t)out % 16 == 0 && (int64_t)rows_per * e * sz % 16 == 0;
    const int lds = (rows_per * 4 + 15) / 16 * 16 + (rows_per * e * sz + 15) / 16 * 16;
    hipStream_t s = mtp_stream(stream);
    const int64_t most = (int64_t)rows_per << 22;  // rows of a launch: a grid holds less than 2^32 threads
    for (int64_t r = 0; r < n; r += most) {
        const int64_t m = n - r < most ? n - r : most;
        const int64_t at = r * ld * sz, to = r * e * sz;
        const void *x = reinterpret_cast<const char *>(scores) + at;
        void *o = reinterpret_cast<char *>(out) + to;
        const dim3 grid((unsigned)((m + rows_per - 1) / rows_per));
#define ROUTE_GRAD(T)                                                                                                          \
    hipLaunchKernelGGL(k_route_grad<T>, grid, dim3(256), lds, s, (const T *)x, m, e, ld, k, normalize, ids + r * k, weights + r * k, \
                       stats + r * 2, g + r * k, (T *)o, rows_per, pieces)
        if (dtype == MTP_FLOAT) ROUTE_GRAD(float);
        else if (dtype == MTP_BFLOAT16) ROUTE_GRAD(__bf16);
        else ROUTE_GRAD(_Float16);
#undef ROUTE_GRAD
        MTP_LAUNCH_CHECK();
    }
    return MTP_OK;
}

extern "C" int64_t mtp_sort_pairs_workspace_bytes(int64_t pairs, int e) {
    if (pairs < 0 || e < 1 || pairs_alone(pairs, e)) return 0;
    return (pairs_blocks(pairs, pairs_run(pairs, e)) + 1) * (int64_t)(e + 1) * 4;
}

extern "C" int mtp_sort_pairs(const int32_t *ids, int64_t pairs, int e, int32_t *offsets, int32_t *order, int32_t *position, void *ws,
                              size_t ws_bytes, void *stream) {
    MTP_REQUIRE(pairs >= 0 && pairs <= 0x7fffffff && e >= 1 && e <= ROUTE_MAX_E, "mtp_sort_pairs: bad shape pairs=%lld e=%d",
                (long long)pairs, e);
    MTP_REQUIRE(offsets && (pairs == 0 || (ids && order && position)), "mtp_sort_pairs: null pointer");
    int bits = 1;
    while ((1 << bits) <= e) ++bits;
    hipStream_t s = mtp_stream(stream);
    if (pairs_alone(pairs, e)) {
        const int run = pairs == 0 ? 1024 : (int)((pairs + 1023) / 1024 * 1024);
        const int lds = (17 * (e + 1) + 16) * 4;
        MTP_SET_MAX_LDS_ONCE(k_pairs_place<16>, 128 * 1024);
        hipLaunchKernelGGL(k_pairs_place<16>, dim3(1), dim3(1024), lds, s, ids, pairs, e, bits, run, (const int32_t *)nullptr,
                           (const int32_t *)nullptr, offsets, order, position);
        MTP_LAUNCH_CHECK();
        return MTP_OK;
    }
    if ((int64_t)ws_bytes < mtp_sort_pairs_workspace_bytes(pairs, e) || ws == nullptr) {
        mtp_set_error("mtp_sort_pairs: workspace of %zu bytes, needs %lld", ws_bytes,
                      (long long)mtp_sort_pairs_workspace_bytes(pairs, e));
        return MTP_E_WORKSPACE;
    }
    const int run = pairs_run(pairs, e), blocks = (int)pairs_blocks(pairs, run);
    int32_t *counts = reinterpret_cast<int32_t *>(ws), *totals = counts + (int64_t)blocks * (e + 1);
    hipLaunchKernelGGL(k_pairs_count, dim3(blocks), dim3(256), (e + 1) * 4, s, ids, pairs, e, run, counts);
    MTP_LAUNCH_CHECK();
    hipLaunchKernelGGL(k_pairs_scan, dim3((e + 16) / 16), dim3(1024), 0, s, counts, blocks, e, totals);
    MTP_LAUNCH_CHECK();
    MTP_SET_MAX_LDS_ONCE(k_pairs_place<4>, (5 * (ROUTE_MAX_E + 1) + 4) * 4);
    hipLaunchKernelGGL(k_pairs_place<4>, dim3(blocks), dim3(256), (5 * (e + 1) + 4) * 4, s, ids, pairs, e, bits, run, counts,
                       totals, offsets, order, position);
    MTP_LAUNCH_CHECK();
    return MTP_OK;
}

#define CHECK_ROWS(who)                                                                                                     \
    MTP_REQUIRE(known_type(dtype), who ": unknown type %d", dtype);                                                         \
    MTP_REQUIRE(n >= 0 && k >= 1 && d >= 1 && d <= (1 << 20) && n * (int64_t)k <= 0x7fffffff, who ": bad shape n=%lld k=%d d=%d", \
                (long long)n, k, d);                                                                                        \
    if (n == 0) return MTP_OK

extern "C" int mtp_dispatch_rows(int dtype, const void *x, int64_t n, int d, int64_t ld, int k, const int32_t *position,
                                 const int32_t *held, void *rows, void *stream) {
    CHECK_ROWS("mtp_dispatch_rows");
    MTP_REQUIRE(ld >= d, "mtp_dispatch_rows: row distance below the row's length");
    MTP_REQUIRE(x && position && held && rows, "mtp_dispatch_rows: null pointer");
    return ROUTE_BY_TYPE(dtype, dispatch)(x, n, d, ld, k, position, held, rows, mtp_stream(stream));
}

extern "C" int mtp_combine_rows(int dtype, const void *rows, int64_t n, int d, int k, const int32_t *position, const int32_t *held,
                                const float *weights, void *y, void *stream) {
    CHECK_ROWS("mtp_combine_rows");
    MTP_REQUIRE(rows && position && held && y, "mtp_combine_rows: null pointer");
    return ROUTE_BY_TYPE(dtype, combine)(rows, n, d, k, position, held, weights, y, mtp_stream(stream));
}

extern "C" int mtp_combine_rows_grad(int dtype, const void *rows, const void *g, int64_t n, int d, int k, const int32_t *position,
                                     const int32_t *held, const float *weights, void *grad_rows, float *grad_weights, void *stream) {
    CHECK_ROWS("mtp_combine_rows_grad");
    MTP_REQUIRE(rows && g && position && held && weights && (grad_rows || grad_weights), "mtp_combine_rows_grad: null pointer");
    return ROUTE_BY_TYPE(dtype, combine_grad)(rows, g, n, d, k, position, held, weights, grad_rows, grad_weights,
                                              mtp_stream(stream));
}
