// Row operators whose order follows from scores: choosing experts for each row (route), the stable
// counting sort of the choices (plan), and the move of the rows into that order and back (dispatch,
// combine), with their gradients.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <cstring>

namespace povs {

// ------------------------------------------------------------------------------------------
// Element types.
// ------------------------------------------------------------------------------------------

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// `BYTES` bytes as one load or store; wider than the element's alignment only where the host has
// checked that every address is a multiple of it.
template <int BYTES> struct Piece;
template <> struct Piece<16> { using type = uint4; };
template <> struct Piece<8> { using type = uint2; };
template <> struct Piece<4> { using type = uint32_t; };
template <> struct Piece<2> { using type = uint16_t; };
template <> struct Piece<1> { using type = uint8_t; };

constexpr unsigned FULL_WARP = 0xffffffffu;

// ------------------------------------------------------------------------------------------
// Route.
// ------------------------------------------------------------------------------------------

struct RouteParams {
    const void* logits; // row r, expert e at logits[r * row_stride + e]
    const float* bias;  // n_experts, or NULL
    int64_t rows;
    int64_t row_stride; // elements
    int32_t n_experts;
    int32_t top_k;
    int32_t sigmoid;
    int32_t n_groups;
    int32_t top_groups;
    int32_t group_max; // a group's score: 1 its highest choice score, 0 the sum of its two highest
    int32_t renormalize;
    float scale;
    int32_t* experts;
    float* weights;
    // Backward only.
    const int32_t* chosen;
    const float* grad_weights;
    void* grad_logits; // contiguous
};

// Order of choice scores as an unsigned number: 0 for what cannot be chosen, 1 for NaN, then the
// numbers from -infinity up (+0 and -0 are the same number).
__device__ __forceinline__ uint64_t order_key(double v)
{
    if (v != v) return 1;
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));
    return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// The largest key of the warp and the lowest index that has it.
__device__ __forceinline__ void warp_best(uint64_t& key, int& index)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint64_t k = __shfl_xor_sync(FULL_WARP, key, o);
        const int i = __shfl_xor_sync(FULL_WARP, index, o);
        if (k > key || (k == key && i < index)) {
            key = k;
            index = i;
        }
    }
}

// One row by one warp with every score in 64 bits, EPL scores per lane (expert lane + 32 * m): the
// definition itself, for rows that 32 bits leave open.
template <typename T, int EPL> __device__ __noinline__ void route_row_exactly(const RouteParams& p, int64_t row)
{
    const int lane = threadIdx.x & 31;
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    const int n = p.n_experts;

    double s[EPL], logit[EPL];
    bool open[EPL]; // can be chosen
#pragma unroll
    for (int m = 0; m < EPL; ++m) {
        const int e = lane + 32 * m;
        s[m] = e < n ? static_cast<double>(to_float(x[e])) : -INFINITY;
        open[m] = e < n && s[m] != -INFINITY;
        logit[m] = s[m];
    }
    if (p.sigmoid) {
#pragma unroll
        for (int m = 0; m < EPL; ++m) s[m] = 1.0 / (1.0 + exp(-s[m]));
    } else {
        double top = -INFINITY;
#pragma unroll
        for (int m = 0; m < EPL; ++m) top = fmax(top, s[m]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(FULL_WARP, top, o));
        if (top == -INFINITY) top = 0.0; // every expert masked, or NaN: exp(-inf) = 0 and NaN stays
        double sum = 0.0;
#pragma unroll
        for (int m = 0; m < EPL; ++m) {
            s[m] = exp(s[m] - top);
            sum += s[m];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL_WARP, sum, o);
        const double inv = 1.0 / sum;
#pragma unroll
        for (int m = 0; m < EPL; ++m) s[m] = open[m] ? s[m] * inv : 0.0;
    }

    // Scores rise with the logits: where nothing is added and no groups are summed the logits' own order
    // stands, also where scores of 64 bits fall together (a NaN score still comes last).
    const bool by_logit = p.bias == nullptr && p.top_groups == p.n_groups;
    uint64_t key[EPL];
#pragma unroll
    for (int m = 0; m < EPL; ++m) {
        const int e = lane + 32 * m;
        const double c = by_logit && s[m] == s[m]         ? logit[m]
                         : p.bias != nullptr && e < n ? s[m] + static_cast<double>(p.bias[e])
                                                      : s[m];
        key[m] = open[m] && c != -INFINITY ? order_key(c) : 0;
    }
    if (p.top_groups < p.n_groups) {
        // Lane g scores group g.  A masked expert counts as -infinity.
        const int size = n / p.n_groups;
        uint64_t mine = 0;
        for (int g = 0; g < p.n_groups; ++g) {
            uint64_t first = 0, second = 0;
            int at = n;
#pragma unroll
            for (int m = 0; m < EPL; ++m) {
                const int e = lane + 32 * m;
                if (e >= g * size && e < (g + 1) * size) {
                    const uint64_t k = key[m] != 0 ? key[m] : order_key(-INFINITY);
                    if (k > first || at == n) {
                        second = first;
                        first = k;
                        at = e;
                    } else if (k > second) {
                        second = k;
                    }
                }
            }
            uint64_t best = first;
            int who = at == n ? n + lane : at;
            warp_best(best, who);
            uint64_t other = who == at ? second : first;
            int unused = 0;
            warp_best(other, unused);
            auto value = [](uint64_t k) {
                return k == 0 ? -INFINITY
                     : k == 1 ? NAN
                              : __longlong_as_double(static_cast<long long>((k >> 63) ? k & 0x7fffffffffffffffull : ~k));
            };
            const double score = p.group_max || size == 1 ? value(best) : value(best) + value(other);
            if (lane == g) mine = order_key(score);
        }
        int before = 0;
        for (int g = 0; g < p.n_groups; ++g) {
            const uint64_t other = __shfl_sync(FULL_WARP, mine, g);
            before += other > mine || (other == mine && g < lane);
        }
        const unsigned kept = __ballot_sync(FULL_WARP, lane < p.n_groups && before < p.top_groups);
#pragma unroll
        for (int m = 0; m < EPL; ++m) {
            const int e = lane + 32 * m;
            if (e < n && !((kept >> (e / size)) & 1)) key[m] = 0;
        }
    }

    int my_expert = -1;
    double my_score = 0.0, total = 0.0;
    for (int j = 0; j < p.top_k; ++j) {
        uint64_t best = 0;
        int at = n;
        double value = 0.0;
#pragma unroll
        for (int m = 0; m < EPL; ++m)
            if (key[m] > best) {
                best = key[m];
                at = lane + 32 * m;
                value = s[m];
            }
        int who = at;
        warp_best(best, who);
        if (best == 0) break;
        const double score = __shfl_sync(FULL_WARP, value, who & 31);
#pragma unroll
        for (int m = 0; m < EPL; ++m)
            if (lane + 32 * m == who) key[m] = 0;
        total += score;
        if (lane == j) {
            my_expert = who;
            my_score = score;
        }
    }
    if (lane < p.top_k) {
        double w = my_expert >= 0 ? my_score * static_cast<double>(p.scale) : 0.0;
        if (p.renormalize) w = total == 0.0 ? 0.0 : w / total;
        p.experts[row * p.top_k + lane] = my_expert;
        p.weights[row * p.top_k + lane] = static_cast<float>(w);
    }
}

__device__ __forceinline__ float warp_max(float v)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(FULL_WARP));
    return r;
}
__device__ __forceinline__ float exp2_fast(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float reciprocal_fast(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
constexpr float LOG2E = 1.44269504f;

// Two highest scores of a group that cancel: their errors grow with each of them, not with their sum.  Elsewhere
// |first| + |second| <= |first + second| + 2.  (A second of -infinity leaves no error.)
__device__ __forceinline__ bool cancels(float first, float second) { return second < -1.0f && first > 1.0f && second > -INFINITY; }

// Chosen scores that sum to less are divided in 64 bits: 32 bits flush scores below 2^-126 to 0, which above
// this is 2^-86 of the sum and less.
constexpr float LEAST_TOTAL = 0x1p-40f;

constexpr int ROUTE_WARPS = 4;

// Choosing in 32 bits what the definition decides in 64.
//
// A choice score c, less the row's highest and plus 3.9998, is a float in [2, 4): its 23 mantissa bits
// are steps of 2^-22, and above an index that counts down they make one whole number per expert whose
// maximum is the next choice, ties by the lowest index (scores 2 and more below the highest all become
// 2 + 2^-22).  Without a bias or groups the order of the scores is the logits', and c is a logit / 8, exact
// but for one rounding of half a step.  Otherwise c is a score from 32-bit arithmetic plus its bias: the
// exponential's argument is rounded by 2^-24 of its size z, z 2^-z <= 0.54, the exponential and the quotient
// are good to 2^-22, a softmax's sum to (EPL + 5) 2^-24: in all below 2^-19 and 2^-24 for each of a lane's
// scores, to which a bias adds 2^-24 of |c|.  Neighbours in the result no further apart than twice that
// (`room` steps), and groups whose scores are as close, are told apart by 64 bits (route_row_exactly), unless logit
// and bias are equal, a tie in either arithmetic.  A group's score has the errors of its two terms, below 2^-18 and
// 2^-23 for each of a lane's scores, and 2^-24 of |first| + |second| and of their sum: `slack` covers two groups'.
// Rows with NaN, infinities, terms that cancel or too few experts end there too.
//
// A warp per row: 2.3 us for 13 rows of 64 experts, 20 us for 16384 x 256 float32 (0.9 TB/s), 36 us for
// 16384 x 512 with a bias.  Bound by instructions (about 950 a row with 8 groups, 560 without).
template <typename T, int EPL, bool VECTOR>
__global__ void __launch_bounds__(32 * ROUTE_WARPS, EPL <= 8 ? 8 : EPL <= 16 ? 5 : 3) povs_route_kernel(const __grid_constant__ RouteParams p)
{
    // Experts of a lane: V neighbours at a time (one load) where the rows' alignment allows.
    constexpr int WIDEST = 16 / sizeof(T), V = !VECTOR ? 1 : EPL < WIDEST ? EPL : WIDEST;
    constexpr int INDEX_BITS = EPL > 16 ? 10 : 9;
    constexpr uint32_t INDEX_MASK = (1u << INDEX_BITS) - 1;
    constexpr float TOP = 3.9998f, LOWEST = 2.0f + 1.0f / (1 << (31 - INDEX_BITS));
    __shared__ float scores[ROUTE_WARPS][32 * EPL + 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = p.n_experts;
    const bool grouped = p.top_groups < p.n_groups, by_logit = p.bias == nullptr && !grouped;
    const int size = n / p.n_groups;
    auto expert = [&](int m) { return (m / V) * 32 * V + lane * V + m % V; };
    // Groups of whole loads, on a run of lanes whose number is a power of two, are scored in registers
    // (`run` lanes), others through shared memory (`span` lanes each).
    const int run = size % V == 0 && size / V <= 32 && (size / V & (size / V - 1)) == 0 ? size / V : 0;
    int span_log2 = 5;
    while ((p.n_groups << span_log2) > 32) --span_log2;
    const int span = 1 << span_log2, my_group = lane >> span_log2, my_place = lane & (span - 1);
    int group[EPL];
#pragma unroll
    for (int m = 0; m < EPL; ++m) group[m] = grouped && expert(m) < n ? expert(m) / size : 0;
    constexpr bool KEEP_BIAS = EPL <= 8; // in registers, over the rows
    float kept_bias[KEEP_BIAS ? EPL : 1];
#pragma unroll
    for (int m = 0; m < (KEEP_BIAS ? EPL : 0); ++m) kept_bias[m] = p.bias != nullptr && expert(m) < n ? p.bias[expert(m)] : 0.0f;

    const int64_t stride = static_cast<int64_t>(gridDim.x) * ROUTE_WARPS;
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * ROUTE_WARPS + warp; row < p.rows; row += stride) {
        const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
        float c[EPL];
#pragma unroll
        for (int i = 0; i < EPL / V; ++i) {
            const int e = expert(i * V);
            struct alignas(V * sizeof(T)) Few {
                T v[V];
            };
            if (e < n) {
                const Few few = *reinterpret_cast<const Few*>(x + e);
#pragma unroll
                for (int j = 0; j < V; ++j) c[i * V + j] = to_float(few.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) c[i * V + j] = -INFINITY;
            }
        }
        // Scores.
        float highest = -INFINITY, inv = 0.0f;
        if (!p.sigmoid || by_logit) {
#pragma unroll
            for (int m = 0; m < EPL; ++m) highest = fmaxf(highest, c[m]);
            highest = warp_max(highest);
        }
        const float top_logit = highest;
        if (!p.sigmoid) {
            float sum = 0.0f;
#pragma unroll
            for (int m = 0; m < EPL; ++m) {
                const float s = exp2_fast((c[m] - top_logit) * LOG2E);
                sum += s;
                if (!by_logit) c[m] = c[m] == -INFINITY ? -INFINITY : s;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(FULL_WARP, sum, o);
            inv = 1.0f / sum;
            if (!by_logit) {
#pragma unroll
                for (int m = 0; m < EPL; ++m) c[m] *= inv;
            }
        } else if (!by_logit) {
#pragma unroll
            for (int m = 0; m < EPL; ++m) c[m] = c[m] == -INFINITY ? -INFINITY : reciprocal_fast(1.0f + exp2_fast(c[m] * -LOG2E));
        }
        bool open = !p.sigmoid && !(inv <= 1.0001f && top_logit > -INFINITY); // NaN, infinities, nothing to choose
        float room = 3.0f;
        if (!by_logit) {
            if (KEEP_BIAS) {
#pragma unroll
                for (int m = 0; m < EPL; ++m) c[m] += kept_bias[KEEP_BIAS ? m : 0];
            } else if (p.bias != nullptr) {
#pragma unroll
                for (int m = 0; m < EPL; ++m) c[m] += expert(m) < n ? __ldg(p.bias + expert(m)) : 0.0f;
            }
            if (grouped && run > 0) {
                // Two highest of each load's V scores, then of the run's lanes.
                float score[EPL / V];
                unsigned taken = 0;
#pragma unroll
                for (int i = 0; i < EPL / V; ++i) {
                    float first = c[i * V], second = -INFINITY;
                    open |= first != first; // minima and maxima would drop a NaN
#pragma unroll
                    for (int j = 1; j < V; ++j) {
                        open |= c[i * V + j] != c[i * V + j];
                        second = fmaxf(second, fminf(first, c[i * V + j]));
                        first = fmaxf(first, c[i * V + j]);
                    }
                    for (int o = 1; o < run; o <<= 1) {
                        const float f = __shfl_xor_sync(FULL_WARP, first, o), s = __shfl_xor_sync(FULL_WARP, second, o);
                        second = fmaxf(fminf(first, f), fmaxf(second, s));
                        first = fmaxf(first, f);
                    }
                    score[i] = p.group_max || size == 1 ? first : first + second;
                    open |= !p.group_max && cancels(first, second);
                    if (expert(i * V) >= n) score[i] = -INFINITY;
                }
                // The best group top_groups times, and once more for the distance to the rest.
                float last = INFINITY;
                for (int k = 0; k <= p.top_groups; ++k) {
                    float best = -INFINITY;
#pragma unroll
                    for (int i = 0; i < EPL / V; ++i) best = fmaxf(best, (taken >> i) & 1 ? -INFINITY : score[i]);
                    best = warp_max(best);
                    if (k == p.top_groups) {
                        open |= !(last - best > 8e-6f + 5e-7f * EPL + 1e-6f * fabsf(last));
                        break;
                    }
                    int lanes = 0;
#pragma unroll
                    for (int i = 0; i < EPL / V; ++i) {
                        const bool hit = score[i] == best && !((taken >> i) & 1);
                        lanes += __popc(__ballot_sync(FULL_WARP, hit));
                        if (hit) taken |= 1u << i;
                    }
                    open |= lanes != run;
                    last = best;
                }
#pragma unroll
                for (int m = 0; m < EPL; ++m)
                    if (!((taken >> (m / V)) & 1)) c[m] = -INFINITY;
            } else if (grouped) {
                // Rows of a group's scores, `span` places apart so that the groups' lanes hit different banks;
                // each group's lanes take its two highest.
                float* mine = scores[warp];
#pragma unroll
                for (int m = 0; m < EPL; ++m)
                    if (expert(m) < n) mine[expert(m) + (group[m] << span_log2)] = c[m];
                __syncwarp();
                float first = -INFINITY, second = -INFINITY;
                if (my_group < p.n_groups)
                    for (int i = my_place; i < size; i += span) {
                        const float v = mine[my_group * (size + span) + i];
                        second = fmaxf(second, fminf(first, v));
                        first = fmaxf(first, v);
                        open |= v != v;
                    }
                __syncwarp();
                for (int o = span / 2; o > 0; o >>= 1) {
                    const float f = __shfl_xor_sync(FULL_WARP, first, o), s = __shfl_xor_sync(FULL_WARP, second, o);
                    second = fmaxf(fminf(first, f), fmaxf(second, s));
                    first = fmaxf(first, f);
                }
                const float score = p.group_max || size == 1 ? first : first + second;
                open |= !p.group_max && cancels(first, second);
                // Groups surely before this one, and groups that may be.
                const float slack = 8e-6f + 5e-7f * EPL + fabsf(score) * 1e-6f;
                int sure = 0, maybe = 0;
                for (int other = 0; other < p.n_groups; ++other) {
                    const float v = __shfl_sync(FULL_WARP, score, other << span_log2);
                    sure += v > score + slack;
                    maybe += other != my_group && !(v < score - slack);
                }
                const bool in = maybe < p.top_groups, real = my_group < p.n_groups;
                open |= real && !in && sure < p.top_groups;
                const unsigned kept = __ballot_sync(FULL_WARP, real && in);
#pragma unroll
                for (int m = 0; m < EPL; ++m)
                    if (!((kept >> (group[m] << span_log2)) & 1)) c[m] = -INFINITY;
            }
            highest = -INFINITY;
#pragma unroll
            for (int m = 0; m < EPL; ++m) highest = fmaxf(highest, c[m]);
            highest = warp_max(highest);
            room = 18.0f + EPL + fabsf(highest);
        }
        const float scale = by_logit ? 0.125f : 1.0f;
        if (by_logit) highest *= 0.125f;
        open |= !(fabsf(highest) < 1000.0f);
        if (__any_sync(FULL_WARP, open)) {
            route_row_exactly<T, EPL>(p, row);
            continue;
        }

        // One whole number per expert, sorted within the lane, highest first.
        const float offset = TOP - highest;
        uint32_t key[EPL];
#pragma unroll
        for (int m = 0; m < EPL; ++m) {
            const uint32_t bits = __float_as_uint(fmaxf(fmaf(c[m], scale, offset), LOWEST)) << 9;
            key[m] = (bits & ~INDEX_MASK) | (INDEX_MASK - expert(m));
        }
#pragma unroll
        for (int span = 2; span <= EPL; span *= 2)
#pragma unroll
            for (int step = span / 2; step > 0; step /= 2)
#pragma unroll
                for (int m = 0; m < EPL; ++m)
                    if ((m & step) == 0) {
                        const uint32_t a = key[m], b = key[m | step];
                        const bool down = (m & span) == 0 || span == EPL;
                        key[m] = down ? max(a, b) : min(a, b);
                        key[m | step] = down ? min(a, b) : max(a, b);
                    }
        auto next = [&] {
            const uint32_t best = __reduce_max_sync(FULL_WARP, key[0]);
            if (key[0] == best) {
#pragma unroll
                for (int m = 0; m + 1 < EPL; ++m) key[m] = key[m + 1];
                key[EPL - 1] = 0;
            }
            return best;
        };
        uint32_t chosen = 0; // lane j: the j-th choice
        for (int j = 0; j < p.top_k; ++j) {
            const uint32_t best = next();
            if (lane == j) chosen = best;
        }
        const int e = static_cast<int>(INDEX_MASK - (chosen & INDEX_MASK));
        const bool active = lane < p.top_k;
        const float logit = active && e < n ? to_float(x[e]) : 0.0f;
        const float bias = active && e < n && p.bias != nullptr ? __ldg(p.bias + e) : 0.0f;
        // Told apart from the choice before?
        constexpr int SHIFT = INDEX_BITS;
        constexpr float STEP = INDEX_BITS > 9 ? 2.0f : 1.0f; // in units of 2^-22
        const uint32_t before = __shfl_up_sync(FULL_WARP, chosen, 1);
        const float logit_before = __shfl_up_sync(FULL_WARP, logit, 1), bias_before = __shfl_up_sync(FULL_WARP, bias, 1);
        bool close = active && lane > 0 && static_cast<float>((before >> SHIFT) - (chosen >> SHIFT)) * STEP <= room &&
                     !(logit == logit_before && bias == bias_before);
        close |= active && ((chosen >> SHIFT) << (SHIFT - 9)) <= (1u << (INDEX_BITS - 9)); // the lowest step
        // And the last from the rest: on past its ties.
        const uint32_t last = __shfl_sync(FULL_WARP, chosen, p.top_k - 1);
        const float logit_last = __shfl_sync(FULL_WARP, logit, p.top_k - 1), bias_last = __shfl_sync(FULL_WARP, bias, p.top_k - 1);
        if (p.top_k < n)
            for (;;) {
                const uint32_t best = next();
                if (static_cast<float>((last >> SHIFT) - (best >> SHIFT)) * STEP > room) break;
                const int other = static_cast<int>(INDEX_MASK - (best & INDEX_MASK));
                if (best == 0 || other >= n) break;
                if (!(to_float(x[other]) == logit_last && (p.bias == nullptr || __ldg(p.bias + other) == bias_last))) {
                    close = true;
                    break;
                }
            }
        float s = 0.0f, total = 1.0f;
        if (active) s = p.sigmoid ? 1.0f / (1.0f + exp2_fast(logit * -LOG2E)) : exp2_fast((logit - top_logit) * LOG2E) * inv;
        if (p.renormalize) {
            total = s;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(FULL_WARP, total, o);
            close |= !(total >= LEAST_TOTAL);
        }
        if (__any_sync(FULL_WARP, close)) {
            route_row_exactly<T, EPL>(p, row);
            continue;
        }
        const float w = s / total * p.scale;
        if (active) {
            p.experts[row * p.top_k + lane] = e;
            p.weights[row * p.top_k + lane] = w;
        }
    }
}

// The same choice with L lanes per row, for batches large enough to fill the GPU with lanes.  A warp brings
// 32 / L rows into shared memory (rows an odd number of 16-byte pieces apart, so that the lanes' loads hit
// different banks); each lane walks its share of a row, no lane waiting for another.  Eight scores at a
// time become whole numbers as above, are sorted by a network of 19 exchanges and merged into the lane's
// eight best (a bitonic half-cleaner and its 12 exchanges), and so are the L lanes' lists at the end; the
// highest number that fell out is kept, as the ninth.  L is what keeps a warp's rows below 9 KB, and so about
// 24 warps on an SM.  Where the order is the logits' and those have 16 bits, the numbers hold them whole and
// nothing is left open.
//
// B200, top 8: 65536 x 256 float32 in 57 us with groups and bias (1.25 TB/s; a warp per row: 94; without the
// bound of 80 registers that lets 24 warps in, 63), 32 us by the logits alone; 32749 x 128 bfloat16 in 11 us (a
// warp per row: 17).  Bound by instructions (530 a row with groups).
constexpr int ROUTE_LIST = 8;
constexpr int ROUTE_LANES_EXPERTS = 256; // at most

__device__ __forceinline__ void exchange(uint32_t& a, uint32_t& b)
{
    const uint32_t high = max(a, b);
    b = min(a, b);
    a = high;
}

__device__ __forceinline__ void sort_down(uint32_t (&v)[ROUTE_LIST])
{
    exchange(v[0], v[1]); exchange(v[2], v[3]); exchange(v[4], v[5]); exchange(v[6], v[7]);
    exchange(v[0], v[2]); exchange(v[1], v[3]); exchange(v[4], v[6]); exchange(v[5], v[7]);
    exchange(v[1], v[2]); exchange(v[5], v[6]);
    exchange(v[0], v[4]); exchange(v[1], v[5]); exchange(v[2], v[6]); exchange(v[3], v[7]);
    exchange(v[2], v[4]); exchange(v[3], v[5]);
    exchange(v[1], v[2]); exchange(v[3], v[4]); exchange(v[5], v[6]);
}

// The eight highest of two falling lists, and the highest number that falls out.
__device__ __forceinline__ void merge_down(uint32_t (&best)[ROUTE_LIST], const uint32_t (&other)[ROUTE_LIST], uint32_t& fell)
{
#pragma unroll
    for (int i = 0; i < ROUTE_LIST; ++i) {
        fell = max(fell, min(best[i], other[ROUTE_LIST - 1 - i]));
        best[i] = max(best[i], other[ROUTE_LIST - 1 - i]);
    }
#pragma unroll
    for (int step = ROUTE_LIST / 2; step > 0; step /= 2)
#pragma unroll
        for (int i = 0; i < ROUTE_LIST; ++i)
            if ((i & step) == 0) exchange(best[i], best[i | step]);
}

// Bytes between two rows of the tile: an odd number of 16-byte pieces.
__host__ __device__ __forceinline__ int route_pitch(int row_bytes) { return (row_bytes / 16 | 1) * 16; }

template <typename T, int L, bool SIGMOID, bool BY_LOGIT, bool GROUPED>
__global__ void __launch_bounds__(32, 24) povs_route_lanes_kernel(const __grid_constant__ RouteParams p)
{
    constexpr bool WHOLE = BY_LOGIT && sizeof(T) == 2; // numbers that hold the logits whole
    constexpr int V = 16 / sizeof(T), INDEX_BITS = WHOLE ? 16 : 9;
    constexpr uint32_t INDEX_MASK = (1u << INDEX_BITS) - 1;
    constexpr float TOP = 3.9998f, LOWEST = 2.0f + 1.0f / (1 << 22);
    extern __shared__ __align__(16) uint8_t memory[];
    const int lane = threadIdx.x, n = p.n_experts, row_bytes = n * static_cast<int>(sizeof(T)), pitch = route_pitch(row_bytes);
    constexpr int ROWS = 32 / L;
    const int place = lane % ROWS, share = lane / ROWS; // this lane's row and which part of it
    const int64_t first_row = static_cast<int64_t>(blockIdx.x) * ROWS, row = first_row + place;
    const int rows = static_cast<int>(min(static_cast<int64_t>(ROWS), p.rows - first_row));
    const int from_e = n / L * share, to_e = from_e + n / L;
    float* bias = reinterpret_cast<float*>(memory + ROWS * pitch); // n, for !BY_LOGIT
    float* group_score = bias + n;                                 // n_groups * ROWS, twice, for GROUPED
    float* group_first = group_score + p.n_groups * ROWS;
    auto over_shares = [&](float v, bool highest) {
#pragma unroll
        for (int o = ROWS; o < 32; o *= 2) {
            const float other = __shfl_xor_sync(FULL_WARP, v, o);
            v = highest ? fmaxf(v, other) : v + other;
        }
        return v;
    };

    {
        const int pieces = row_bytes / 16;
        const uint8_t* from = static_cast<const uint8_t*>(p.logits) + first_row * p.row_stride * static_cast<int64_t>(sizeof(T));
        for (int r = 0, c = lane; r < rows;) {
            if (c < pieces) {
                const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(memory + r * pitch + c * 16));
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to),
                             "l"(from + r * p.row_stride * static_cast<int64_t>(sizeof(T)) + c * 16) : "memory");
                c += 32;
            }
            while (c >= pieces && r < rows) {
                c -= pieces;
                ++r;
            }
        }
        if (!BY_LOGIT)
            for (int e = lane; e < n; e += 32) bias[e] = p.bias != nullptr ? p.bias[e] : 0.0f;
        asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    const bool active = place < rows;
    const uint8_t* mine = memory + (active ? place : 0) * pitch;
    auto read = [&](int e, float (&x)[8]) {
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            T v[V];
            const uint4 raw = *reinterpret_cast<const uint4*>(mine + (e + i) * sizeof(T));
            memcpy(v, &raw, sizeof(raw));
#pragma unroll
            for (int j = 0; j < V; ++j) x[i + j] = to_float(v[j]);
        }
    };
    float x[8];
    float top = -INFINITY, inv = 0.0f;
    if (!SIGMOID || (BY_LOGIT && !WHOLE)) {
        for (int e = from_e; e < to_e; e += 8) {
            read(e, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, x[j]);
        }
        top = over_shares(top, true);
    }
    bool open = false;
    if (!SIGMOID) {
        float sums[2] = {0.0f, 0.0f};
        for (int e = from_e; e < to_e; e += 8) {
            read(e, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) sums[j & 1] += exp2_fast((x[j] - top) * LOG2E);
        }
        inv = reciprocal_fast(over_shares(sums[0] + sums[1], false));
        open = !(inv <= 1.0001f && top > -INFINITY); // NaN, infinities, nothing to choose
    }
    // A choice score; masked experts stay at -infinity.
    auto choice = [&](float logit, float b) {
        const float s = SIGMOID ? reciprocal_fast(1.0f + exp2_fast(logit * -LOG2E)) : exp2_fast((logit - top) * LOG2E) * inv;
        return logit == -INFINITY ? -INFINITY : s + b;
    };
    // The error that scores of 32 bits may have: as in the kernel above, with sums over n / 2 scores.
    const float sum_error = SIGMOID ? 0.0f : 3e-8f * static_cast<float>(n);
    float highest = BY_LOGIT ? top * 0.125f : -INFINITY;
    unsigned kept = 0xffffffffu;
    const int size = n / p.n_groups;
    if (!BY_LOGIT) {
        int g = p.n_groups / L * share, left = size;
        float first = -INFINITY, second = -INFINITY;
        for (int e = from_e; e < to_e; e += 8) {
            read(e, x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float c = choice(x[j], bias[e + j]);
                if (GROUPED) {
                    second = fmaxf(second, fminf(first, c));
                    open |= c != c;
                }
                first = fmaxf(first, c);
            }
            if (GROUPED && (left -= 8) == 0) {
                group_score[g * ROWS + place] = p.group_max ? first : first + second;
                open |= !p.group_max && cancels(first, second);
                group_first[g * ROWS + place] = first;
                first = second = -INFINITY;
                left = size;
                ++g;
            }
        }
        if (!GROUPED) highest = over_shares(first, true);
    }
    if (GROUPED) {
        kept = 0;
        highest = -INFINITY;
        __syncwarp();
        for (int g = p.n_groups / L * share; g < p.n_groups / L * (share + 1); ++g) {
            const float score = group_score[g * ROWS + place];
            const float slack = 8e-6f + 2.0f * sum_error + fabsf(score) * 1e-6f;
            int sure = 0, maybe = 0; // groups surely before this one, and groups that may be
            for (int other = 0; other < p.n_groups; ++other) {
                const float v = group_score[other * ROWS + place];
                sure += v > score + slack;
                maybe += other != g && !(v < score - slack);
            }
            if (maybe < p.top_groups) {
                kept |= 1u << g;
                highest = fmaxf(highest, group_first[g * ROWS + place]);
            } else {
                open |= sure < p.top_groups;
            }
        }
        highest = over_shares(highest, true);
    }
    const float room = BY_LOGIT ? 3.0f : 18.0f + fabsf(highest) + 8.4e6f * sum_error; // in steps of 2^-22
    if (!WHOLE) open |= !(fabsf(highest) < 1000.0f);

    uint32_t best[ROUTE_LIST], fell = 0;
#pragma unroll
    for (int i = 0; i < ROUTE_LIST; ++i) best[i] = 0;
    const float offset = TOP - highest;
    int g = p.n_groups / L * share, left = size;
    for (int e = from_e; e < to_e; e += 8) {
        uint32_t key[ROUTE_LIST];
        if constexpr (WHOLE) {
            const uint4 raw = *reinterpret_cast<const uint4*>(mine + e * sizeof(T));
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t high = j & 1 ? words[j / 2] & 0xffff0000u : words[j / 2] << 16; // the logit's bits, in order:
                const uint32_t ordered = high == 0x80000000u ? 0x80000000u : high ^ (static_cast<uint32_t>(static_cast<int32_t>(high) >> 31) | 0x80000000u);
                key[j] = (ordered & 0xffff0000u) | (INDEX_MASK - (e + j));
            }
        } else {
            read(e, x);
            const bool in = !GROUPED || (kept >> g & 1);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float c = BY_LOGIT ? x[j] * 0.125f : in ? choice(x[j], bias[e + j]) : -INFINITY;
                key[j] = __float_as_uint(fmaxf(c + offset, LOWEST)) << 9 | (INDEX_MASK - (e + j));
            }
            if (GROUPED && (left -= 8) == 0) {
                left = size;
                ++g;
            }
        }
        sort_down(key);
        merge_down(best, key, fell);
    }
#pragma unroll
    for (int o = ROWS; o < 32; o *= 2) {
        uint32_t other[ROUTE_LIST];
#pragma unroll
        for (int i = 0; i < ROUTE_LIST; ++i) other[i] = __shfl_xor_sync(FULL_WARP, best[i], o);
        fell = max(fell, __shfl_xor_sync(FULL_WARP, fell, o));
        merge_down(best, other, fell);
        open |= __shfl_xor_sync(FULL_WARP, static_cast<int>(open), o) != 0;
    }

    // The chosen, told apart from one another and from the rest.
    float score[ROUTE_LIST], total = 0.0f, logit_before = 0.0f, bias_before = 0.0f;
    int chosen[ROUTE_LIST];
#pragma unroll
    for (int j = 0; j < ROUTE_LIST; ++j) {
        score[j] = 0.0f;
        chosen[j] = 0;
        const uint32_t next = j + 1 < ROUTE_LIST ? best[j + 1] : fell;
        if (j < p.top_k) {
            const int e = min(static_cast<int>(INDEX_MASK - (best[j] & INDEX_MASK)), n - 1);
            const float logit = to_float(reinterpret_cast<const T*>(mine)[e]), b = BY_LOGIT ? 0.0f : bias[e];
            if (WHOLE) {
                open |= !(logit > -INFINITY);
            } else {
                open |= best[j] >> 9 <= 1;
                if (j > 0)
                    open |= static_cast<float>((best[j - 1] >> 9) - (best[j] >> 9)) <= room && !(logit == logit_before && b == bias_before);
                if (j == p.top_k - 1 && p.top_k < n) open |= static_cast<float>((best[j] >> 9) - (next >> 9)) <= room;
            }
            logit_before = logit;
            bias_before = b;
            score[j] = SIGMOID ? reciprocal_fast(1.0f + exp2_fast(logit * -LOG2E)) : exp2_fast((logit - top) * LOG2E) * inv;
            total += score[j];
            chosen[j] = e;
        }
    }
    open |= p.renormalize && !(total >= LEAST_TOTAL);
    const float part = p.renormalize ? 1.0f / total : 1.0f;
    if (active && !open && share == 0) {
        int32_t* experts = p.experts + row * p.top_k;
        float* weights = p.weights + row * p.top_k;
#pragma unroll
        for (int j = 0; j < ROUTE_LIST; ++j)
            if (j < p.top_k) {
                experts[j] = chosen[j];
                weights[j] = score[j] * part * p.scale;
            }
    }
    for (unsigned rest = __ballot_sync(FULL_WARP, active && open && share == 0); rest != 0; rest &= rest - 1)
        route_row_exactly<T, ROUTE_LANES_EXPERTS / 32>(p, first_row + __ffs(rest) - 1);
}

// Gradient of the weights with respect to the scores' logits, one warp per row.  With f_j the
// chosen scores, S their sum (1 without renormalisation) and g the weights' gradient:
//   df_j = scale (g_j - sum_i g_i f_i / S [renormalised]) / S
//   softmax: dx_i = s_i (df_i - sum_j f_j df_j);  sigmoid: dx_i = s_i (1 - s_i) df_i
// (df is 0 outside the chosen experts).  For a chosen expert, df_i - sum_j f_j df_j
//   = df_i (1 - sum_j f_j) + sum_j f_j (df_i - df_j), 1 - sum_j f_j the sum of the others,
// keeps its accuracy where the first form is a difference of near numbers.  The logits are read three or four times (once
// for renormalised weights, a sigmoid's chosen ones alone), all but the first from cache.  B200: 26 us with the forward
// pass for 32749 x 128 bfloat16, 72 for 65536 x 256 float32.
template <typename T>
__global__ void __launch_bounds__(128) povs_route_backward_kernel(const __grid_constant__ RouteParams p)
{
    const int lane = threadIdx.x & 31;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    T* dx = static_cast<T*>(p.grad_logits) + row * p.n_experts;
    const int n = p.n_experts;
    int e = -1;
    float g = 0.0f, v = 0.0f;
    if (lane < p.top_k) {
        e = p.chosen[row * p.top_k + lane];
        if (e < 0 || e >= n) e = -1;
        if (e >= 0) {
            g = p.grad_weights[row * p.top_k + lane];
            v = to_float(x[e]);
        }
    }
    auto warp_sum = [](float a) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(FULL_WARP, a, o);
        return a;
    };
    float top = -INFINITY, sum = 0.0f;
    bool no_scores = false; // a softmax's row with NaN or +infinity
    if (!p.sigmoid && p.renormalize) {
        for (int i = lane; i < n; i += 32) no_scores |= !(to_float(x[i]) < INFINITY);
        no_scores = __any_sync(FULL_WARP, no_scores);
    } else if (!p.sigmoid) {
        for (int i = lane; i < n; i += 32) top = fmaxf(top, to_float(x[i]));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL_WARP, top, o));
        if (top == -INFINITY) top = 0.0f;
        for (int i = lane; i < n; i += 32) sum += expf(to_float(x[i]) - top);
        sum = warp_sum(sum);
    }
    const float inv = 1.0f / sum;
    // Score f of a chosen expert; 1 - f of a sigmoid, from the logit too, as f may be rounded to 1.
    float f = 0.0f, complement = 1.0f;
    if (p.sigmoid) {
        const float t = expf(-fabsf(v)), r = 1.0f / (1.0f + t);
        complement = v > 0.0f ? t * r : r;
        f = e < 0 ? 0.0f : v > 0.0f ? r : t * r;
    } else if (!p.renormalize) {
        f = e < 0 ? 0.0f : expf(v - top) * inv;
    }
    // sum_j weight_j (g - g_j) with the weights' sum.  Gradients are taken relative to that of the highest weight, which
    // differs from the others by no more than top_k times such a sum: near gradients, or one weight near the sum, cost
    // no accuracy.
    auto apart = [&](float weight, float weights) {
        const unsigned most = __reduce_max_sync(FULL_WARP, __float_as_uint(weight));
        const float from = __shfl_sync(FULL_WARP, g, __ffs(__ballot_sync(FULL_WARP, __float_as_uint(weight) == most)) - 1);
        return fmaf(weights, g - from, -warp_sum(weight * (g - from)));
    };
    float mine, common = 0.0f;
    if (p.renormalize) {
        // Quotients of the scores over a common factor, the highest chosen one's, so that none is lost where 32 bits
        // flush the scores themselves to 0.  They do not depend on that factor: common is 0 exactly.
        float most = e < 0 ? -INFINITY : v;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(FULL_WARP, most, o));
        if (most == -INFINITY || (p.sigmoid && most > 0.0f)) most = 0.0f;
        const float part = e < 0 ? 0.0f : p.sigmoid && v > 0.0f ? f : expf(v - most) * complement;
        const float total = warp_sum(part);
        const float w = total == 0.0f ? 0.0f : part / total;
        mine = w * complement * apart(w, 1.0f);
        if (no_scores) mine = NAN;
    } else if (p.sigmoid) {
        mine = f * complement * g;
    } else {
        common = warp_sum(f * g);
        // Where the others make a quarter of the sum, g less the mean is not small beside both (34 us for a training
        // step of 32749 x 128 with the others' sum always, against 26).
        constexpr float MOST = 0.75f;
        float away = g - common;
        if (__reduce_add_sync(FULL_WARP, __float2uint_rn(f * 0x1p20f)) > static_cast<unsigned>(MOST * 0x1p20f)) {
            unsigned out = 0; // bit m: expert lane + 32 m is chosen
            for (int j = 0; j < p.top_k; ++j) {
                const int other = __shfl_sync(FULL_WARP, e, j);
                if (other >= 0 && (other & 31) == lane) out |= 1u << (other >> 5);
            }
            float rest = 0.0f; // the others' sum
            for (int i = lane; i < n; i += 32, out >>= 1) rest += out & 1 ? 0.0f : expf(to_float(x[i]) - top);
            away = fmaf(g, warp_sum(rest) * inv, apart(f, warp_sum(f)));
        }
        mine = f * away;
    }
    // The scale comes last: differences of the given numbers are exact where those are near.
    mine *= p.scale;
    common *= p.scale;
    for (int i = lane; i < n; i += 32) {
        const float xi = to_float(x[i]);
        dx[i] = from_float<T>(common == 0.0f || xi == -INFINITY ? 0.0f : -expf(xi - top) * inv * common);
    }
    __syncwarp();
    if (e >= 0) dx[e] = from_float<T>(mine);
}

// ------------------------------------------------------------------------------------------
// Plan: stable counting sort of the chosen experts.
// ------------------------------------------------------------------------------------------

struct PlanRowsParams {
    const void* experts; // n entries, int32 or int64
    int32_t id_bytes;
    int32_t n_experts;
    int64_t n;
    int64_t chunk;       // entries per block
    int32_t* counts;     // [blocks][n_experts], written by the counting kernel
    int32_t* slots;      // n
    int32_t* sources;    // n
    int32_t* offsets;    // n_experts + 1
};

constexpr int PLAN_MAX_EXPERTS = 4096;
constexpr int PLAN_THREADS = 512;
constexpr int PLAN_WARPS = PLAN_THREADS / 32;

// The entry's expert, or -1 for an entry that takes no slot.
__device__ __forceinline__ int plan_expert(const PlanRowsParams& p, int64_t i)
{
    const int64_t e = p.id_bytes == 4 ? static_cast<int64_t>(static_cast<const int32_t*>(p.experts)[i])
                                      : static_cast<const int64_t*>(p.experts)[i];
    return e >= 0 && e < p.n_experts ? static_cast<int>(e) : -1;
}

__global__ void __launch_bounds__(PLAN_THREADS) povs_plan_count_kernel(const __grid_constant__ PlanRowsParams p)
{
    extern __shared__ int32_t count[];
    for (int e = threadIdx.x; e < p.n_experts; e += PLAN_THREADS) count[e] = 0;
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.chunk;
    const int64_t last = min(first + p.chunk, p.n);
    for (int64_t i = first + threadIdx.x; i < last; i += PLAN_THREADS) {
        const int e = plan_expert(p, i);
        if (e >= 0) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < p.n_experts; e += PLAN_THREADS)
        p.counts[static_cast<int64_t>(blockIdx.x) * p.n_experts + e] = count[e];
}

// Every block places its own entries: a slot is the expert's offset, plus the entries of the
// blocks before, of the warps before and of the lanes before with the same expert.  Each warp takes
// a contiguous run of the block's chunk, so the order within an expert is the entries' order
// whatever the timing.  3 us for up to 4096 entries (one block, one launch); 12 us for 131072 entries and 256
// experts (64 blocks), most of it the latency of two launches and of reading the blocks' counts.  `warps` warps
// count (each holds a row of n_experts counters).
__global__ void __launch_bounds__(PLAN_THREADS) povs_plan_place_kernel(const __grid_constant__ PlanRowsParams p, int warps)
{
    extern __shared__ int32_t smem[];
    int32_t* base = smem;                  // [n_experts]: first slot of this block's entries
    int32_t* run = smem + p.n_experts;     // [warps][n_experts]
    __shared__ int32_t warp_total[PLAN_WARPS];
    __shared__ int32_t used;
    const int n_e = p.n_experts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int blocks = gridDim.x;

    for (int i = threadIdx.x; i < warps * n_e; i += PLAN_THREADS) run[i] = 0;
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.chunk;
    const int64_t last = min(first + p.chunk, p.n);
    const int64_t per = ((p.chunk + warps - 1) / warps + 31) / 32 * 32;
    const int64_t w_first = first + warp * per, w_last = min(w_first + per, last);
    if (warp < warps)
        for (int64_t i = w_first + lane; i < w_last; i += 32) {
            const int e = plan_expert(p, i);
            if (e >= 0) atomicAdd(&run[warp * n_e + e], 1);
        }
    __syncthreads();

    // Column sums: entries of the blocks before, and of all blocks.  A single block has its own.
    for (int e0 = 0; e0 < n_e; e0 += PLAN_THREADS) {
        const int e = e0 + threadIdx.x;
        int32_t before = 0, all = 0;
        if (e < n_e) {
            if (blocks == 1) {
                for (int w = 0; w < warps; ++w) all += run[w * n_e + e];
            } else {
#pragma unroll 8
                for (int b = 0; b < blocks; ++b) {
                    const int32_t c = p.counts[static_cast<int64_t>(b) * n_e + e];
                    all += c;
                    if (b < static_cast<int>(blockIdx.x)) before += c;
                }
            }
        }
        // Exclusive scan of `all` over the experts of this round.
        int32_t inc = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t up = __shfl_up_sync(FULL_WARP, inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 31) warp_total[warp] = inc;
        __syncthreads();
        int32_t start = e0 == 0 ? 0 : used;
        for (int w = 0; w < warp; ++w) start += warp_total[w];
        const int32_t offset = start + inc - all;
        if (e < n_e) {
            base[e] = offset + before;
            if (blockIdx.x == 0) {
                p.offsets[e] = offset;
                if (e == n_e - 1) p.offsets[n_e] = offset + all;
            }
        }
        __syncthreads();
        if (threadIdx.x == PLAN_THREADS - 1) used = start + inc;
        __syncthreads();
    }
    // Counters become the first slot of each warp's entries.
    for (int e = threadIdx.x; e < n_e; e += PLAN_THREADS) {
        int32_t at = base[e];
        for (int w = 0; w < warps; ++w) {
            const int32_t c = run[w * n_e + e];
            run[w * n_e + e] = at;
            at += c;
        }
    }
    __syncthreads();
    if (warp < warps)
        for (int64_t i0 = w_first; i0 < w_last; i0 += 32) {
            const int64_t i = i0 + lane;
            const int e = i < w_last ? plan_expert(p, i) : -1;
            const unsigned same = __match_any_sync(FULL_WARP, e);
            const int rank = __popc(same & ((1u << lane) - 1));
            int slot = -1;
            if (e >= 0) slot = run[warp * n_e + e] + rank;
            __syncwarp();
            if (e >= 0 && rank == 0) run[warp * n_e + e] += __popc(same);
            __syncwarp();
            if (i < w_last) {
                p.slots[i] = slot;
                if (slot >= 0) p.sources[slot] = static_cast<int32_t>(i);
            }
        }
    // Slots behind the last entry have no source.
    const int64_t stride = static_cast<int64_t>(blocks) * PLAN_THREADS;
    for (int64_t i = used + static_cast<int64_t>(blockIdx.x) * PLAN_THREADS + threadIdx.x; i < p.n; i += stride)
        p.sources[i] = -1;
}

// ------------------------------------------------------------------------------------------
// Dispatch: rows copied to their slots.
// ------------------------------------------------------------------------------------------

struct DispatchParams {
    const uint8_t* data; // row r at data + r * row_stride
    uint8_t* out;        // slot s at out + s * row_bytes
    const int32_t* slots; // rows * top_k
    const int32_t* used;  // slots in use: the rows of `out` behind them are zeroed
    int64_t rows;
    int64_t row_bytes;
    int64_t row_stride; // bytes
    int64_t n_slots;
    int32_t top_k;
    int32_t split_log2; // 2^split_log2 warps per row
};

constexpr int MOVE_WARPS = 8; // warps per block of the moving kernels

// A warp reads runs of 32 * UNROLL pieces of a row, all in flight, and writes each run to the row's
// slots: every row is read once.  Bound by DRAM writes (each row leaves top_k times): 203 us for 16384
// rows of 8 KB to 8 places each, 91 % of the copy rate; streaming stores gave 3 to 11 % on decks of 0.2 GB.
template <int BYTES, int UNROLL>
__global__ void __launch_bounds__(32 * MOVE_WARPS) povs_dispatch_kernel(const __grid_constant__ DispatchParams p)
{
    using V = typename Piece<BYTES>::type;
    constexpr int RUN = 32 * UNROLL;
    const int lane = threadIdx.x & 31;
    const int64_t pieces = p.row_bytes / BYTES;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * MOVE_WARPS;
    const int64_t me = static_cast<int64_t>(blockIdx.x) * MOVE_WARPS + (threadIdx.x >> 5);
    const int64_t step = static_cast<int64_t>(RUN) << p.split_log2;
    for (int64_t u = me; u < p.rows << p.split_log2; u += warps) {
        const int64_t row = u >> p.split_log2;
        const V* src = reinterpret_cast<const V*>(p.data + row * p.row_stride);
        const int32_t* slots = p.slots + row * p.top_k;
        const int first = lane < p.top_k ? slots[lane] : -1;
        for (int64_t c = (u & ((1 << p.split_log2) - 1)) * RUN + lane; c - lane < pieces; c += step) {
            V v[UNROLL];
#pragma unroll
            for (int i = 0; i < UNROLL; ++i)
                if (c + 32 * i < pieces) v[i] = __ldg(src + c + 32 * i);
            for (int j = 0; j < p.top_k; ++j) {
                const int slot = j < 32 ? __shfl_sync(FULL_WARP, first, j) : slots[j];
                if (slot < 0 || slot >= p.n_slots) continue;
                V* dst = reinterpret_cast<V*>(p.out + slot * p.row_bytes) + c;
                if (c - lane + RUN <= pieces) {
#pragma unroll
                    for (int i = 0; i < UNROLL; ++i) __stcs(dst + 32 * i, v[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < UNROLL; ++i)
                        if (c + 32 * i < pieces) __stcs(dst + 32 * i, v[i]);
                }
            }
        }
    }
    const int64_t used = max(0, *p.used);
    for (int64_t slot = used + me; slot < p.n_slots; slot += warps) {
        V* dst = reinterpret_cast<V*>(p.out + slot * p.row_bytes);
        for (int64_t c = lane; c < pieces; c += 32) dst[c] = V{};
    }
}

// ------------------------------------------------------------------------------------------
// Combine: weighted sums of each row's slots, and the gradients.
// ------------------------------------------------------------------------------------------

struct CombineParams {
    const void* data;      // slot s at data + s * data_stride elements
    const int32_t* slots;  // rows * top_k
    const float* weights;  // rows * top_k, or NULL for ones
    void* out;             // rows, contiguous
    int64_t rows;
    int64_t width;
    int64_t data_stride;   // elements
    int64_t n_slots;
    int32_t top_k;
    int32_t split_log2;    // 2^split_log2 warps per row
    // Backward only.
    const int32_t* used;
    const void* grad;      // rows, contiguous
    void* grad_data;       // n_slots rows, contiguous, or NULL
    float* grad_weights;   // rows * top_k, or NULL
};

// N elements as one load, and as floats.
template <typename T, int N> struct Pack {
    using Raw = typename Piece<N * sizeof(T)>::type;
    static __device__ __forceinline__ void unpack(const Raw& raw, float (&v)[N])
    {
        T e[N];
        memcpy(e, &raw, sizeof(raw));
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_float(e[i]);
    }
    static __device__ __forceinline__ Raw pack(const float (&v)[N])
    {
        T e[N];
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = from_float<T>(v[i]);
        Raw raw;
        memcpy(&raw, e, sizeof(raw));
        return raw;
    }
};

// A warp sums runs of 32 * UNROLL pieces of N elements: the pieces of AT_ONCE slots are in flight
// together, sums are taken in 32 bits in the order of the slots and rounded once.  Bound by DRAM reads:
// 184 us for 16384 rows of 8 KB from 8 slots each, the copy rate.
template <typename T, int N, int UNROLL, int AT_ONCE>
__global__ void __launch_bounds__(32 * MOVE_WARPS) povs_combine_kernel(const __grid_constant__ CombineParams p)
{
    using P = Pack<T, N>;
    using Raw = typename P::Raw;
    constexpr int RUN = 32 * UNROLL;
    const int lane = threadIdx.x & 31;
    const int64_t pieces = p.width / N;
    const int64_t warps = static_cast<int64_t>(gridDim.x) * MOVE_WARPS;
    const int64_t step = static_cast<int64_t>(RUN) << p.split_log2;
    for (int64_t u = static_cast<int64_t>(blockIdx.x) * MOVE_WARPS + (threadIdx.x >> 5); u < p.rows << p.split_log2; u += warps) {
        const int64_t row = u >> p.split_log2;
        for (int64_t c = (u & ((1 << p.split_log2) - 1)) * RUN + lane; c - lane < pieces; c += step) {
            const bool full = c - lane + RUN <= pieces;
            float sum[UNROLL][N];
#pragma unroll
            for (int i = 0; i < UNROLL; ++i)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[i][e] = 0.0f;
            for (int j0 = 0; j0 < p.top_k; j0 += 32) {
                int slot = -1;
                float weight = 0.0f; // of what is left out
                if (j0 + lane < p.top_k) {
                    slot = p.slots[row * p.top_k + j0 + lane];
                    if (slot < 0 || slot >= p.n_slots) slot = -1;
                    else weight = p.weights != nullptr ? p.weights[row * p.top_k + j0 + lane] : 1.0f;
                }
                const unsigned valid = __ballot_sync(FULL_WARP, slot >= 0);
                for (int j = 0; j < min(32, p.top_k - j0); j += AT_ONCE) {
                    Raw y[AT_ONCE][UNROLL];
                    constexpr unsigned EVERY = (1u << AT_ONCE) - 1;
                    const Raw* src[AT_ONCE];
#pragma unroll
                    for (int a = 0; a < AT_ONCE; ++a) {
                        const int at = __shfl_sync(FULL_WARP, slot, j + a); // -1 behind the last
                        src[a] = reinterpret_cast<const Raw*>(static_cast<const T*>(p.data) + max(at, 0) * p.data_stride) + c;
                    }
                    if (full && (valid >> j & EVERY) == EVERY) {
#pragma unroll
                        for (int a = 0; a < AT_ONCE; ++a)
#pragma unroll
                            for (int i = 0; i < UNROLL; ++i) y[a][i] = __ldg(src[a] + 32 * i);
                    } else {
#pragma unroll
                        for (int a = 0; a < AT_ONCE; ++a)
#pragma unroll
                            for (int i = 0; i < UNROLL; ++i) {
                                y[a][i] = Raw{};
                                if ((valid >> (j + a) & 1) && c + 32 * i < pieces) y[a][i] = __ldg(src[a] + 32 * i);
                            }
                    }
#pragma unroll
                    for (int a = 0; a < AT_ONCE; ++a) {
                        const float w = __shfl_sync(FULL_WARP, weight, j + a);
#pragma unroll
                        for (int i = 0; i < UNROLL; ++i) {
                            float v[N];
                            P::unpack(y[a][i], v);
#pragma unroll
                            for (int e = 0; e < N; ++e) sum[i][e] = fmaf(w, v[e], sum[i][e]);
                        }
                    }
                }
            }
            Raw* dst = reinterpret_cast<Raw*>(static_cast<T*>(p.out) + row * p.width) + c;
#pragma unroll
            for (int i = 0; i < UNROLL; ++i)
                if (c + 32 * i < pieces) dst[32 * i] = P::pack(sum[i]);
        }
    }
}

// 2^split_log2 warps of a block share a row: for AT_ONCE slots at a time, grad_data[slot] = w grad[row] and
// grad_weights = <data[slot], grad[row]> from one reading of each.  Afterwards the slots that no entry
// uses are zeroed in grad_data.  Bound by DRAM: 372 us for 16384 rows of 8 KB and 8 slots, 93 % of the copy
// rate.
template <typename T, int N, int UNROLL, int AT_ONCE>
__global__ void __launch_bounds__(32 * MOVE_WARPS) povs_combine_backward_kernel(const __grid_constant__ CombineParams p)
{
    using P = Pack<T, N>;
    using Raw = typename P::Raw;
    __shared__ float part[MOVE_WARPS][AT_ONCE];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int split = 1 << p.split_log2, mine = warp & (split - 1), rows_at_once = MOVE_WARPS >> p.split_log2;
    const int64_t pieces = p.width / N;
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * rows_at_once; base < p.rows;
         base += static_cast<int64_t>(gridDim.x) * rows_at_once) {
        const int64_t row = base + (warp >> p.split_log2);
        const bool there = row < p.rows;
        const Raw* g = reinterpret_cast<const Raw*>(static_cast<const T*>(p.grad) + row * p.width);
        for (int j0 = 0; j0 < p.top_k; j0 += AT_ONCE) {
            int at[AT_ONCE];
            float w[AT_ONCE], dot[AT_ONCE];
#pragma unroll
            for (int a = 0; a < AT_ONCE; ++a) {
                const bool is = there && j0 + a < p.top_k;
                at[a] = is ? p.slots[row * p.top_k + j0 + a] : -1;
                if (at[a] >= p.n_slots) at[a] = -1;
                w[a] = is && p.weights != nullptr ? p.weights[row * p.top_k + j0 + a] : 1.0f;
                dot[a] = 0.0f;
            }
            if (there)
                for (int64_t c = mine * 32 * UNROLL + lane; c < pieces; c += 32 * UNROLL * split) {
                    Raw up[UNROLL], y[AT_ONCE][UNROLL];
#pragma unroll
                    for (int i = 0; i < UNROLL; ++i) {
                        up[i] = Raw{};
                        if (c + 32 * i < pieces) up[i] = __ldg(g + c + 32 * i);
                    }
                    if (p.grad_weights != nullptr) {
#pragma unroll
                        for (int a = 0; a < AT_ONCE; ++a) {
                            const Raw* src = reinterpret_cast<const Raw*>(static_cast<const T*>(p.data) + max(at[a], 0) * p.data_stride);
#pragma unroll
                            for (int i = 0; i < UNROLL; ++i) {
                                y[a][i] = Raw{};
                                if (at[a] >= 0 && c + 32 * i < pieces) y[a][i] = __ldg(src + c + 32 * i);
                            }
                        }
                    }
#pragma unroll
                    for (int i = 0; i < UNROLL; ++i) {
                        float d[N], v[N];
                        P::unpack(up[i], d);
#pragma unroll
                        for (int a = 0; a < AT_ONCE; ++a) {
                            if (p.grad_weights != nullptr) {
                                P::unpack(y[a][i], v);
                                if (at[a] >= 0) {
#pragma unroll
                                    for (int e = 0; e < N; ++e) dot[a] = fmaf(d[e], v[e], dot[a]);
                                }
                            }
                            if (p.grad_data != nullptr && at[a] >= 0 && c + 32 * i < pieces) {
#pragma unroll
                                for (int e = 0; e < N; ++e) v[e] = w[a] * d[e];
                                __stcs(reinterpret_cast<Raw*>(static_cast<T*>(p.grad_data) + at[a] * p.width) + c + 32 * i, P::pack(v));
                            }
                        }
                    }
                }
            if (p.grad_weights != nullptr) {
#pragma unroll
                for (int a = 0; a < AT_ONCE; ++a) {
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) dot[a] += __shfl_xor_sync(FULL_WARP, dot[a], o);
                    if (lane == 0) part[warp][a] = dot[a];
                }
                if (split > 1) __syncthreads();
                else __syncwarp();
                if (mine == 0 && lane < AT_ONCE && there && j0 + lane < p.top_k) {
                    float total = 0.0f;
                    for (int i = 0; i < split; ++i) total += part[warp + i][lane];
                    p.grad_weights[row * p.top_k + j0 + lane] = total;
                }
                if (split > 1) __syncthreads();
                else __syncwarp();
            }
        }
    }
    if (p.grad_data == nullptr) return;
    const int64_t used = max(0, *p.used);
    for (int64_t slot = used + static_cast<int64_t>(blockIdx.x) * MOVE_WARPS + warp; slot < p.n_slots;
         slot += static_cast<int64_t>(gridDim.x) * MOVE_WARPS) {
        Raw* dst = reinterpret_cast<Raw*>(static_cast<T*>(p.grad_data) + slot * p.width);
        for (int64_t c = lane; c < pieces; c += 32) dst[c] = Raw{};
    }
}

} // namespace povs
