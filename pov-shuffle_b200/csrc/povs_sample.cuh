// Drawing one id per row from scores, with temperature, top-k, top-p and min-p, from given random
// numbers.
#pragma once

#include <cstdint>

#include "povs_rows.cuh"

namespace povs {

struct SampleParams {
    const void* logits; // row r, id i at logits[r * row_stride + i]
    int64_t rows;
    int64_t width;
    int64_t row_stride; // elements
    const void* uniforms;
    int32_t uniform_bytes; // 4 or 8
    int32_t weight_bits;   // a weight of 1 is 2^weight_bits; the row's sum stays below 2^63
    // One value per row, or NULL for the value beside it.
    const float* temperatures;
    const int32_t* top_ks;
    const float* top_ps;
    const float* min_ps;
    double temperature;
    double top_p;
    double min_p;
    int64_t top_k;
    int64_t* ids;
};

// Order of scores as an unsigned number: 0 for what is never drawn (NaN, -infinity), then the
// numbers from the lowest up (+0 and -0 are the same number).
__device__ __forceinline__ uint32_t score_key(float v)
{
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b >> 31) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }

// Weight of a score: exp((v - top) / temperature) as a whole number of 2^-weight_bits.  Whole
// numbers add up the same in every order, so the running sums that decide the id do not depend on
// how the row is split.
__device__ __forceinline__ double score_weight(float v, float top, double inv_temperature)
{
    return v == top ? 1.0 : exp((static_cast<double>(v) - static_cast<double>(top)) * inv_temperature);
}

constexpr int SAMPLE_THREADS = 1024;

template <typename U> __device__ __forceinline__ U warp_inclusive(U v, int lane)
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const U up = __shfl_up_sync(FULL_WARP, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// One block per row.
template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS) povs_sample_kernel(const __grid_constant__ SampleParams p)
{
    __shared__ unsigned long long bins[256];
    __shared__ unsigned long long warp_part[32];
    __shared__ uint32_t shared_key;
    __shared__ unsigned long long shared_left;
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.logits) + row * p.row_stride;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const double temperature = p.temperatures != nullptr ? p.temperatures[row] : p.temperature;
    const double top_p = p.top_ps != nullptr ? p.top_ps[row] : p.top_p;
    const double min_p = p.min_ps != nullptr ? p.min_ps[row] : p.min_p;
    const int64_t top_k = p.top_ks != nullptr ? p.top_ks[row] : p.top_k;

    // Highest key, and the lowest index that has it.
    unsigned long long best = 0;
    for (int64_t i = t; i < p.width; i += SAMPLE_THREADS) {
        const unsigned long long k = score_key(to_float(x[i]));
        best = max(best, (k << 32) | (0xffffffffu - static_cast<uint32_t>(i)));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(FULL_WARP, best, o));
    if (lane == 0) warp_part[warp] = best;
    __syncthreads();
    best = warp_part[lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(FULL_WARP, best, o));
    const uint32_t top_key = static_cast<uint32_t>(best >> 32);
    if (top_key == 0 || !(temperature > 0.0)) {
        if (t == 0) p.ids[row] = top_key == 0 ? -1 : static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(best));
        return;
    }
    const float top = key_score(top_key);
    const double inv_temperature = 1.0 / temperature;
    const double unit = static_cast<double>(1ull << p.weight_bits);

    // Kept are the keys above `cut` and, in index order, the first `ties` of those equal to it.
    uint32_t cut = 0;
    unsigned long long ties = 0;

    // The key at which a running sum from the highest key down first reaches `want`: counts of ids
    // (by_mass false) or their weights (by_mass true), over the ids kept so far.  Returns what is
    // left of `want` at that key in shared_left, and the key in shared_key.
    auto search = [&](bool by_mass, double want) {
        uint32_t prefix = 0;
        double left = want;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int b = t; b < 256; b += SAMPLE_THREADS) bins[b] = 0;
            __syncthreads();
            for (int64_t i = t; i < p.width; i += SAMPLE_THREADS) {
                const float v = to_float(x[i]);
                const uint32_t k = score_key(v);
                if (k == 0 || k < cut || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
                // Ties at the cut are put in afterwards, by their number.
                if (by_mass && cut != 0 && k == cut) continue;
                const unsigned long long add =
                    by_mass ? static_cast<unsigned long long>(llrint(score_weight(v, top, inv_temperature) * unit)) : 1ull;
                atomicAdd(&bins[(k >> shift) & 255u], add);
            }
            __syncthreads();
            if (t == 0) {
                if (by_mass && cut != 0 && (shift == 24 || (cut >> (shift + 8)) == prefix))
                    bins[(cut >> shift) & 255u] +=
                        ties * static_cast<unsigned long long>(llrint(score_weight(key_score(cut), top, inv_temperature) * unit));
                int b = 255;
                while (b > 0 && static_cast<double>(bins[b]) < left) left -= static_cast<double>(bins[b--]);
                shared_key = (prefix << 8) | static_cast<uint32_t>(b);
                shared_left = static_cast<unsigned long long>(__double_as_longlong(left));
            }
            __syncthreads();
            prefix = shared_key;
            left = __longlong_as_double(static_cast<long long>(shared_left));
            __syncthreads();
        }
        return left;
    };
    auto block_sum = [&](unsigned long long v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_WARP, v, o);
        __syncthreads();
        if (lane == 0) warp_part[warp] = v;
        __syncthreads();
        v = warp_part[lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_WARP, v, o);
        __syncthreads();
        return v;
    };

    if (top_k > 0) {
        unsigned long long valid = 0;
        for (int64_t i = t; i < p.width; i += SAMPLE_THREADS) valid += score_key(to_float(x[i])) != 0;
        valid = block_sum(valid);
        if (static_cast<unsigned long long>(top_k) < valid) {
            const double left = search(false, static_cast<double>(top_k));
            cut = shared_key;
            ties = static_cast<unsigned long long>(left);
        }
    }
    if (top_p < 1.0) {
        unsigned long long mass = 0;
        for (int64_t i = t; i < p.width; i += SAMPLE_THREADS) {
            const float v = to_float(x[i]);
            const uint32_t k = score_key(v);
            if (k > cut) mass += static_cast<unsigned long long>(llrint(score_weight(v, top, inv_temperature) * unit));
        }
        mass = block_sum(mass);
        if (cut != 0)
            mass += ties * static_cast<unsigned long long>(llrint(score_weight(key_score(cut), top, inv_temperature) * unit));
        // The first id is always kept (half a unit is below every weight that is not 0).
        const double want = fmax(0.5, top_p * static_cast<double>(mass));
        const double left = search(true, want);
        const uint32_t key = shared_key;
        if (key != 0 && key >= cut) { // 0: rounding put `want` above the whole sum, everything stays
            // Ids with this key are kept while the sum before them is below `want`.
            const double w = rint(score_weight(key_score(key), top, inv_temperature) * unit);
            double count = fmin(ceil(left / w), static_cast<double>(p.width));
            if (key == cut) count = fmin(count, static_cast<double>(ties));
            cut = key;
            ties = static_cast<unsigned long long>(count);
        }
    }

    // The draw, in index order: thread t holds ids [t * per, (t + 1) * per).
    const int64_t per = (p.width + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
    const int64_t first = t * per, last = min(first + per, p.width);
    auto block_exclusive = [&](unsigned long long v, unsigned long long& total) {
        const unsigned long long inc = warp_inclusive(v, lane);
        __syncthreads();
        if (lane == 31) warp_part[warp] = inc;
        __syncthreads();
        const unsigned long long others = warp_inclusive(warp_part[lane], lane);
        const unsigned long long before = warp > 0 ? __shfl_sync(FULL_WARP, others, warp - 1) : 0;
        total = __shfl_sync(FULL_WARP, others, 31);
        return before + inc - v;
    };
    unsigned long long my_ties = 0, all_ties = 0;
    if (cut != 0)
        for (int64_t i = first; i < last; ++i) my_ties += score_key(to_float(x[i])) == cut;
    const unsigned long long ties_before = block_exclusive(my_ties, all_ties);
    // Weight of id i, given the ties before it.
    auto kept_weight = [&](int64_t i, unsigned long long& seen) -> unsigned long long {
        const float v = to_float(x[i]);
        const uint32_t k = score_key(v);
        if (k == 0 || k < cut) return 0;
        if (cut != 0 && k == cut && seen++ >= ties) return 0;
        const double w = score_weight(v, top, inv_temperature);
        return w >= min_p || k == top_key ? static_cast<unsigned long long>(llrint(w * unit)) : 0;
    };
    unsigned long long mine = 0, total = 0, seen = ties_before;
    for (int64_t i = first; i < last; ++i) mine += kept_weight(i, seen);
    const unsigned long long before = block_exclusive(mine, total);
    double u = p.uniform_bytes == 4 ? static_cast<const float*>(p.uniforms)[row]
                                    : static_cast<const double*>(p.uniforms)[row];
    u = u > 0.0 ? u : 0.0;
    const double target = u * static_cast<double>(total);
    const unsigned long long want = target < static_cast<double>(total) ? static_cast<unsigned long long>(target) : total - 1;
    if (mine != 0 && before <= want && want < before + mine) {
        unsigned long long sum = before;
        seen = ties_before;
        for (int64_t i = first; i < last; ++i) {
            sum += kept_weight(i, seen);
            if (sum > want) {
                p.ids[row] = i;
                break;
            }
        }
    }
}

} // namespace povs
