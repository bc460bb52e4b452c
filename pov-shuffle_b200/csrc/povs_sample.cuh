// Drawing one id per row from scores, with temperature, top-k, top-p and min-p, from given random
// numbers.
//
// A row is read once.  While it streams by, a cluster of 1 to 8 blocks keeps the highest score, the
// sum of the weights w = exp((x - reference) / temperature), and a list of every score at or above a
// threshold that a probe of the row's scores put near the last rank that can matter.  The filters and the
// draw then work on the list alone, in shared memory.  Only a row whose list turns out too short or too
// long (a nucleus of thousands of ids, top_k in the thousands, rows of equal scores) is read again, to
// find the border by bins of the score's distance from the highest.
#pragma once

#include <cooperative_groups.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "povs_rows.cuh"

namespace povs {

namespace cg = cooperative_groups;

struct SampleParams {
    const void* logits; // row r, id i at logits[r * row_stride + i]
    int64_t rows;
    int64_t width;
    int64_t row_stride; // elements
    const void* uniforms;
    int32_t uniform_bytes; // 4 or 8
    int32_t weight_bits;   // in sums of whole numbers a weight of 1 is 2^weight_bits; a row's sum stays below 2^63
    int32_t cluster;       // blocks per row
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
    double taylor[5]; // (ln 2)^i / i!, i = 1 .. 5: in constant memory, where an operand costs no register
};

constexpr int SAMPLE_THREADS = 256;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int SAMPLE_MAX_CLUSTER = 8;
constexpr int SAMPLE_LIST = 2048;   // listed scores per block, and per row
constexpr int SAMPLE_TARGET = 1024; // listed scores aimed at where no top_k says how many
constexpr int SAMPLE_PROBE = 4096;  // scores probed
constexpr int SAMPLE_BINS = 1024;

// Order of scores as an unsigned number: 0 for what is never drawn (NaN, -infinity), then the
// numbers from the lowest up (+0 and -0 are the same number).
__device__ __forceinline__ uint32_t score_key(float v)
{
    if (!(v > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b >> 31) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }

constexpr uint32_t LOWEST_KEY = 0x00800000u; // the lowest finite score's

// A highest score below this, or +infinity, leaves weights to the scores equal to it alone: float's
// next lower score is 2^104 away, which the highest temperature that counts (1e28) makes 2000.
constexpr float LONE = -3.0e38f;

// Weights of many scores, for loops that a whole warp runs together: exp((v - reference) * inv) up to
// a factor common to all, to 2^-48 relative.  With z = v * inv / ln 2 = n / 32 + r, |r| <= 1/64, and n0
// the n of the reference, the weight is 2^((n - n0) >> 5) * 2^(((n - n0) & 31) / 32) * 2^r: the second
// factor sits in the lanes' registers (one shuffle in place of a table in memory, whose banks would
// clash), and 2^r is its Taylor polynomial of degree 5 (the next term is (r ln 2)^6 / 720 < 2.3e-15).
// The products with inv / ln 2 are exact in both fused operations, so large scores lose nothing.
// Ten operations in 64 bits a score: at half the rate of 32 bits about what its 4 bytes cost to read.
// Scores 500 or more below the reference in z, NaN and -infinity weigh 2^-500 to 2^-1000: nothing beside
// the highest score's.  References stay above LONE, where the float 500 below exists.
struct WarpExp {
    double step;   // 2^(lane / 32)
    double scale;  // inv / ln 2, or so much that one of float's steps at the reference makes 250
    double magic;  // rounds to steps of 1/32, less n0
    double factor; // times this, a weight is relative to the reference
    float floor;
    __device__ WarpExp(int lane) : step(exp2(lane * 0.03125)), scale(0.0), magic(0.0), factor(0.0), floor(-INFINITY) {}
    __device__ __forceinline__ void refer(float reference, double inv)
    {
        constexpr double MAGIC = 6755399441055744.0 / 32; // 1.5 * 2^52 steps of 1/32
        const double here = static_cast<double>(reference);
        const double spacing = fmax(fabs(here) * 5.9604644775390625e-8, 1.401298464324817e-45);
        scale = fmin(inv * 1.4426950408889634074, 250.0 / spacing);
        const double n0 = rint(here * scale * 32.0);
        magic = MAGIC - n0 * 0.03125;
        factor = exp2(fma(-here, scale, n0 * 0.03125));
        floor = __double2float_rd(here - 500.0 / scale);
    }
    __device__ __forceinline__ double operator()(float v, const double* __restrict__ taylor) const
    {
        const double x = static_cast<double>(fmaxf(v, floor));
        const double t = fma(x, scale, magic);
        const double r = fma(x, scale, magic - t);
        const int n = __double2loint(t);
        double q = fma(r, taylor[4], taylor[3]);
        q = fma(r, q, taylor[2]);
        q = fma(r, q, taylor[1]);
        q = fma(r, q, taylor[0]);
        const double at = __shfl_sync(FULL_WARP, step, n & 31);
        const double base = __hiloint2double(__double2hiint(at) + (n & ~31) * (1 << 15), __double2loint(at));
        return fma(base * r, q, base);
    }
};

// The same weight for single scores.
__device__ __forceinline__ double score_weight(float v, float top, double inv_temperature)
{
    return v == top ? 1.0 : exp((static_cast<double>(v) - static_cast<double>(top)) * inv_temperature);
}

template <typename T> __device__ __forceinline__ T warp_sum(T v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_WARP, v, o);
    return v;
}

template <typename U> __device__ __forceinline__ U warp_inclusive(U v, int lane)
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const U up = __shfl_up_sync(FULL_WARP, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// A row's scores in groups of 16 bytes.  Group g holds the ids g * N - lead + j, j < N, where `lead` puts
// every group on a 16-byte boundary; places outside the row read as -infinity.
template <typename T> struct RowGroups {
    static constexpr int N = 16 / sizeof(T);
    const T* x;
    int64_t width;
    int lead;
    int groups;
    __device__ RowGroups(const T* x_, int64_t width_) : x(x_), width(width_)
    {
        lead = static_cast<int>((reinterpret_cast<uint64_t>(x) / sizeof(T)) % N);
        groups = static_cast<int>((width + lead + N - 1) / N);
    }
    __device__ __forceinline__ int64_t id(int g) const { return static_cast<int64_t>(g) * N - lead; }
    __device__ __forceinline__ void load(int g, float (&v)[N]) const
    {
        const int64_t i = id(g);
        if (i >= 0 && i + N <= width) {
            union {
                uint4 raw;
                T e[N];
            } u;
            u.raw = __ldg(reinterpret_cast<const uint4*>(x + i));
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = to_float(u.e[j]);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = i + j >= 0 && i + j < width ? to_float(x[i + j]) : -INFINITY;
        }
    }
};

struct SampleShared {
    unsigned long long list[SAMPLE_LIST]; // key << 32 | ~id: descending order is by score, then by lowest id
    double weight[SAMPLE_LIST];
    unsigned long long bins[SAMPLE_BINS];
    unsigned int counts[SAMPLE_BINS];
    // Read by the other blocks of the cluster.
    unsigned long long best[SAMPLE_WARPS]; // highest key << 32 | ~lowest id that has it
    double mass[SAMPLE_WARPS];             // of each warp's ids, which follow one another
    float reference[SAMPLE_WARPS];
    unsigned int ties[SAMPLE_WARPS];
    unsigned long long exchange[2];
    unsigned int listed;
    int outcome;
    uint32_t cut;
    unsigned long long cut_ties;
    // This block's own.
    unsigned long long part[SAMPLE_WARPS];
    double part_mass[SAMPLE_WARPS];
    double listed_mass;
    unsigned int probe_counts[16];
    uint32_t probe_low;
    uint32_t lowest;
    int few;
    int few_at[32];
    unsigned long long found;
    unsigned long long left;
};

// Grid: rows * cluster blocks, `cluster` neighbours per row.
template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS, 4) povs_sample_kernel(const __grid_constant__ SampleParams p)
{
    constexpr int N = RowGroups<T>::N;
    constexpr int UNROLL = 4;
    __shared__ SampleShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int blocks = p.cluster, rank = blockIdx.x % blocks;
    const int64_t row = blockIdx.x / blocks;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const RowGroups<T> x(static_cast<const T*>(p.logits) + row * p.row_stride, p.width);

    const double temperature = p.temperatures != nullptr ? p.temperatures[row] : p.temperature;
    const double top_p = p.top_ps != nullptr ? p.top_ps[row] : p.top_p;
    const double min_p = p.min_ps != nullptr ? p.min_ps[row] : p.min_p;
    const int64_t top_k_given = p.top_ks != nullptr ? p.top_ks[row] : p.top_k;
    const int64_t top_k = top_k_given > 0 && top_k_given < p.width ? top_k_given : 0;
    const bool greedy = !(temperature > 0.0);
    const double inv = fmin(fmax(1.0 / temperature, 1e-28), 1e36); // so that 0 * inv stays 0
    const bool nucleus = top_p < 1.0, floor_p = min_p > 0.0;
    const bool filtered = !greedy && (nucleus || floor_p || top_k > 0);
    // The sum of all weights: without a filter, or for a nucleus of the whole row.
    const bool need_mass = !greedy && top_k == 0 && (nucleus || !floor_p);

    // This block's groups, and within them each warp's, in id order.
    const int per_block = (x.groups + blocks - 1) / blocks;
    const int first_group = min(rank * per_block, x.groups), last_group = min(first_group + per_block, x.groups);
    const int per_warp = (per_block + SAMPLE_WARPS - 1) / SAMPLE_WARPS;
    const int warp_first = min(first_group + warp * per_warp, last_group), warp_last = min(warp_first + per_warp, last_group);

    auto everyone = [&] {
        if (blocks > 1) cluster.sync();
        else __syncthreads();
    };
    auto block_at = [&](int r) -> SampleShared& { return blocks > 1 ? *cluster.map_shared_rank(&sh, r) : sh; };

    if (t == 0) sh.listed = 0;
    if (t < 16) sh.probe_counts[t] = 0;
    if (t == 0) sh.probe_low = 0xffffffffu;
    __syncthreads();

    // The probe: scores spread evenly over the row.  Its rank that corresponds to the ids wanted,
    // with four standard deviations to spare where top_k must be met, gives the list's threshold (its
    // upper 16 bits, found bit by bit).  Every block of the row finds the same one.
    uint32_t threshold = LOWEST_KEY;
    bool listing = filtered;
    if (filtered && p.width > SAMPLE_LIST) {
        constexpr int PER = SAMPLE_PROBE / SAMPLE_THREADS;
        uint32_t k[PER];
        uint32_t low = 0xffffffffu;
#pragma unroll
        for (int m = 0; m < PER / N; ++m) {
            float v[N];
            x.load(static_cast<int>(static_cast<int64_t>(m * SAMPLE_THREADS + t) * x.groups / (SAMPLE_PROBE / N)), v);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                k[m * N + j] = score_key(v[j]);
                if (k[m * N + j] != 0) low = min(low, k[m * N + j]);
            }
        }
        low = __reduce_min_sync(FULL_WARP, low);
        if (lane == 0) atomicMin(&sh.probe_low, low);
        const double share = static_cast<double>(SAMPLE_PROBE) / static_cast<double>(p.width);
        const double room = 0.8 * SAMPLE_LIST * share;
        double want = SAMPLE_TARGET * share;
        if (top_k > 0) {
            want = static_cast<double>(top_k) * share;
            if (want > room) listing = false;
            want = fmin(want + 4.0 * sqrt(want) + 6.0, room);
        }
        const unsigned int rank_wanted = static_cast<unsigned int>(fmax(want, 1.0));
        uint32_t found = 0;
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t candidate = found | (1u << bit);
            unsigned int c = 0;
#pragma unroll
            for (int m = 0; m < PER; ++m) c += k[m] >= candidate;
            c = __reduce_add_sync(FULL_WARP, c);
            if (lane == 0) atomicAdd(&sh.probe_counts[bit - 16], c);
            __syncthreads();
            if (sh.probe_counts[bit - 16] >= rank_wanted) found = candidate;
        }
        threshold = max(found, LOWEST_KEY);
    }
    const float list_from = listing ? key_score(threshold) : INFINITY; // +infinity: see `lone` below

    // The stream.
    WarpExp weight_of(lane);
    {
        float top = -INFINITY, reference = -INFINITY, limit = -INFINITY;
        int top_group = 0;
        double sum = 0.0;
        for (int g0 = warp_first; g0 < warp_last; g0 += 32 * UNROLL) {
            float v[UNROLL][N];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int g = g0 + 32 * u + lane;
                if (g < warp_last) {
                    x.load(g, v[u]);
                } else {
#pragma unroll
                    for (int j = 0; j < N; ++j) v[u][j] = -INFINITY;
                }
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int g = g0 + 32 * u + lane;
                float most = -INFINITY;
#pragma unroll
                for (int j = 0; j < N; ++j) most = fmaxf(most, v[u][j]);
                if (most > top) {
                    top = most;
                    top_group = g;
                }
                if (most >= list_from) {
                    const uint32_t id = static_cast<uint32_t>(x.id(g));
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        if (v[u][j] >= list_from) {
                            const unsigned int at = atomicAdd(&sh.listed, 1u);
                            if (at < SAMPLE_LIST)
                                sh.list[at] = (static_cast<unsigned long long>(score_key(v[u][j])) << 32) | (~(id + j));
                        }
                }
                if (need_mass) {
                    // The reference is the first scores' highest, renewed only when a weight would pass e^64.
                    if (__any_sync(FULL_WARP, most > limit)) {
                        float higher = most;
#pragma unroll
                        for (int o = 16; o > 0; o >>= 1) higher = fmaxf(higher, __shfl_xor_sync(FULL_WARP, higher, o));
                        const double old_factor = weight_of.factor;
                        weight_of.refer(higher, inv);
                        sum = reference > LONE ? sum * old_factor * score_weight(reference, higher, inv) / weight_of.factor : 0.0;
                        reference = higher;
                        limit = static_cast<float>(static_cast<double>(reference) + 64.0 / inv);
                    }
#pragma unroll
                    for (int j = 0; j < N; ++j) sum += weight_of(v[u][j], p.taylor);
                }
            }
        }
        // The warp's highest score and the lowest id that has it.
        unsigned long long best = 0;
        if (top > -INFINITY) {
            float v[N];
            x.load(top_group, v);
#pragma unroll
            for (int j = N - 1; j >= 0; --j)
                if (v[j] == top)
                    best = (static_cast<unsigned long long>(score_key(top)) << 32) | ~static_cast<uint32_t>(x.id(top_group) + j);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(FULL_WARP, best, o));
        sum = warp_sum(sum);
        if (lane == 0) {
            sh.best[warp] = best;
            sh.mass[warp] = reference > LONE ? sum * weight_of.factor : 0.0;
            sh.reference[warp] = reference;
        }
    }
    everyone();

    // Every warp of every block works out the row's totals for itself: lane l takes the warps 2 l and
    // 2 l + 1 of the cluster, which follow one another in id order.
    const int parts = blocks * SAMPLE_WARPS;
    unsigned long long best = 0;
    unsigned int listed = 0;
    for (int e = lane; e < parts; e += 32) best = max(best, block_at(e / SAMPLE_WARPS).best[e % SAMPLE_WARPS]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(FULL_WARP, best, o));
    const uint32_t top_key = static_cast<uint32_t>(best >> 32);
    const float top = key_score(top_key);
    if (top_key == 0 || greedy) {
        if (rank == 0 && t == 0) p.ids[row] = top_key == 0 ? -1 : static_cast<int64_t>(~static_cast<uint32_t>(best));
        everyone();
        return;
    }
    const bool lone = top == INFINITY || top < LONE; // no list, no sums
    double part_mass[2] = {0.0, 0.0};
    unsigned long long part_ties[2] = {0, 0};
    double total = 0.0; // sum of all weights, relative to the highest score
    if (need_mass && !lone) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = 2 * lane + h;
            if (e < parts) {
                SampleShared& from = block_at(e / SAMPLE_WARPS);
                const double m = from.mass[e % SAMPLE_WARPS];
                if (m > 0.0) part_mass[h] = m / score_weight(top, from.reference[e % SAMPLE_WARPS], inv);
            }
        }
        total = warp_sum(part_mass[0] + part_mass[1]);
    }
    for (int r = 0; r < blocks; ++r) listed += block_at(r).listed;

    double u = p.uniform_bytes == 4 ? static_cast<const float*>(p.uniforms)[row]
                                    : static_cast<const double*>(p.uniforms)[row];
    u = u > 0.0 ? u : 0.0;
    const double unit = static_cast<double>(1ull << p.weight_bits);
    auto whole = [&](double w) { return static_cast<unsigned long long>(llrint(w * unit)); };
    int id_bits = 0;
    while (id_bits < 32 && (p.width - 1) >> id_bits) ++id_bits;

    auto block_total = [&](unsigned long long v) {
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh.part[warp] = v;
        __syncthreads();
        unsigned long long s = 0;
#pragma unroll
        for (int w = 0; w < SAMPLE_WARPS; ++w) s += sh.part[w];
        return s;
    };
    // The first bin at which the running sum over sh.bins reaches `want`: its number in sh.found (~0:
    // none) and what is left of `want` in it in sh.left.
    auto crossing = [&](auto bins, unsigned long long want) {
        constexpr int PER = decltype(bins)::value / SAMPLE_THREADS;
        unsigned long long mine = 0;
#pragma unroll
        for (int b = 0; b < PER; ++b) mine += sh.bins[t * PER + b];
        unsigned long long upto = warp_inclusive(mine, lane);
        if (lane == 31) sh.part[warp] = upto;
        if (t == 0) sh.found = ~0ull;
        __syncthreads();
        for (int w = 0; w < warp; ++w) upto += sh.part[w];
        if (upto >= want && upto - mine < want) {
            unsigned long long left = want - (upto - mine);
            int at = t * PER;
            while (sh.bins[at] < left) left -= sh.bins[at++];
            sh.found = at;
            sh.left = left;
        }
        __syncthreads();
    };
    // Of the list's first n entries, from the highest down, the one at which the running sum of `amount`
    // reaches `want`, digit by digit; 0 where the whole sum stays below.  by_id looks at the lower
    // half (~id) alone: ids in ascending order.
    auto select = [&](int n, bool by_id, unsigned long long want, auto&& amount) -> unsigned long long {
        unsigned long long prefix = 0;
        for (int shift = by_id ? 24 : 56; shift >= 0; shift -= 8) {
            if (shift < 32 && shift >= id_bits) { // ~id has ones there
                prefix = (prefix << 8) | 255;
                continue;
            }
            sh.bins[t] = 0;
            __syncthreads();
            for (int i = t; i < n; i += SAMPLE_THREADS) {
                const unsigned long long c = by_id ? sh.list[i] & 0xffffffffull : sh.list[i];
                if (shift < 56 && (c >> (shift + 8)) != prefix) continue;
                const unsigned long long a = amount(i);
                if (a != 0) atomicAdd(&sh.bins[255 - ((c >> shift) & 255)], a);
            }
            __syncthreads();
            crossing(std::integral_constant<int, 256>{}, want);
            const unsigned long long found = sh.found;
            want = sh.left;
            __syncthreads();
            if (found == ~0ull) return 0;
            prefix = (prefix << 8) | (255 - found);
        }
        return prefix;
    };
    // The same by bins of a number that does not rise along the order (bin_of: a bin for an entry): one
    // round of sums, then the few entries of the bin that holds the border.  Where those are more than
    // a warp has lanes, digit by digit.
    auto border_of = [&](int n, bool by_id, unsigned long long want, auto&& bin_of, auto&& amount) -> unsigned long long {
        for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.bins[b] = 0;
        if (t == 0) sh.few = 0;
        __syncthreads();
        for (int i = t; i < n; i += SAMPLE_THREADS) {
            const unsigned long long a = amount(i);
            if (a != 0) atomicAdd(&sh.bins[bin_of(sh.list[i])], a);
        }
        __syncthreads();
        crossing(std::integral_constant<int, SAMPLE_BINS>{}, want);
        const unsigned long long found = sh.found, left = sh.left;
        if (found == ~0ull) {
            __syncthreads();
            return 0;
        }
        for (int i = t; i < n; i += SAMPLE_THREADS)
            if (bin_of(sh.list[i]) == static_cast<int>(found) && amount(i) != 0) {
                const int at = atomicAdd(&sh.few, 1);
                if (at < 32) sh.few_at[at] = i;
            }
        __syncthreads();
        const int few = sh.few;
        if (few > 32) return select(n, by_id, left, [&](int i) { return bin_of(sh.list[i]) == static_cast<int>(found) ? amount(i) : 0ull; });
        if (warp == 0) {
            const int i = lane < few ? sh.few_at[lane] : 0;
            const unsigned long long c = by_id ? sh.list[i] & 0xffffffffull : sh.list[i];
            const unsigned long long a = lane < few ? static_cast<unsigned long long>(amount(i)) : 0;
            unsigned long long before = 0;
            for (int o = 0; o < few; ++o) {
                const unsigned long long other = __shfl_sync(FULL_WARP, c, o), b = __shfl_sync(FULL_WARP, a, o);
                if (other > c) before += b;
            }
            if (lane < few && before < left && before + a >= left) sh.found = c;
        }
        __syncthreads();
        const unsigned long long entry = sh.found;
        __syncthreads();
        return entry;
    };
    // The other blocks' listed entries, appended to this block's (rank 0).
    auto gather = [&] {
        unsigned int at = min(sh.listed, static_cast<unsigned int>(SAMPLE_LIST));
        for (int r = 1; r < blocks; ++r) {
            SampleShared& from = block_at(r);
            const unsigned int c = from.listed;
            for (unsigned int i = t; i < c && at + i < SAMPLE_LIST; i += SAMPLE_THREADS) sh.list[at + i] = from.list[i];
            at += c;
        }
        __syncthreads();
    };

    double listed_mass = 0.0; // weight of the scores from `below` up
    float below = INFINITY;
    if (listing && !lone && listed <= SAMPLE_LIST) {
        if (rank == 0) {
            const int n = static_cast<int>(listed);
            const bool complete = threshold == LOWEST_KEY;
            gather();
            if (t == 0) sh.lowest = 0xffffffffu;
            __syncthreads();
            uint32_t lowest = 0xffffffffu;
            for (int i = t; i < n; i += SAMPLE_THREADS) {
                const uint32_t k = static_cast<uint32_t>(sh.list[i] >> 32);
                lowest = min(lowest, k);
                sh.weight[i] = score_weight(key_score(k), top, inv);
            }
            lowest = __reduce_min_sync(FULL_WARP, lowest);
            if (lane == 0) atomicMin(&sh.lowest, lowest);
            __syncthreads();
            const float spread = top - key_score(sh.lowest);
            const float per_score = spread > 0.0f ? SAMPLE_BINS / spread : 0.0f;
            const float per_id = static_cast<float>(SAMPLE_BINS) / static_cast<float>(p.width);
            auto score_bin = [&](unsigned long long c) {
                return min(SAMPLE_BINS - 1, static_cast<int>((top - key_score(static_cast<uint32_t>(c >> 32))) * per_score));
            };
            auto id_bin = [&](unsigned long long c) {
                return min(SAMPLE_BINS - 1, static_cast<int>(static_cast<float>(~static_cast<uint32_t>(c)) * per_id));
            };
            bool resolved = true;
            unsigned long long cut = 0; // kept are the entries from here up
            if (top_k > 0) {
                if (n >= top_k) cut = border_of(n, false, static_cast<unsigned long long>(top_k), score_bin, [](int) { return 1ull; });
                else resolved = complete;
            }
            if (resolved && nucleus) {
                double mass = total;
                if (top_k > 0) {
                    unsigned long long m = 0;
                    for (int i = t; i < n; i += SAMPLE_THREADS) m += sh.list[i] >= cut ? whole(sh.weight[i]) : 0;
                    mass = static_cast<double>(block_total(m)) / unit;
                }
                const double want = ceil(top_p * mass * unit);
                const unsigned long long from = cut;
                const unsigned long long border = border_of(n, false, want > 1.0 ? static_cast<unsigned long long>(want) : 1ull, score_bin,
                                                            [&](int i) { return sh.list[i] >= from ? whole(sh.weight[i]) : 0ull; });
                if (border != 0) cut = border;
                else if (top_k == 0) resolved = complete; // every listed id is in the nucleus, and more may be
            }
            // min_p alone ends inside the list where the threshold's own weight is below it.
            if (floor_p && !resolved && top_k == 0) resolved = score_weight(key_score(threshold), top, inv) < min_p;
            else if (floor_p && !nucleus && top_k == 0) resolved = complete || score_weight(key_score(threshold), top, inv) < min_p;
            if (resolved) {
                auto kept = [&](int i) -> unsigned long long {
                    const unsigned long long c = sh.list[i];
                    const double w = sh.weight[i];
                    return c >= cut && (w >= min_p || static_cast<uint32_t>(c >> 32) == top_key) ? whole(w) : 0;
                };
                unsigned long long m = 0;
                for (int i = t; i < n; i += SAMPLE_THREADS) m += kept(i);
                m = block_total(m);
                const double target = u * static_cast<double>(m);
                const unsigned long long want = target < static_cast<double>(m) ? min(static_cast<unsigned long long>(target) + 1, m) : m;
                const unsigned long long at = border_of(n, true, want, id_bin, kept);
                if (t == 0) p.ids[row] = static_cast<int64_t>(~static_cast<uint32_t>(at));
            }
            if (!resolved) {
                unsigned long long m = 0;
                for (int i = t; i < n; i += SAMPLE_THREADS) m += whole(sh.weight[i]);
                m = block_total(m);
                if (t == 0) sh.listed_mass = static_cast<double>(m) / unit;
            }
            if (t == 0) sh.outcome = resolved;
        }
        everyone();
        const bool done = block_at(0).outcome != 0;
        listed_mass = block_at(0).listed_mass;
        below = key_score(threshold);
        everyone();
        if (done) return;
    }

    // From here on all blocks of the row work together, each on its own groups.
    uint32_t cut = 0;            // kept are the keys above, and, in id order, the first `ties` of those equal to it
    unsigned long long ties = 0; // (0: every key is kept)
    int parity = 0;
    auto cluster_total = [&](unsigned long long v) {
        v = block_total(v);
        if (blocks == 1) return v;
        if (t == 0) sh.exchange[parity] = v;
        cluster.sync();
        v = 0;
        for (int r = 0; r < blocks; ++r) v += block_at(r).exchange[parity];
        parity ^= 1;
        return v;
    };
    auto each = [&](auto&& f) {
        for (int g = first_group + t; g < last_group; g += SAMPLE_THREADS) {
            float v[N];
            x.load(g, v);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t k = score_key(v[j]);
                if (k != 0) f(v[j], k, static_cast<uint32_t>(x.id(g) + j));
            }
        }
    };
    // Sum over the cluster's bins and counts, in every block.
    auto cluster_bins = [&] {
        if (blocks == 1) return;
        cluster.sync();
        constexpr int PER = SAMPLE_BINS / SAMPLE_THREADS;
        unsigned long long b[PER];
        unsigned int c[PER];
#pragma unroll
        for (int m = 0; m < PER; ++m) {
            b[m] = 0;
            c[m] = 0;
            for (int r = 0; r < blocks; ++r) {
                SampleShared& from = block_at(r);
                b[m] += from.bins[m * SAMPLE_THREADS + t];
                c[m] += from.counts[m * SAMPLE_THREADS + t];
            }
        }
        cluster.sync();
#pragma unroll
        for (int m = 0; m < PER; ++m) {
            sh.bins[m * SAMPLE_THREADS + t] = b[m];
            sh.counts[m * SAMPLE_THREADS + t] = c[m];
        }
        __syncthreads();
    };
    // Narrows `cut` and `ties` to the ids before which the running sum, from the highest score down, is
    // below `want` (counts, or weights with by_mass).
    auto narrow = [&](bool by_mass, unsigned long long want) {
        float hi = top, lo = -FLT_MAX;
        unsigned long long left = want;
        double range = static_cast<double>(top) - static_cast<double>(key_score(sh.probe_low));
        if (by_mass) range = fmin(range, 45.0 / inv); // weights further down are below 2^-64
        // A round parts the lowest from the highest score of its range, and cuts the range of evenly
        // spread scores 1024-fold; float's exponents end it within 40 rounds.
        for (int round = 0; round < 64; ++round) {
            const double scale = range > 0.0 ? SAMPLE_BINS / range : 0.0;
            auto bin_of = [&](float v) {
                const double b = (static_cast<double>(hi) - static_cast<double>(v)) * scale;
                return b < SAMPLE_BINS - 1 ? static_cast<int>(b) : SAMPLE_BINS - 1;
            };
            for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
                sh.bins[b] = 0;
                sh.counts[b] = 0;
            }
            __syncthreads();
            each([&](float v, uint32_t k, uint32_t) {
                if (k <= cut || v > hi || v < lo) return;
                const int b = bin_of(v);
                const unsigned long long a = by_mass ? whole(score_weight(v, top, inv)) : 1ull;
                if (a != 0) atomicAdd(&sh.bins[b], a);
                atomicAdd(&sh.counts[b], 1u);
            });
            __syncthreads();
            cluster_bins();
            crossing(std::integral_constant<int, SAMPLE_BINS>{}, left);
            const unsigned long long found = sh.found;
            if (found == ~0ull) { // first round only: the ids above the cut do not reach `want`
                unsigned long long sum = 0;
                for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) sum += sh.bins[b];
                sum = block_total(sum);
                if (cut != 0 && by_mass) {
                    const unsigned long long w = whole(score_weight(key_score(cut), top, inv));
                    if (w != 0) ties = min(ties, (left - sum + w - 1) / w);
                }
                return;
            }
            const int b = static_cast<int>(found);
            left = sh.left;
            const unsigned int in_bin = sh.counts[b];
            __syncthreads();
            if (in_bin <= SAMPLE_LIST) {
                if (t == 0) sh.listed = 0;
                __syncthreads();
                each([&](float v, uint32_t k, uint32_t id) {
                    if (k <= cut || v > hi || v < lo || bin_of(v) != b) return;
                    const unsigned int at = atomicAdd(&sh.listed, 1u);
                    if (at < SAMPLE_LIST) sh.list[at] = (static_cast<unsigned long long>(k) << 32) | ~id;
                });
                everyone();
                if (rank == 0) {
                    const int n = static_cast<int>(in_bin);
                    gather();
                    for (int i = t; i < n; i += SAMPLE_THREADS)
                        sh.weight[i] = score_weight(key_score(static_cast<uint32_t>(sh.list[i] >> 32)), top, inv);
                    __syncthreads();
                    const unsigned long long border =
                        select(n, false, left, [&](int i) { return by_mass ? whole(sh.weight[i]) : 1ull; });
                    unsigned long long equal = 0;
                    for (int i = t; i < n; i += SAMPLE_THREADS) equal += sh.list[i] >= border && (sh.list[i] >> 32) == (border >> 32);
                    equal = block_total(equal);
                    if (t == 0) {
                        sh.cut = static_cast<uint32_t>(border >> 32);
                        sh.cut_ties = equal;
                    }
                }
                everyone();
                cut = block_at(0).cut;
                ties = block_at(0).cut_ties;
                everyone();
                return;
            }
            // Too many for the list: the bin's own lowest and highest score bound the next round.
            uint32_t low = 0xffffffffu, high = 0;
            each([&](float v, uint32_t k, uint32_t) {
                if (k <= cut || v > hi || v < lo || bin_of(v) != b) return;
                low = min(low, k);
                high = max(high, k);
            });
            low = __reduce_min_sync(FULL_WARP, low);
            high = __reduce_max_sync(FULL_WARP, high);
            if (lane == 0) sh.part[warp] = (static_cast<unsigned long long>(~low) << 32) | high;
            __syncthreads();
            for (int w = 0; w < SAMPLE_WARPS; ++w) {
                low = min(low, ~static_cast<uint32_t>(sh.part[w] >> 32));
                high = max(high, static_cast<uint32_t>(sh.part[w]));
            }
            if (blocks > 1) {
                if (t == 0) sh.exchange[parity] = (static_cast<unsigned long long>(~low) << 32) | high;
                cluster.sync();
                for (int r = 0; r < blocks; ++r) {
                    const unsigned long long e = block_at(r).exchange[parity];
                    low = min(low, ~static_cast<uint32_t>(e >> 32));
                    high = max(high, static_cast<uint32_t>(e));
                }
                parity ^= 1;
            }
            __syncthreads();
            if (low == high) { // one score, many ids
                const unsigned long long w = by_mass ? whole(score_weight(key_score(low), top, inv)) : 1ull;
                cut = low;
                ties = (left + w - 1) / w;
                return;
            }
            hi = key_score(high);
            lo = key_score(low);
            range = static_cast<double>(hi) - static_cast<double>(lo);
        }
    };

    // Whether part_mass and part_ties hold what each warp's ids keep (without a filter the stream left it).
    bool summed = !filtered && !lone;
    if (lone) {
        unsigned long long c = 0;
        each([&](float, uint32_t k, uint32_t) { c += k == top_key; });
        c = cluster_total(c);
        if (top_k > 0) c = min(c, static_cast<unsigned long long>(top_k));
        if (filtered && nucleus) c = static_cast<unsigned long long>(fmax(1.0, ceil(top_p * static_cast<double>(c))));
        cut = top_key;
        ties = c;
    } else if (filtered && top_k > 0) {
        narrow(false, static_cast<unsigned long long>(top_k));
        if (nucleus) {
            unsigned long long m = 0;
            each([&](float v, uint32_t k, uint32_t) { m += k > cut ? whole(score_weight(v, top, inv)) : 0; });
            m = cluster_total(m);
            if (cut != 0) m += ties * whole(score_weight(key_score(cut), top, inv));
            const double want = ceil(top_p * static_cast<double>(m));
            narrow(true, want > 1.0 ? static_cast<unsigned long long>(want) : 1ull);
        }
    } else if (filtered && nucleus) {
        // The border lies below the list.  Counts of the scores below it by bins of their distance from the
        // top, each taken at its bin's middle, place the border to a small part of a bin; the next
        // reading sums the weights above a window around that place and lists the window, and the
        // border is found inside.  Should it lie outside, it is narrowed down from the top instead.
        const double need = top_p * total;
        const float range = static_cast<float>(fmin(static_cast<double>(top) - static_cast<double>(key_score(sh.probe_low)), 45.0 / inv));
        const float per = range > 0.0f ? SAMPLE_BINS / range : 0.0f;
        for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
            sh.bins[b] = 0;
            sh.counts[b] = 0;
        }
        __syncthreads();
        for (int g = first_group + t; g < last_group; g += SAMPLE_THREADS) {
            float v[N];
            x.load(g, v);
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (v[j] < below && v[j] > -INFINITY)
                    atomicAdd(&sh.counts[static_cast<int>(fminf((top - v[j]) * per, SAMPLE_BINS - 1))], 1u);
        }
        __syncthreads();
        cluster_bins();
        for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS)
            sh.bins[b] = whole(exp(-(b + 0.5) / per * inv)) * sh.counts[b];
        __syncthreads();
        const double wanted = (need - listed_mass) * unit;
        crossing(std::integral_constant<int, SAMPLE_BINS>{}, wanted > 1.0 ? static_cast<unsigned long long>(wanted) : 1ull);
        const unsigned long long found = sh.found;
        bool settled = found != ~0ull;
        if (settled) {
            const float count = static_cast<float>(sh.counts[found]);
            const float place = static_cast<float>(found) + static_cast<float>(static_cast<double>(sh.left) / static_cast<double>(sh.bins[found]));
            const float half = fminf(1.0f, 700.0f / count);
            const float from = place - half, to = place + half;
            if (t == 0) sh.listed = 0;
            __syncthreads();
            double sum = 0.0;
            weight_of.refer(top, inv);
            for (int g0 = warp_first; g0 < warp_last; g0 += 32) {
                const int g = g0 + lane;
                float v[N];
                if (g < warp_last) {
                    x.load(g, v);
                } else {
#pragma unroll
                    for (int j = 0; j < N; ++j) v[j] = -INFINITY;
                }
                bool any = false;
                const uint32_t id = static_cast<uint32_t>(x.id(g));
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float y = (top - v[j]) * per;
                    if (y < from) {
                        any = true;
                    } else {
                        if (y <= to && v[j] > -INFINITY) {
                            const unsigned int at = atomicAdd(&sh.listed, 1u);
                            if (at < SAMPLE_LIST) sh.list[at] = (static_cast<unsigned long long>(score_key(v[j])) << 32) | ~(id + j);
                        }
                        v[j] = -INFINITY;
                    }
                }
                if (__any_sync(FULL_WARP, any)) {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const double w = weight_of(v[j], p.taylor);
                        if (v[j] > -INFINITY) sum += w;
                    }
                }
            }
            sum = warp_sum(sum);
            if (lane == 0) sh.mass[warp] = sum * weight_of.factor;
            everyone();
            listed = 0;
            for (int r = 0; r < blocks; ++r) listed += block_at(r).listed;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int e = 2 * lane + h;
                part_mass[h] = e < parts ? block_at(e / SAMPLE_WARPS).mass[e % SAMPLE_WARPS] : 0.0;
            }
            const double rest = (need - warp_sum(part_mass[0] + part_mass[1])) * unit;
            settled = listed <= SAMPLE_LIST && rest >= 1.0;
            if (settled && rank == 0) {
                const int n = static_cast<int>(listed);
                gather();
                for (int i = t; i < n; i += SAMPLE_THREADS)
                    sh.weight[i] = score_weight(key_score(static_cast<uint32_t>(sh.list[i] >> 32)), top, inv);
                __syncthreads();
                const float finer = SAMPLE_BINS / (to - from);
                auto bin_of = [&](unsigned long long c) {
                    const float y = (top - key_score(static_cast<uint32_t>(c >> 32))) * per;
                    return static_cast<int>(fminf(fmaxf(y - from, 0.0f) * finer, SAMPLE_BINS - 1));
                };
                const unsigned long long border = border_of(n, false, static_cast<unsigned long long>(ceil(rest)), bin_of,
                                                            [&](int i) { return whole(sh.weight[i]); });
                for (int e = t; e < SAMPLE_BINS; e += SAMPLE_THREADS) {
                    sh.bins[e] = 0;
                    sh.counts[e] = 0;
                }
                if (t == 0) sh.few = 0;
                __syncthreads();
                const uint32_t key = static_cast<uint32_t>(border >> 32);
                for (int i = t; i < n; i += SAMPLE_THREADS) {
                    const unsigned long long c = sh.list[i];
                    const uint32_t k = static_cast<uint32_t>(c >> 32);
                    if (k < key) continue;
                    // The warp whose ids hold it.
                    const int g = static_cast<int>((static_cast<int64_t>(~static_cast<uint32_t>(c)) + x.lead) / N);
                    const int e = g / per_block * SAMPLE_WARPS + g % per_block / per_warp;
                    if (k > key) atomicAdd(&sh.bins[e], whole(sh.weight[i]));
                    else atomicAdd(&sh.counts[e], 1u);
                    if (k == key && c >= border) atomicAdd(&sh.few, 1);
                }
                __syncthreads();
                if (t == 0) {
                    sh.cut = key;
                    sh.cut_ties = sh.few;
                }
            }
            everyone();
            if (settled) {
                cut = block_at(0).cut;
                ties = block_at(0).cut_ties;
                settled = cut != 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int e = 2 * lane + h;
                    if (e < parts) {
                        part_mass[h] += static_cast<double>(block_at(0).bins[e]) / unit;
                        part_ties[h] = block_at(0).counts[e];
                    }
                }
                summed = settled && !floor_p;
            }
            everyone();
        }
        if (!settled) {
            const double want = ceil(need * unit);
            narrow(true, want > 1.0 ? static_cast<unsigned long long>(want) : 1ull);
        }
    }

    // Each warp's kept weight, ties apart.
    const double cut_weight = cut != 0 ? score_weight(key_score(cut), top, inv) : 0.0;
    weight_of.refer(lone ? 0.0f : top, inv);
    const double min_weight = min_p / weight_of.factor; // in the units of weight_of
    if (!summed) {
        double sum = 0.0;
        unsigned int equal = 0;
        for (int g0 = warp_first; g0 < warp_last; g0 += 32) {
            const int g = g0 + lane;
            float v[N];
            if (g < warp_last) {
                x.load(g, v);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) v[j] = -INFINITY;
            }
            bool any = false;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t k = score_key(v[j]);
                if (cut != 0 && k == cut) ++equal;
                if (k <= cut) v[j] = -INFINITY;
                any |= k > cut;
            }
            if (__any_sync(FULL_WARP, any)) {
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const double w = weight_of(v[j], p.taylor);
                    if (v[j] > -INFINITY && (w >= min_weight || v[j] == top)) sum += w;
                }
            }
        }
        sum = warp_sum(sum) * weight_of.factor;
        equal = __reduce_add_sync(FULL_WARP, equal);
        if (lane == 0) {
            sh.mass[warp] = sum;
            sh.ties[warp] = equal;
        }
        everyone();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = 2 * lane + h;
            part_mass[h] = 0.0;
            if (e < parts) {
                SampleShared& from = block_at(e / SAMPLE_WARPS);
                part_mass[h] = from.mass[e % SAMPLE_WARPS];
                part_ties[h] = from.ties[e % SAMPLE_WARPS];
            }
        }
    }
    everyone(); // the last look at the other blocks

    const bool ties_drawn = cut != 0 && (cut_weight >= min_p || cut == top_key);
    auto clipped = [&](unsigned long long before, unsigned long long have) -> double {
        if (!ties_drawn || before >= ties) return 0.0;
        return static_cast<double>(min(have, ties - before)) * cut_weight;
    };
    const unsigned long long two_ties = part_ties[0] + part_ties[1];
    const unsigned long long ties_before = warp_inclusive(two_ties, lane) - two_ties;
    part_mass[0] += clipped(ties_before, part_ties[0]);
    part_mass[1] += clipped(ties_before + part_ties[0], part_ties[1]);
    const double upto = warp_inclusive(part_mass[0] + part_mass[1], lane);
    const double all = __shfl_sync(FULL_WARP, upto, 31);
    const double target = u * all;
    // The part that holds the target; where rounding leaves none, the last one with a weight.
    auto first_above = [&](double sum_upto, double own) {
        unsigned hit = __ballot_sync(FULL_WARP, sum_upto > target && own > 0.0);
        if (hit != 0) return __ffs(hit) - 1;
        hit = __ballot_sync(FULL_WARP, own > 0.0);
        return 31 - __clz(hit);
    };
    const int pair = first_above(upto, part_mass[0] + part_mass[1]);
    const double pair_before = __shfl_sync(FULL_WARP, upto - part_mass[0] - part_mass[1], pair);
    const double even = __shfl_sync(FULL_WARP, part_mass[0], pair), odd = __shfl_sync(FULL_WARP, part_mass[1], pair);
    const unsigned long long pair_ties = __shfl_sync(FULL_WARP, ties_before, pair);
    const unsigned long long even_ties = __shfl_sync(FULL_WARP, part_ties[0], pair);
    const bool second = !(even > 0.0 && pair_before + even > target) && odd > 0.0;
    const int part = 2 * pair + second;
    if (part / SAMPLE_WARPS != rank) return;

    // This block holds it: its threads share the part's groups, each a run of them in id order.
    const double rest = target - (pair_before + (second ? even : 0.0));
    const unsigned long long seen_before = pair_ties + (second ? even_ties : 0);
    const int part_first = min(first_group + (part % SAMPLE_WARPS) * per_warp, last_group);
    const int part_last = min(part_first + per_warp, last_group);
    const int per_thread = (part_last - part_first + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
    const int mine_first = min(part_first + t * per_thread, part_last), mine_last = min(mine_first + per_thread, part_last);
    double sum = 0.0;
    unsigned long long equal = 0;
    for (int i = 0; i < per_thread; ++i) { // the same count for every lane: weights are worked out together
        float v[N];
        if (mine_first + i < mine_last) {
            x.load(mine_first + i, v);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t k = score_key(v[j]);
            if (cut != 0 && k == cut) ++equal;
            if (k <= cut) v[j] = -INFINITY;
            const double w = weight_of(v[j], p.taylor);
            if (v[j] > -INFINITY && (w >= min_weight || v[j] == top)) sum += w;
        }
    }
    sum *= weight_of.factor;
    // Running sums over the block: of the ties, then of the weights with the ties that are kept.
    const unsigned long long equal_upto = warp_inclusive(equal, lane);
    __syncthreads();
    if (lane == 31) sh.part[warp] = equal_upto;
    __syncthreads();
    unsigned long long seen = seen_before + equal_upto - equal;
    for (int w = 0; w < warp; ++w) seen += sh.part[w];
    const double mine = sum + clipped(seen, equal);
    const double mine_upto = warp_inclusive(mine, lane);
    if (lane == 31) sh.part_mass[warp] = mine_upto;
    if (t == 0) sh.found = ~0ull;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < warp; ++w) before += sh.part_mass[w];
    // The lowest thread whose running sum passes the rest, else the last one with a weight.
    if (mine > 0.0) {
        const bool passes = before + mine_upto > rest;
        atomicMin(&sh.found, passes ? static_cast<unsigned long long>(t) : static_cast<unsigned long long>(2 * SAMPLE_THREADS - t));
    }
    __syncthreads();
    const unsigned long long chosen = sh.found;
    if (chosen != static_cast<unsigned long long>(t) && chosen != static_cast<unsigned long long>(2 * SAMPLE_THREADS - t)) return;
    if (!(mine > 0.0)) return;
    double running = before + mine_upto - mine;
    int64_t id = -1;
    for (int g = mine_first; g < mine_last; ++g) {
        float v[N];
        x.load(g, v);
        for (int j = 0; j < N; ++j) {
            const uint32_t k = score_key(v[j]);
            if (k == 0 || k < cut) continue;
            if (cut != 0 && k == cut && seen++ >= ties) continue;
            const double w = score_weight(v[j], top, inv);
            if (!(w >= min_p || k == top_key) || w == 0.0) continue;
            id = x.id(g) + j;
            running += w;
            if (running > rest) {
                p.ids[row] = id;
                return;
            }
        }
    }
    p.ids[row] = id;
}

} // namespace povs
