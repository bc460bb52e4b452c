// Drawing one id per row from scores, with temperature, top-k, top-p and min-p, from given random
// numbers.
//
// A row is read once.  While it streams by, a cluster of 1 to 8 blocks keeps the highest score, the
// sum of the weights w = exp((x - reference) / temperature), and a list of every score at or above a
// threshold that a probe of the row's scores put near the last rank that can matter.  The filters and the
// draw then work on the list alone, in shared memory.  Only a row whose list turns out too short or too
// long (a nucleus of thousands of ids, top_k in the thousands, rows of equal scores) is read again, to
// find the border by bins of the score's distance from the highest.
//
// Ids have to be those of exact arithmetic, and two borders of a row of 10^5 ids can lie 10^-10 of its sum
// apart: weights and sums have 64 bits.  B200, 512 rows of 131072 float32 (41 us to read at the copy rate):
// 55 us for the reading alone, 75 with top-k 50 (the list), 114 without a filter (the weights: nine 64-bit
// operations a score), 165 for narrow nuclei (both), 285 where one row in five has a nucleus of thousands.
// One row of 50021 with top-k and top-p: 15 us, the latency of about ten steps between barriers.
#pragma once

#include <cooperative_groups.h>

#include <cfloat>
#include <cstdint>
#include <cstring>

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
    int32_t weight_bits;   // in sums of whole numbers over a row a weight of 1 is 2^weight_bits; they stay below 2^63
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
    double poly[4]; // WarpExp's polynomial from r on: in constant memory, where an operand costs no register
};

constexpr int SAMPLE_THREADS = 256;
constexpr int SAMPLE_WARPS = SAMPLE_THREADS / 32;
constexpr int SAMPLE_MAX_CLUSTER = 8;
constexpr int SAMPLE_LIST = 2048;   // listed scores per block, and per row
constexpr double LIST_UNIT = 0x1p51; // a weight of 1 in sums over a list: those stay at or below 2^62
constexpr int SAMPLE_TARGET = 1024; // listed scores aimed at where no top_k says how many
constexpr int SAMPLE_PROBE = 4096;  // scores probed
constexpr int SAMPLE_BINS = 1024;
constexpr int SAMPLE_PARTS = 64; // runs of ids whose weights are summed apart, per row

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
// a factor common to all, to 2^-43 relative.  With z = v * inv / ln 2 = n / 32 + r, |r| <= 1/64, and n0
// the n of the reference, the weight is 2^((n - n0) >> 5) * 2^(((n - n0) & 31) / 32) * 2^r: the second
// factor sits in the lanes' registers (one shuffle in place of a table in memory, whose banks would
// clash), and 2^r is its Taylor polynomial of degree 5 with the last term economised into the lower
// ones by the Chebyshev polynomial T5, which leaves (ln 2)^5 / 120 / 64^5 / 16 < 2^-43.
// The products with inv / ln 2 are exact in both fused operations, so large scores lose nothing.
// Nine operations in 64 bits a score: at half the rate of 32 bits about what its 4 bytes cost to read.
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
    __device__ __forceinline__ double operator()(float v, const double* __restrict__ poly) const
    {
        const double x = static_cast<double>(fmaxf(v, floor));
        const double t = fma(x, scale, magic);
        const double r = fma(x, scale, magic - t);
        const int n = __double2loint(t);
        double q = fma(r, poly[3], poly[2]);
        q = fma(r, q, poly[1]);
        q = fma(r, q, poly[0]);
        const double at = __shfl_sync(FULL_WARP, step, n); // lane n modulo 32
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
    __device__ __forceinline__ void unpack(const uint4& raw, float (&v)[N]) const
    {
        T e[N];
        memcpy(e, &raw, sizeof(raw));
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = to_float(e[j]);
    }
    __device__ __forceinline__ void load_if(bool there, int g, float (&v)[N]) const
    {
        if (there) {
            load(g, v);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = -INFINITY;
        }
    }
    __device__ __forceinline__ void load(int g, float (&v)[N]) const
    {
        const int64_t i = id(g);
        if (i >= 0 && i + N <= width) {
            unpack(__ldg(reinterpret_cast<const uint4*>(x + i)), v);
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
    uint32_t best[SAMPLE_WARPS]; // each warp's highest key
    double mass[SAMPLE_PARTS];     // of each of this block's parts, which follow one another in id order
    float reference[SAMPLE_PARTS]; // that the mass is relative to
    unsigned int ties[SAMPLE_PARTS];
    unsigned long long exchange[2];
    unsigned int listed;
    int outcome;
    uint32_t cut;
    unsigned long long cut_ties;
    // This block's own.
    unsigned long long part[SAMPLE_WARPS];
    unsigned long long part_high[SAMPLE_WARPS];
    unsigned int listed_of[SAMPLE_MAX_CLUSTER];
    double part_mass[SAMPLE_WARPS];
    double listed_mass;
    uint32_t most[SAMPLE_THREADS];
    unsigned int probe_counts[16];
    uint32_t probe_low;
    int few;
    int few_at[32];
    unsigned long long found;
    unsigned long long left;
};

// One block's share of the work on a row.  All blocks of the row's cluster take the same steps: what
// decides them is worked out by each from the same numbers.
template <typename T> struct SampleRow {
    using Groups = RowGroups<T>;
    static constexpr int N = Groups::N;
    using Entry = unsigned long long; // an entry of the list
    using Whole = unsigned long long; // a weight in units, or a count

    const SampleParams& p;
    SampleShared& sh;
    cg::cluster_group cluster;
    Groups x;
    WarpExp weight_of;
    int blocks, rank, t, lane, warp;
    // This block's groups, and within them its parts' (as many to each warp), in id order.
    int per_block, per_part, first_group, last_group;
    int parts, warp_parts; // of this block, of each warp
    // The row's settings.
    int64_t top_k;
    double top_p, min_p, inv, u;
    bool nucleus, floor_p, filtered, need_mass;
    double unit;
    // The list's threshold (`list_from` +infinity: no list).
    uint32_t threshold;
    float list_from;
    bool listing;
    // What the stream leaves.
    float top, warp_top, reference;
    uint32_t top_key;
    // Kept are the keys above `cut` and, in id order, the first `ties` of those equal to it (0: all), of these the
    // ones from `lowest` up.
    uint32_t cut = 0, lowest = LOWEST_KEY;
    Whole ties = 0;
    int parity = 0;
    // Parts 2 lane and 2 lane + 1 of the row.
    double part_mass[2] = {0.0, 0.0};
    Whole part_ties[2] = {0, 0};

    __device__ __forceinline__ SampleRow(const SampleParams& p_, SampleShared& sh_, int64_t row)
        : p(p_), sh(sh_), cluster(cg::this_cluster()), x(static_cast<const T*>(p_.logits) + row * p_.row_stride, p_.width),
          weight_of(threadIdx.x & 31)
    {
        blocks = p.cluster;
        rank = blockIdx.x % blocks;
        t = threadIdx.x;
        lane = t & 31;
        warp = t >> 5;
        per_block = (x.groups + blocks - 1) / blocks;
        parts = SAMPLE_PARTS / blocks;
        warp_parts = parts / SAMPLE_WARPS;
        per_part = (per_block + parts - 1) / parts;
        first_group = min(rank * per_block, x.groups);
        last_group = min(first_group + per_block, x.groups);
        const double temperature = p.temperatures != nullptr ? p.temperatures[row] : p.temperature;
        top_p = p.top_ps != nullptr ? p.top_ps[row] : p.top_p;
        min_p = p.min_ps != nullptr ? p.min_ps[row] : p.min_p;
        top_k = p.top_ks != nullptr ? p.top_ks[row] : p.top_k;
        inv = fmin(fmax(1.0 / temperature, 1e-28), 1e36); // so that 0 * inv stays 0
        nucleus = top_p < 1.0;
        floor_p = min_p > 0.0;
        if (!(temperature > 0.0)) { // the highest score's lowest id is the draw at top_k = 1, at any temperature
            inv = 1.0;
            top_k = 1;
            nucleus = floor_p = false;
        }
        if (!floor_p) min_p = 0.0;
        if (top_k < 0 || top_k >= p.width) top_k = 0;
        filtered = nucleus || floor_p || top_k > 0;
        // The sum of all weights: without a filter, or for a nucleus of the whole row.
        need_mass = top_k == 0 && (nucleus || !floor_p);
        u = p.uniform_bytes == 4 ? static_cast<const float*>(p.uniforms)[row] : static_cast<const double*>(p.uniforms)[row];
        u = u > 0.0 ? u : 0.0;
        unit = static_cast<double>(1ull << p.weight_bits);
    }

    __device__ __forceinline__ void everyone()
    {
        if (blocks > 1) cluster.sync();
        else __syncthreads();
    }
    __device__ __forceinline__ SampleShared& block_at(int r) { return blocks > 1 ? *cluster.map_shared_rank(&sh, r) : sh; }
    __device__ __forceinline__ int part_first(int q) const { return min(first_group + q * per_part, last_group); }
    // Weights as whole numbers, whose sums no order of adding changes: in a row's units for sums over all of it,
    // in the list's own (good to 2^-41 in all) for sums over a list.
    __device__ __forceinline__ Whole whole(double w) const { return static_cast<Whole>(llrint(w * unit)); }
    __device__ __forceinline__ static Whole list_units(double w) { return static_cast<Whole>(llrint(w * LIST_UNIT)); }
    // The least whole number not below `want`, at least 1; beyond a list's whole sum any number is the same.
    __device__ __forceinline__ static Whole least_of(double want) { return want > 1.0 ? static_cast<Whole>(ceil(fmin(want, 0x1p63))) : Whole{1}; }
    __device__ __forceinline__ static float score_of(Entry c) { return key_score(static_cast<uint32_t>(c >> 32)); }

    __device__ __forceinline__ Whole block_total(Whole v)
    {
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh.part[warp] = v;
        __syncthreads();
        Whole s = 0;
#pragma unroll
        for (int w = 0; w < SAMPLE_WARPS; ++w) s += sh.part[w];
        return s;
    }
    __device__ __forceinline__ Whole cluster_total(Whole v)
    {
        v = block_total(v);
        if (blocks == 1) return v;
        if (t == 0) sh.exchange[parity] = v;
        cluster.sync();
        v = 0;
        for (int r = 0; r < blocks; ++r) v += block_at(r).exchange[parity];
        parity ^= 1;
        return v;
    }

    // --- The probe: scores spread evenly over the row.  Its rank that corresponds to the ids wanted,
    // with about three standard deviations to spare where top_k must be met, gives the list's threshold (its
    // upper 16 bits, found bit by bit).  Every block of the row finds the same one.
    __device__ __forceinline__ void probe()
    {
        threshold = LOWEST_KEY;
        listing = filtered;
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
                want = fmin(want + 2.6 * sqrt(want) + 3.6, room);
            }
            const unsigned int rank_wanted = static_cast<unsigned int>(fmax(want, 1.0));
            // Few wanted: that rank among the threads' highest is a little lower, and each warp finds it alone.
            const bool few = rank_wanted <= SAMPLE_THREADS / 4;
            uint32_t most = 0;
#pragma unroll
            for (int m = 0; m < PER; ++m) most = max(most, k[m]);
            sh.most[t] = most;
            __syncthreads();
            uint32_t found = 0;
            if (few) {
                uint32_t of_lane[SAMPLE_WARPS];
#pragma unroll
                for (int m = 0; m < SAMPLE_WARPS; ++m) of_lane[m] = sh.most[m * 32 + lane];
                for (int bit = 31; bit >= 16; --bit) {
                    const uint32_t candidate = found | (1u << bit);
                    unsigned int c = 0;
#pragma unroll
                    for (int m = 0; m < SAMPLE_WARPS; ++m) c += of_lane[m] >= candidate;
                    if (__reduce_add_sync(FULL_WARP, c) >= rank_wanted) found = candidate;
                }
            } else {
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
            }
            threshold = max(found, LOWEST_KEY);
        }
        list_from = listing ? key_score(threshold) : INFINITY;
    }

    // --- The stream.
    // One batch: MANY vectors of this lane, vector u being group g + 32 u.
    template <bool MASS, bool LIST, int MANY>
    __device__ __forceinline__ void take(const float (&v)[MANY][N], int g, float& limit, double (&sums)[2])
    {
        float most = v[0][0];
#pragma unroll
        for (int i = 0; i < MANY; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) most = fmaxf(most, v[i][j]);
        warp_top = fmaxf(warp_top, most);
        if (LIST && most >= list_from) {
#pragma unroll
            for (int i = 0; i < MANY; ++i) {
                const uint32_t id = static_cast<uint32_t>(x.id(g + 32 * i));
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (v[i][j] >= list_from) {
                        const unsigned int at = atomicAdd(&sh.listed, 1u);
                        if (at < SAMPLE_LIST) sh.list[at] = (static_cast<Entry>(score_key(v[i][j])) << 32) | ~(id + j);
                    }
            }
        }
        if (MASS) {
            // The reference is the first scores' highest, renewed only when a weight would pass e^64.
            if (__any_sync(FULL_WARP, most > limit)) {
                float higher = most > -INFINITY ? most : -INFINITY;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) higher = fmaxf(higher, __shfl_xor_sync(FULL_WARP, higher, o));
                const double old_factor = weight_of.factor;
                weight_of.refer(higher, inv);
                const bool keep = reference > LONE;
                const double rescale = keep ? old_factor * score_weight(reference, higher, inv) / weight_of.factor : 0.0;
                sums[0] = keep ? sums[0] * rescale : 0.0;
                sums[1] = keep ? sums[1] * rescale : 0.0;
                reference = higher;
                limit = static_cast<float>(static_cast<double>(reference) + 64.0 / inv);
            }
#pragma unroll
            for (int i = 0; i < MANY; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) sums[j & 1] += weight_of(v[i][j], p.poly);
        }
    }
    // Groups wholly inside the row are read UNROLL vectors a lane at a time; the row's first and last
    // group, which may reach outside, go by themselves.
    template <bool MASS, bool LIST> __device__ __forceinline__ void stream()
    {
        constexpr int UNROLL = 16 / N;
        float limit = -INFINITY;
        warp_top = reference = -INFINITY;
        const uint4* vectors = reinterpret_cast<const uint4*>(x.x - x.lead);
        // Without sums to keep apart, a warp's parts are one run.
        for (int q = warp * warp_parts; q < (warp + 1) * warp_parts; q += MASS ? 1 : warp_parts) {
            double sums[2] = {0.0, 0.0};
            const int from = part_first(q), to = part_first(MASS ? q + 1 : q + warp_parts);
            const int full_first = max(from, x.lead > 0 ? 1 : 0);
            const int full_last = min(to, static_cast<int>((x.width + x.lead) / N));
            int g = full_first + lane;
            uint4 next[UNROLL];
            if (!MASS && g - lane + 32 * UNROLL <= full_last) {
#pragma unroll
                for (int i = 0; i < UNROLL; ++i) next[i] = __ldg(vectors + g + 32 * i);
            }
            for (; g - lane + 32 * UNROLL <= full_last; g += 32 * UNROLL) {
                float v[UNROLL][N];
                if (MASS) {
#pragma unroll
                    for (int i = 0; i < UNROLL; ++i) next[i] = __ldg(vectors + g + 32 * i);
                }
#pragma unroll
                for (int i = 0; i < UNROLL; ++i) x.unpack(next[i], v[i]);
                // Without sums a batch ahead is in flight (82 -> 77 us for top_k on 512 rows of 131072; with
                // sums the registers that takes cost more than it gains).
                if (!MASS && g - lane + 64 * UNROLL <= full_last) {
#pragma unroll
                    for (int i = 0; i < UNROLL; ++i) next[i] = __ldg(vectors + g + 32 * (UNROLL + i));
                }
                take<MASS, LIST, UNROLL>(v, g, limit, sums);
            }
            for (; g - lane < full_last; g += 32) {
                float v[1][N];
                x.load_if(g < full_last, g, v[0]);
                take<MASS, LIST, 1>(v, g, limit, sums);
            }
#pragma unroll 1
            for (int end = 0; end < 2; ++end) {
                const int at = end == 0 ? 0 : x.groups - 1;
                const bool outside = end == 0 ? x.lead > 0 : at >= full_last && (at > 0 || x.lead == 0);
                if (outside && from <= at && at < to) {
                    float v[1][N];
                    x.load_if(lane == 0, at, v[0]);
                    take<MASS, LIST, 1>(v, at, limit, sums);
                }
            }
            if (MASS) {
                const double sum = warp_sum(sums[0] + sums[1]);
                if (lane == 0) {
                    sh.mass[q] = reference > LONE && sum > 1e-90 ? sum * weight_of.factor : 0.0; // masked scores alone: 0
                    sh.reference[q] = reference;
                }
            }
        }
    }

    // --- Work on a list of n entries in sh.list, their weights in sh.weight.
    // The first of BINS bins at which the running sum over sh.bins reaches `want`: its number in sh.found
    // (~0: none) and what is left of `want` in it in sh.left.
    template <int BINS> __device__ __forceinline__ void crossing(Whole want)
    {
        constexpr int PER = BINS / SAMPLE_THREADS;
        Whole mine = 0;
#pragma unroll
        for (int b = 0; b < PER; ++b) mine += sh.bins[t * PER + b];
        Whole upto = warp_inclusive(mine, lane);
        if (lane == 31) sh.part[warp] = upto;
        if (t == 0) sh.found = ~0ull;
        __syncthreads();
        for (int w = 0; w < warp; ++w) upto += sh.part[w];
        if (upto >= want && upto - mine < want) {
            Whole left = want - (upto - mine);
            int at = t * PER;
            while (sh.bins[at] < left) left -= sh.bins[at++];
            sh.found = at;
            sh.left = left;
        }
        __syncthreads();
    }
    // Lowest and highest of a block's numbers (nothing to give: ~0 and 0).
    __device__ __forceinline__ void block_range(Entry& low, Entry& high)
    {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            low = min(low, __shfl_xor_sync(FULL_WARP, low, o));
            high = max(high, __shfl_xor_sync(FULL_WARP, high, o));
        }
        __syncthreads();
        if (lane == 0) {
            sh.part[warp] = low;
            sh.part_high[warp] = high;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SAMPLE_WARPS; ++w) {
            low = min(low, sh.part[w]);
            high = max(high, sh.part_high[w]);
        }
    }
    // Of the list's first n entries, in descending order, the one at which the running sum of `amount` reaches
    // `want`; 0 where the whole sum stays below.  BY_ID orders by the lower half (~id) alone: ids ascend.
    // A round sums into bins between the highest and the lowest entry, by score or, where those are
    // equal, by id, and goes on with the entries of the bin that holds the border, until a warp can hold
    // them.  Evenly spread entries end in one round, those of 16-bit scores, many equal, in two.
    template <bool BY_ID, typename Amount> __device__ __forceinline__ Entry border_of(int n, Whole want, Amount amount)
    {
        auto order = [&](int i) { return BY_ID ? sh.list[i] & 0xffffffffull : sh.list[i]; };
        Entry low = ~0ull, high = 0; // the entries still in question
        for (int i = t; i < n; i += SAMPLE_THREADS)
            if (amount(i) != 0) {
                low = min(low, order(i));
                high = max(high, order(i));
            }
        block_range(low, high);
        if (low > high) return 0;
        for (;;) {
            for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) sh.bins[b] = 0;
            if (t == 0) sh.few = 0;
            __syncthreads();
            const uint32_t id_high = static_cast<uint32_t>(high), id_range = id_high - static_cast<uint32_t>(low);
            const bool by_id = (low >> 32) == (high >> 32);
            const double score_high = score_of(high), spread = score_high - score_of(low);
            const double per_score = spread > 0.0 ? SAMPLE_BINS / spread : 0.0, per_id = SAMPLE_BINS / (id_range + 1.0);
            auto bin_of = [&](Entry c) {
                const double b = by_id ? (id_high - static_cast<uint32_t>(c)) * per_id : (score_high - score_of(c)) * per_score;
                return b < SAMPLE_BINS - 1 ? static_cast<int>(b) : SAMPLE_BINS - 1;
            };
            for (int i = t; i < n; i += SAMPLE_THREADS) {
                const Entry c = order(i);
                if (c < low || c > high) continue;
                const Whole a = amount(i);
                if (a != 0) atomicAdd(&sh.bins[bin_of(c)], a);
            }
            __syncthreads();
            crossing<SAMPLE_BINS>(want);
            const Whole found = sh.found;
            want = sh.left;
            if (found == ~0ull) {
                __syncthreads();
                return 0;
            }
            const int bin = static_cast<int>(found);
            Entry next_low = ~0ull, next_high = 0;
            for (int i = t; i < n; i += SAMPLE_THREADS) {
                const Entry c = order(i);
                if (c < low || c > high || bin_of(c) != bin || amount(i) == 0) continue;
                next_low = min(next_low, c);
                next_high = max(next_high, c);
                const int at = atomicAdd(&sh.few, 1);
                if (at < 32) sh.few_at[at] = i;
            }
            __syncthreads();
            const int few = sh.few;
            if (few <= 32) {
                if (warp == 0) {
                    const int i = lane < few ? sh.few_at[lane] : 0;
                    const Entry c = order(i);
                    const Whole a = lane < few ? amount(i) : Whole{0};
                    Whole before = 0;
                    for (int o = 0; o < few; ++o) {
                        const Entry other = __shfl_sync(FULL_WARP, c, o);
                        const Whole b = __shfl_sync(FULL_WARP, a, o);
                        if (other > c) before += b;
                    }
                    if (lane < few && before < want && before + a >= want) sh.found = c;
                }
                __syncthreads();
                const Entry entry = sh.found;
                __syncthreads();
                return entry;
            }
            block_range(next_low, next_high);
            low = next_low;
            high = next_high;
        }
    }
    // The other blocks' listed entries, appended to rank 0's, and all their weights.
    __device__ __forceinline__ void gather(int n)
    {
        if (blocks > 1) {
            // Where each block's entries go; every thread then fetches its own, all on their way at once.
            if (t < blocks) sh.listed_of[t] = block_at(t).listed;
            __syncthreads();
            for (int i = static_cast<int>(sh.listed_of[0]) + t; i < n; i += SAMPLE_THREADS) {
                unsigned int at = i, r = 0;
                while (at >= sh.listed_of[r]) at -= sh.listed_of[r++];
                sh.list[i] = block_at(r).list[at];
            }
            __syncthreads();
        }
        for (int i = t; i < n; i += SAMPLE_THREADS)
            sh.weight[i] = score_weight(key_score(static_cast<uint32_t>(sh.list[i] >> 32)), top, inv);
        __syncthreads();
    }
    // A short list, an entry per thread: each sums what stands before it in the order of the scores, and
    // then in that of the ids, over all others.
    __device__ __forceinline__ bool draw_from_short_list(int n, double total, int64_t row, bool complete)
    {
        const Entry mine = t < n ? sh.list[t] : 0;
        const double w = t < n ? sh.weight[t] : 0.0;
        const Whole units = t < n ? list_units(w) : 0;
        sh.bins[t] = units;
        __syncthreads();
        int rank_of_mine = 0;
        Whole before = 0;
#pragma unroll 4
        for (int i = 0; i < n; ++i)
            if (sh.list[i] > mine) {
                ++rank_of_mine;
                before += sh.bins[i];
            }
        bool keep = t < n && (top_k == 0 || rank_of_mine < top_k), resolved = top_k == 0 || n >= top_k || complete;
        if (resolved && nucleus) {
            const Whole mass = block_total(keep ? units : 0);
            const Whole least = least_of(top_p * (top_k > 0 ? static_cast<double>(mass) : total * LIST_UNIT));
            keep &= before < least;
            if (top_k == 0) resolved = complete || mass >= least;
        }
        if (!ends_inside(resolved, complete, n)) return false;
        keep &= w >= min_p || static_cast<uint32_t>(mine >> 32) == top_key;
        if (u == 0.0) {
            Entry first = keep && w > 0.0 ? static_cast<Entry>(static_cast<uint32_t>(~mine)) : ~0ull, unused = 0;
            block_range(first, unused);
            if (t == 0) p.ids[row] = static_cast<int64_t>(first);
            return true;
        }
        const Whole kept = keep ? units : 0;
        const Whole m = block_total(kept);
        sh.bins[t] = kept;
        __syncthreads();
        Whole upto = 0;
        const uint32_t order = static_cast<uint32_t>(mine); // ~id
#pragma unroll 4
        for (int i = 0; i < n; ++i)
            if (static_cast<uint32_t>(sh.list[i]) >= order) upto += sh.bins[i];
        const double target = u * static_cast<double>(m);
        const Whole want = target < static_cast<double>(m) ? min(static_cast<Whole>(target) + 1, m) : m;
        if (kept != 0 && upto >= want && upto - kept < want) p.ids[row] = static_cast<int64_t>(~order);
        return true;
    }
    // Whether the filters' borders lie inside the list; else its weight is left in sh.listed_mass.  min_p ends
    // inside where the threshold's own weight is below it.
    __device__ __forceinline__ bool ends_inside(bool resolved, bool complete, int n)
    {
        if (floor_p && top_k == 0 && (!resolved || !nucleus))
            resolved = complete || score_weight(key_score(threshold), top, inv) < min_p;
        if (resolved) return true;
        Whole m = 0;
        for (int i = t; i < n; i += SAMPLE_THREADS) m += list_units(sh.weight[i]);
        m = block_total(m);
        if (t == 0) sh.listed_mass = static_cast<double>(m) / LIST_UNIT;
        return false;
    }
    // Rank 0: the filters and the draw on the list, which holds every score from the threshold up; false
    // where they reach below it.
    __device__ __forceinline__ bool draw_from_list(int n, double total, int64_t row)
    {
        const bool complete = threshold == LOWEST_KEY;
        gather(n);
        if (n <= SAMPLE_THREADS) return draw_from_short_list(n, total, row, complete);
        bool resolved = true;
        Entry border = 0; // kept are the entries from here up
        if (top_k > 0) {
            if (n >= top_k) border = border_of<false>(n, static_cast<Whole>(top_k), [](int) { return Whole{1}; });
            else resolved = complete;
        }
        if (resolved && nucleus) {
            const Entry from = border;
            Whole m = 0;
            for (int i = t; i < n; i += SAMPLE_THREADS) m += sh.list[i] >= from ? list_units(sh.weight[i]) : Whole{0};
            m = block_total(m);
            const Whole least = least_of(top_p * (top_k > 0 ? static_cast<double>(m) : total * LIST_UNIT));
            if (m >= least)
                border = max(from, border_of<false>(n, least, [&](int i) { return sh.list[i] >= from ? list_units(sh.weight[i]) : Whole{0}; }));
            else if (top_k == 0)
                resolved = complete; // every listed id is in the nucleus, and more may be
        }
        if (!ends_inside(resolved, complete, n)) return false;
        const Entry from = border;
        auto kept = [&](int i) {
            const double w = sh.weight[i];
            return sh.list[i] >= from && (w >= min_p || static_cast<uint32_t>(sh.list[i] >> 32) == top_key) ? list_units(w) : Whole{0};
        };
        if (u == 0.0) { // the lowest id kept, however small its weight
            Entry first = ~0ull, unused = 0;
            for (int i = t; i < n; i += SAMPLE_THREADS)
                if (sh.list[i] >= from && sh.weight[i] > 0.0 && (sh.weight[i] >= min_p || static_cast<uint32_t>(sh.list[i] >> 32) == top_key))
                    first = min(first, static_cast<Entry>(static_cast<uint32_t>(~sh.list[i])));
            block_range(first, unused);
            if (t == 0) p.ids[row] = static_cast<int64_t>(first);
            return true;
        }
        Whole m = 0;
        for (int i = t; i < n; i += SAMPLE_THREADS) m += kept(i);
        m = block_total(m);
        const double target = u * static_cast<double>(m);
        const Whole want = target < static_cast<double>(m) ? min(static_cast<Whole>(target) + 1, m) : m;
        const Entry at = border_of<true>(n, want, kept);
        if (t == 0) p.ids[row] = static_cast<int64_t>(~static_cast<uint32_t>(at));
        return true;
    }

    // --- Rows that are read again, all blocks together, each on its own groups.
    // f(scores, group) for the groups first, first + step, ... below last, four in flight; the same number
    // of calls for every `first` of a run of `step` lanes or threads, groups past `last` as -infinity.
    template <typename F> __device__ __forceinline__ void groups_of(int first, int step, int last, int rounds, F f)
    {
        for (int i = 0; i < rounds; i += 4) {
            float v[4][N];
#pragma unroll
            for (int m = 0; m < 4; ++m) x.load_if(i + m < rounds && first + (i + m) * step < last, first + (i + m) * step, v[m]);
#pragma unroll
            for (int m = 0; m < 4; ++m)
                if (i + m < rounds) f(v[m], first + (i + m) * step);
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f)
    {
        const int rounds = (last_group - first_group + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
        groups_of(first_group + t, SAMPLE_THREADS, last_group, rounds, [&](float (&v)[N], int g) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t k = score_key(v[j]);
                if (k != 0) f(v[j], k, static_cast<uint32_t>(x.id(g) + j));
            }
        });
    }
    // f(scores, group) for a part's groups, the warp together.
    template <typename F> __device__ __forceinline__ void each_of_part(int q, F f)
    {
        const int from = part_first(q), to = part_first(q + 1);
        groups_of(from + lane, 32, to, (to - from + 31) / 32, f);
    }
    __device__ __forceinline__ void clear_bins()
    {
        for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
            sh.bins[b] = 0;
            sh.counts[b] = 0;
        }
        __syncthreads();
    }
    // Sums of the cluster's bins and counts, in every block.
    __device__ __forceinline__ void cluster_bins()
    {
        __syncthreads();
        if (blocks == 1) return;
        cluster.sync();
        constexpr int PER = SAMPLE_BINS / SAMPLE_THREADS;
        Whole b[PER];
        unsigned int c[PER];
#pragma unroll
        for (int m = 0; m < PER; ++m) {
            b[m] = 0;
            c[m] = 0;
        }
#pragma unroll 2
        for (int r = 0; r < blocks; ++r) {
            SampleShared& from = block_at(r);
#pragma unroll
            for (int m = 0; m < PER; ++m) {
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
    }
    __device__ __forceinline__ unsigned int cluster_listed()
    {
        unsigned int n = 0;
        for (int r = 0; r < blocks; ++r) n += block_at(r).listed;
        return n;
    }
    // Narrows `cut` and `ties` to the ids before which the running sum, from the highest score down, is
    // below `want` (counts, or weights with BY_MASS), by bins of the distance from the highest score.
    // A round parts the lowest from the highest score of its range, and cuts the range of evenly spread
    // scores 1024-fold; float's exponents end it within 40 rounds.
    template <bool BY_MASS> __device__ __forceinline__ void narrow(Whole want)
    {
        float hi = top, lo = -FLT_MAX;
        Whole left = want;
        double range = static_cast<double>(top) - static_cast<double>(key_score(sh.probe_low));
        if (BY_MASS) range = fmin(range, 45.0 / inv); // weights further down are below 2^-64
        for (int round = 0; round < 64; ++round) {
            const double scale = range > 0.0 ? SAMPLE_BINS / range : 0.0;
            auto bin_of = [&](float v) {
                const double b = (static_cast<double>(hi) - static_cast<double>(v)) * scale;
                return b < SAMPLE_BINS - 1 ? static_cast<int>(b) : SAMPLE_BINS - 1;
            };
            clear_bins();
            each([&](float v, uint32_t k, uint32_t) {
                if (k <= cut || v > hi || v < lo) return;
                const int b = bin_of(v);
                const Whole a = BY_MASS ? whole(score_weight(v, top, inv)) : Whole{1};
                if (a != 0) atomicAdd(&sh.bins[b], a);
                atomicAdd(&sh.counts[b], 1u);
            });
            cluster_bins();
            crossing<SAMPLE_BINS>(left);
            const Whole found = sh.found;
            if (found == ~0ull) { // first round only: the ids above the cut do not reach `want`
                Whole sum = 0;
                for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) sum += sh.bins[b];
                sum = block_total(sum);
                if (cut != 0 && BY_MASS) {
                    const Whole w = whole(score_weight(key_score(cut), top, inv));
                    if (w != 0) ties = min(ties, (left - sum + w - 1) / w);
                }
                return;
            }
            const int bin = static_cast<int>(found);
            left = sh.left;
            const unsigned int in_bin = sh.counts[bin];
            if (t == 0) sh.listed = 0;
            __syncthreads();
            if (in_bin <= SAMPLE_LIST) {
                each([&](float v, uint32_t k, uint32_t id) {
                    if (k <= cut || v > hi || v < lo || bin_of(v) != bin) return;
                    const unsigned int at = atomicAdd(&sh.listed, 1u);
                    if (at < SAMPLE_LIST) sh.list[at] = (static_cast<Entry>(k) << 32) | ~id;
                });
                everyone();
                if (rank == 0) {
                    const int n = static_cast<int>(in_bin);
                    gather(n);
                    const Entry border = border_of<false>(n, left, [&](int i) { return BY_MASS ? whole(sh.weight[i]) : Whole{1}; });
                    Whole equal = 0;
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
                if (k <= cut || v > hi || v < lo || bin_of(v) != bin) return;
                low = min(low, k);
                high = max(high, k);
            });
            low = __reduce_min_sync(FULL_WARP, low);
            high = __reduce_max_sync(FULL_WARP, high);
            if (lane == 0) sh.part[warp] = (static_cast<Whole>(~low) << 32) | high;
            __syncthreads();
            for (int w = 0; w < SAMPLE_WARPS; ++w) {
                low = min(low, ~static_cast<uint32_t>(sh.part[w] >> 32));
                high = max(high, static_cast<uint32_t>(sh.part[w]));
            }
            if (blocks > 1) {
                if (t == 0) sh.exchange[parity] = (static_cast<Whole>(~low) << 32) | high;
                cluster.sync();
                for (int r = 0; r < blocks; ++r) {
                    const Whole e = block_at(r).exchange[parity];
                    low = min(low, ~static_cast<uint32_t>(e >> 32));
                    high = max(high, static_cast<uint32_t>(e));
                }
                parity ^= 1;
            }
            __syncthreads();
            if (low == high) { // one score, many ids
                const Whole w = BY_MASS ? whole(score_weight(key_score(low), top, inv)) : Whole{1};
                cut = low;
                ties = (left + w - 1) / w;
                return;
            }
            hi = key_score(high);
            lo = key_score(low);
            range = static_cast<double>(hi) - static_cast<double>(lo);
        }
    }
    // A nucleus whose border lies below the list (scores from `below` up weigh listed_mass).  Counts of the
    // scores below it by bins of their distance from the top, each taken at its bin's middle or mean, place
    // the border to a small part of a bin; the next reading sums the weights above a window around that
    // place and lists the window, and the border is found inside, with each part's kept weight.  False
    // where it lies outside (none of 256 rows of 131072 normal scores at three temperatures and shares).
    __device__ __forceinline__ bool border_in_window(double need, double listed_mass, float below)
    {
        const float range = static_cast<float>(fmin(static_cast<double>(top) - static_cast<double>(key_score(sh.probe_low)), 45.0 / inv));
        const float per = range > 0.0f ? SAMPLE_BINS / range : 0.0f;
        // Scores of 16 bits sit unevenly in a bin: the sum of their places in it, in steps of 1/256, gives the mean.
        constexpr bool UNEVEN = sizeof(T) == 2;
        unsigned int* places = reinterpret_cast<unsigned int*>(sh.weight); // the list's weights are done with
        if (UNEVEN)
            for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) places[b] = 0;
        clear_bins();
        groups_of(first_group + t, SAMPLE_THREADS, last_group, (last_group - first_group + SAMPLE_THREADS - 1) / SAMPLE_THREADS,
                  [&](float (&v)[N], int) {
#pragma unroll
                      for (int j = 0; j < N; ++j)
                          if (v[j] < below && v[j] > -INFINITY) {
                              const float y = (top - v[j]) * per;
                              const int bin = static_cast<int>(fminf(y, SAMPLE_BINS - 1));
                              atomicAdd(&sh.counts[bin], 1u);
                              if (UNEVEN) atomicAdd(&places[bin], static_cast<unsigned int>(fminf((y - bin) * 256.0f, 255.0f)));
                          }
                  });
        __syncthreads();
        for (int b = t; b < SAMPLE_BINS; b += SAMPLE_THREADS) {
            const unsigned int c = sh.counts[b];
            const double mean = UNEVEN && c != 0 ? (places[b] / static_cast<double>(c) + 0.5) / 256 : 0.5;
            sh.bins[b] = whole(exp(-(b + mean) / per * inv)) * c;
        }
        cluster_bins();
        const double wanted = (need - listed_mass) * unit;
        crossing<SAMPLE_BINS>(wanted > 1.0 ? static_cast<Whole>(wanted) : Whole{1});
        const Whole found = sh.found;
        if (found == ~0ull) {
            __syncthreads();
            return false;
        }
        // The window [from, to) in bins: the border's bin and up to three on either side (scores of 16 bits sit
        // unevenly in their bins), or one, as far as the list holds them; of a bin too full for it, the part
        // around the border's place.
        constexpr unsigned int ROOM = SAMPLE_LIST - 200;
        const int bin = static_cast<int>(found);
        const float place = static_cast<float>(static_cast<double>(sh.left) / static_cast<double>(sh.bins[bin]));
        auto count_of = [&](int b) { return b >= 0 && b < SAMPLE_BINS ? sh.counts[b] : 0u; };
        unsigned int inside_window = sh.counts[bin];
        float from = static_cast<float>(bin), to = from + 1.0f;
        if (inside_window > ROOM) {
            from += place - 700.0f / static_cast<float>(inside_window);
            to = from + 1400.0f / static_cast<float>(inside_window);
        } else if (inside_window + count_of(bin - 1) + count_of(bin + 1) > ROOM) {
            if (place < 0.5f && inside_window + count_of(bin - 1) <= ROOM) from -= 1.0f;
            if (place >= 0.5f && inside_window + count_of(bin + 1) <= ROOM) to += 1.0f;
        } else {
            for (int around = 1; around <= 3; ++around) {
                inside_window += count_of(bin - around) + count_of(bin + around);
                if (around > 1 && inside_window > ROOM / 2) break;
                from -= 1.0f;
                to += 1.0f;
            }
        }
        if (t == 0) sh.listed = 0;
        __syncthreads();
        for (int q = warp * warp_parts; q < (warp + 1) * warp_parts; ++q) {
            double sum = 0.0;
            each_of_part(q, [&](float (&v)[N], int g) {
                bool any = false;
                const uint32_t id = static_cast<uint32_t>(x.id(g));
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float y = (top - v[j]) * per;
                    if (y < from) {
                        any = true;
                    } else {
                        if (y < to && v[j] > -INFINITY) {
                            const unsigned int at = atomicAdd(&sh.listed, 1u);
                            if (at < SAMPLE_LIST) sh.list[at] = (static_cast<Entry>(score_key(v[j])) << 32) | ~(id + j);
                        }
                        v[j] = -INFINITY;
                    }
                }
                if (__any_sync(FULL_WARP, any)) {
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        const double w = weight_of(v[j], p.poly);
                        if (v[j] > -INFINITY) sum += w;
                    }
                }
            });
            sum = warp_sum(sum);
            if (lane == 0) sh.mass[q] = sum * weight_of.factor;
        }
        everyone();
        const unsigned int listed = cluster_listed();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = 2 * lane + h;
            part_mass[h] = block_at(e / parts).mass[e % parts];
        }
        const double rest = (need - warp_sum(part_mass[0] + part_mass[1])) * LIST_UNIT;
        const bool inside = listed <= SAMPLE_LIST && rest >= 1.0;
        if (inside && rank == 0) {
            const int n = static_cast<int>(listed);
            gather(n);
            const Entry border = border_of<false>(n, least_of(rest), [&](int i) { return list_units(sh.weight[i]); });
            clear_bins();
            if (t == 0) sh.few = 0;
            __syncthreads();
            const uint32_t key = static_cast<uint32_t>(border >> 32);
            for (int i = t; i < n; i += SAMPLE_THREADS) {
                const Entry c = sh.list[i];
                const uint32_t k = static_cast<uint32_t>(c >> 32);
                if (k < key) continue;
                // The part that holds it.
                const int g = static_cast<int>((static_cast<int64_t>(~static_cast<uint32_t>(c)) + x.lead) / N);
                const int e = g / per_block * parts + g % per_block / per_part;
                if (k > key) atomicAdd(&sh.bins[e], list_units(sh.weight[i]));
                else atomicAdd(&sh.counts[e], 1u);
                if (c >= border && k == key) atomicAdd(&sh.few, 1);
            }
            __syncthreads();
            if (t == 0) {
                sh.cut = key;
                sh.cut_ties = sh.few;
            }
        }
        everyone();
        if (inside) {
            cut = block_at(0).cut;
            ties = block_at(0).cut_ties;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int e = 2 * lane + h;
                part_mass[h] += static_cast<double>(block_at(0).bins[e]) / LIST_UNIT;
                part_ties[h] = block_at(0).counts[e];
            }
        }
        everyone();
        return inside && cut != 0;
    }

    // --- The draw in id order, with `cut` and `ties` settled.
    // The lowest key that sums and draw count, the same for both.  Scores whose weight is below 2^-400 (masks of a
    // finite value) are left out: WarpExp gives them 2^-500 and more, where in 64 bits they weigh nothing that a
    // random number could tell.
    __device__ __forceinline__ uint32_t lowest_counted() const
    {
        const float v = __double2float_ru(static_cast<double>(top) - 400.0 * 0.69314718055994530942 / inv);
        return min(max(score_key(v), LOWEST_KEY), top_key);
    }
    // The lowest key whose weight is `least` or more (the highest score's always is): a warp's 32 lanes cut the
    // range of keys 33-fold a round, with the weights that the list is filtered by.
    __device__ __forceinline__ uint32_t lowest_of(double least) const
    {
        uint32_t below = LOWEST_KEY - 1, kept = top_key;
        while (kept - below > 1) {
            const uint32_t at = below + static_cast<uint32_t>(static_cast<uint64_t>(kept - below) * (lane + 1) / 33);
            const unsigned in = __ballot_sync(FULL_WARP, at > below && score_weight(key_score(at), top, inv) >= least);
            const uint32_t last_out = __shfl_sync(FULL_WARP, at, in == 0 ? 31 : max(__ffs(in) - 2, 0));
            const uint32_t first_in = __shfl_sync(FULL_WARP, at, in == 0 ? 0 : __ffs(in) - 1);
            if (!(in & 1)) below = last_out;
            if (in != 0) kept = first_in;
        }
        return kept;
    }
    // Weight of `have` ids equal to the cut, `before` of them before.
    __device__ __forceinline__ double tied(Whole before, Whole have, double cut_weight) const
    {
        return before >= ties ? 0.0 : static_cast<double>(min(have, ties - before)) * cut_weight;
    }
    // Adds a group's kept weights, ties apart, in units of weight_of.  The whole warp takes part.
    __device__ __forceinline__ void add_kept(float (&v)[N], double& sum, Whole& equal)
    {
        bool any = false;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t k = score_key(v[j]);
            const bool in = k > cut && k >= lowest;
            equal += cut != 0 && k == cut;
            if (!in) v[j] = -INFINITY;
            any |= in;
        }
        if (__any_sync(FULL_WARP, any)) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const double w = weight_of(v[j], p.poly);
                if (v[j] > -INFINITY) sum += w;
            }
        }
    }
    __device__ __forceinline__ void sum_parts()
    {
        for (int q = warp * warp_parts; q < (warp + 1) * warp_parts; ++q) {
            double sum = 0.0;
            Whole equal = 0;
            each_of_part(q, [&](float (&v)[N], int) { add_kept(v, sum, equal); });
            sum = warp_sum(sum) * weight_of.factor;
            equal = warp_sum(equal);
            if (lane == 0) {
                sh.mass[q] = sum;
                sh.ties[q] = static_cast<unsigned int>(equal);
            }
        }
        everyone();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int e = 2 * lane + h;
            SampleShared& from = block_at(e / parts);
            part_mass[h] = from.mass[e % parts];
            part_ties[h] = from.ties[e % parts];
        }
    }
    __device__ __forceinline__ void draw(int64_t row)
    {
        const double w_cut = cut != 0 ? score_weight(key_score(cut), top, inv) : 0.0;
        const double cut_weight = cut >= lowest ? w_cut : 0.0;
        const Whole two_ties = part_ties[0] + part_ties[1];
        const Whole ties_before = warp_inclusive(two_ties, lane) - two_ties;
        part_mass[0] += tied(ties_before, part_ties[0], cut_weight);
        part_mass[1] += tied(ties_before + part_ties[0], part_ties[1], cut_weight);
        // A part of nothing but scores left out would be one without an id to draw.  (A draw at 0 counts every
        // score with a weight in 64 bits, and its sums are above 0 where there is one.)
        const double least = u == 0.0 ? 0.0 : warp_sum(part_mass[0] + part_mass[1]) * 0x1p-200;
#pragma unroll
        for (int h = 0; h < 2; ++h) part_mass[h] = part_mass[h] > least ? part_mass[h] : 0.0;
        const double two = part_mass[0] + part_mass[1];
        const double upto = warp_inclusive(two, lane);
        const double target = u * __shfl_sync(FULL_WARP, upto, 31);
        // The pair that holds the target; where rounding leaves none, the last one with a weight.
        const unsigned above = __ballot_sync(FULL_WARP, upto > target && two > 0.0), some = __ballot_sync(FULL_WARP, two > 0.0);
        const int pair = above != 0 ? __ffs(above) - 1 : 31 - __clz(some);
        // What lies before it: the sum that was compared with the target there, not one rebuilt by a
        // subtraction, which may round to above the target.
        const double before_lane = __shfl_up_sync(FULL_WARP, upto, 1);
        const double before_pair = __shfl_sync(FULL_WARP, lane == 0 ? 0.0 : before_lane, pair);
        const double even = __shfl_sync(FULL_WARP, part_mass[0], pair), odd = __shfl_sync(FULL_WARP, part_mass[1], pair);
        const Whole pair_ties = __shfl_sync(FULL_WARP, ties_before, pair), even_ties = __shfl_sync(FULL_WARP, part_ties[0], pair);
        const bool second = !(even > 0.0 && before_pair + even > target) && odd > 0.0;
        const int part = 2 * pair + second;
        if (some == 0 || part / parts != rank) return;

        // This block holds it: its threads share the part's groups, each a run of them in id order.
        const double rest = fmax(target - (before_pair + (second ? even : 0.0)), 0.0);
        const int from = part_first(part % parts), to = part_first(part % parts + 1);
        const int per_thread = (to - from + SAMPLE_THREADS - 1) / SAMPLE_THREADS;
        const int mine_first = min(from + t * per_thread, to), mine_last = min(mine_first + per_thread, to);
        double sum = 0.0;
        Whole equal = 0;
        groups_of(mine_first, 1, mine_last, per_thread, [&](float (&v)[N], int) { add_kept(v, sum, equal); });
        // Running sums over the block: of the ties, then of the weights with the ties that are kept.
        const Whole equal_upto = warp_inclusive(equal, lane);
        __syncthreads();
        if (lane == 31) sh.part[warp] = equal_upto;
        __syncthreads();
        Whole seen = pair_ties + (second ? even_ties : 0) + equal_upto - equal;
        for (int w = 0; w < warp; ++w) seen += sh.part[w];
        const double mine = sum * weight_of.factor + tied(seen, equal, cut_weight);
        const double mine_upto = warp_inclusive(mine, lane), up = __shfl_up_sync(FULL_WARP, mine_upto, 1);
        if (lane == 31) sh.part_mass[warp] = mine_upto;
        if (t == 0) sh.found = ~0ull;
        __syncthreads();
        double before = 0.0;
        for (int w = 0; w < warp; ++w) before += sh.part_mass[w];
        // The lowest thread whose running sum passes the rest, else the last one with a weight.
        const Whole ticket = before + mine_upto > rest ? t : 2 * SAMPLE_THREADS - t;
        if (mine > 0.0) atomicMin(&sh.found, ticket);
        __syncthreads();
        if (!(mine > 0.0) || sh.found != ticket) return;
        double running = lane == 0 ? before : before + up;
        bool done = false;
        int64_t id = -1; // the thread's first kept id whatever the sums say, then the next ones
        for (int g = mine_first; g < mine_last; ++g) {
            float v[N];
            x.load(g, v);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t k = score_key(v[j]);
                if (k < lowest || k < cut) continue;
                if (cut != 0 && k == cut && seen++ >= ties) continue;
                if (done) continue;
                id = x.id(g) + j;
                running += score_weight(v[j], top, inv);
                done = running > rest;
            }
            if (done) break;
        }
        p.ids[row] = id;
    }

    __device__ __forceinline__ void run(int64_t row)
    {
        if (t == 0) {
            sh.listed = 0;
            sh.probe_low = 0xffffffffu;
        }
        if (t < 16) sh.probe_counts[t] = 0;
        __syncthreads();
        probe();
        if (listing && need_mass) stream<true, true>();
        else if (listing) stream<false, true>();
        else if (need_mass) stream<true, false>();
        else stream<false, false>();
        {
            const uint32_t key = __reduce_max_sync(FULL_WARP, score_key(warp_top));
            if (lane == 0) sh.best[warp] = key;
        }
        everyone();

        // Every warp of every block works out the row's totals for itself.
        top_key = 0;
        for (int e = lane; e < blocks * SAMPLE_WARPS; e += 32) top_key = max(top_key, block_at(e / SAMPLE_WARPS).best[e % SAMPLE_WARPS]);
        top_key = __reduce_max_sync(FULL_WARP, top_key);
        top = key_score(top_key);
        const unsigned int listed = cluster_listed();
        const bool lone = top == INFINITY || top < LONE; // no list, no sums
        double total = 0.0; // sum of all weights, relative to the highest score
        if (top_key != 0 && !lone && need_mass) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int e = 2 * lane + h;
                SampleShared& from = block_at(e / parts);
                const double m = from.mass[e % parts];
                if (m > 0.0) part_mass[h] = m / score_weight(top, from.reference[e % parts], inv);
            }
            total = warp_sum(part_mass[0] + part_mass[1]);
        }
        if (top_key == 0) {
            if (rank == 0 && t == 0) p.ids[row] = -1;
            everyone(); // the last look at the other blocks
            return;
        }
        double listed_mass = 0.0; // weight of the scores from `below` up
        float below = INFINITY;
        if (listing && !lone && listed <= SAMPLE_LIST) {
            if (rank == 0) {
                const bool done = draw_from_list(static_cast<int>(listed), total, row);
                if (t == 0) sh.outcome = done;
            }
            everyone();
            const bool done = block_at(0).outcome != 0;
            listed_mass = block_at(0).listed_mass;
            below = key_score(threshold);
            everyone();
            if (done) return;
        }

        weight_of.refer(lone ? 0.0f : top, inv);
        lowest = lowest_counted();
        if (u == 0.0 && !lone) lowest = lowest_of(fmax(min_p, 4.9406564584124654e-324));
        else if (floor_p && !lone) lowest = max(lowest, lowest_of(min_p));
        bool summed = !filtered && !lone && u != 0.0; // part_mass and part_ties hold what each part's ids keep
        if (lone) {
            Whole c = 0;
            each([&](float, uint32_t k, uint32_t) { c += k == top_key; });
            c = cluster_total(c);
            if (top_k > 0) c = min(c, static_cast<Whole>(top_k));
            if (nucleus) c = static_cast<Whole>(fmax(1.0, ceil(top_p * static_cast<double>(c))));
            cut = top_key;
            ties = c;
        } else if (top_k > 0) {
            narrow<false>(static_cast<Whole>(top_k));
            if (nucleus) {
                Whole m = 0;
                each([&](float v, uint32_t k, uint32_t) { m += k > cut ? whole(score_weight(v, top, inv)) : Whole{0}; });
                m = cluster_total(m);
                if (cut != 0) m += ties * whole(score_weight(key_score(cut), top, inv));
                const double want = ceil(top_p * static_cast<double>(m));
                narrow<true>(want > 1.0 ? static_cast<Whole>(want) : Whole{1});
            }
        } else if (nucleus) {
            const double need = top_p * total;
            if (border_in_window(need, listed_mass, below)) {
                summed = !floor_p && u != 0.0;
            } else {
                const double want = ceil(need * unit);
                narrow<true>(want > 1.0 ? static_cast<Whole>(want) : Whole{1});
            }
        }
        if (!summed) sum_parts();
        everyone(); // the last look at the other blocks
        draw(row);
    }
};

// Grid: rows * cluster blocks, `cluster` neighbours per row.
template <typename T>
__global__ void __launch_bounds__(SAMPLE_THREADS, 4) povs_sample_kernel(const __grid_constant__ SampleParams p)
{
    __shared__ SampleShared sh;
    const int64_t row = blockIdx.x / p.cluster;
    SampleRow<T>(p, sh, row).run(row);
}

} // namespace povs
