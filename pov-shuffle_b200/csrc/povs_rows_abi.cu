// C ABI of the row operators (route, plan, dispatch, combine) and of sampling: argument checks and
// launches.  Declarations are in include/povs.h.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <initializer_list>

#include "povs_host.h"
#include "povs_rows.cuh"
#include "povs_sample.cuh"

using povs_host::cuda_fail;
using povs_host::DeviceGuard;
using povs_host::fail;
using povs_host::g_err;
using povs_host::MAX_DEVICES;

namespace {

std::atomic<int> g_sms[MAX_DEVICES]; // 0: not asked yet

// Makes `device` current and returns its SM count.  No allocation and no stream operation, so the
// first call may be inside a stream capture.
int enter(DeviceGuard& dg, int32_t device, int* sms)
{
    if (device < 0 || device >= MAX_DEVICES) return fail(POVS_ERR_INVALID_ARGUMENT, "device %d out of range", device);
    int r = dg.enter(device);
    if (r != POVS_OK) return r;
    int n = g_sms[device].load(std::memory_order_relaxed);
    if (n == 0) {
        int major = 0;
        POVS_CUDA_TRY(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device));
        if (major < 10) return fail(POVS_ERR_UNSUPPORTED, "device %d is sm_%dx; this library is built for sm_100a (B200)", device, major);
        POVS_CUDA_TRY(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device));
        g_sms[device].store(n, std::memory_order_relaxed);
    }
    *sms = n;
    return POVS_OK;
}

int launched(const char* what)
{
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? POVS_OK : cuda_fail(e, what);
}

int element_bytes(int32_t dtype) { return dtype == POVS_FLOAT32 ? 4 : 2; }

int check_dtype(int32_t dtype)
{
    if (dtype != POVS_FLOAT32 && dtype != POVS_BFLOAT16 && dtype != POVS_FLOAT16)
        return fail(POVS_ERR_INVALID_ARGUMENT, "dtype (%d) must be POVS_FLOAT32, POVS_BFLOAT16 or POVS_FLOAT16", dtype);
    return POVS_OK;
}

// Largest power of two up to 16 that divides every number given.
int common_alignment(std::initializer_list<uint64_t> numbers)
{
    uint64_t all = 16;
    for (uint64_t v : numbers) all |= v;
    return static_cast<int>(all & (~all + 1));
}

uint64_t address(const void* p) { return reinterpret_cast<uint64_t>(p); }

// The kernels load whole elements: one that is not on a multiple of its size would be a fault on the GPU.
struct Elements {
    const char* name;
    const void* p;
    int64_t size;
};
int check_aligned(std::initializer_list<Elements> all)
{
    for (const Elements& e : all)
        if (address(e.p) % e.size != 0)
            return fail(POVS_ERR_INVALID_ARGUMENT, "%s is not aligned to its elements of %lld bytes", e.name, static_cast<long long>(e.size));
    return POVS_OK;
}

// Blocks of a grid-stride kernel: one per `per_block` units, at most `waves` per SM.
int grid_for(int64_t units, int64_t per_block, int sms, int waves)
{
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((units + per_block - 1) / per_block,
                                                                   static_cast<int64_t>(sms) * waves)));
}

int check_route(const povs::RouteParams& p, int32_t dtype, int32_t scoring, int32_t group_score)
{
    int r = check_dtype(dtype);
    if (r != POVS_OK) return r;
    if (p.rows < 0) return fail(POVS_ERR_INVALID_ARGUMENT, "rows (%lld) must not be negative", static_cast<long long>(p.rows));
    if (p.n_experts < 1) return fail(POVS_ERR_INVALID_ARGUMENT, "n_experts (%d) must be at least 1", p.n_experts);
    if (p.n_experts > POVS_MAX_ROUTE_EXPERTS)
        return fail(POVS_ERR_UNSUPPORTED, "%d experts exceed the limit of %d", p.n_experts, POVS_MAX_ROUTE_EXPERTS);
    if (p.row_stride < 0) return fail(POVS_ERR_INVALID_ARGUMENT, "row_stride must not be negative");
    if (p.rows > 0 && p.logits == nullptr) return fail(POVS_ERR_INVALID_ARGUMENT, "logits is NULL");
    if (scoring != POVS_SCORE_SOFTMAX && scoring != POVS_SCORE_SIGMOID)
        return fail(POVS_ERR_INVALID_ARGUMENT, "scoring (%d) must be POVS_SCORE_SOFTMAX or POVS_SCORE_SIGMOID", scoring);
    if (group_score != POVS_GROUP_TOP2 && group_score != POVS_GROUP_MAX)
        return fail(POVS_ERR_INVALID_ARGUMENT, "group_score (%d) must be POVS_GROUP_TOP2 or POVS_GROUP_MAX", group_score);
    if (p.n_groups < 1 || p.n_experts % p.n_groups != 0)
        return fail(POVS_ERR_INVALID_ARGUMENT, "n_groups (%d) must divide n_experts (%d)", p.n_groups, p.n_experts);
    if (p.n_groups > 32) return fail(POVS_ERR_UNSUPPORTED, "%d groups exceed the limit of 32", p.n_groups);
    if (p.top_groups < 1 || p.top_groups > p.n_groups)
        return fail(POVS_ERR_INVALID_ARGUMENT, "top_groups (%d) must be in [1, n_groups = %d]", p.top_groups, p.n_groups);
    const int reach = p.n_experts / p.n_groups * p.top_groups;
    if (p.top_k < 1 || p.top_k > reach)
        return fail(POVS_ERR_INVALID_ARGUMENT, "top_k (%d) must be in [1, %d], the experts of the kept groups", p.top_k, reach);
    if (p.top_k > POVS_MAX_TOP_K)
        return fail(POVS_ERR_UNSUPPORTED, "top_k (%d) exceeds the limit of %d", p.top_k, POVS_MAX_TOP_K);
    if (!std::isfinite(p.scale)) return fail(POVS_ERR_INVALID_ARGUMENT, "scale must be finite");
    if (p.rows > (int64_t{1} << 31) / 4) // one block holds four rows
        return fail(POVS_ERR_UNSUPPORTED, "rows (%lld) exceed the limit of 2^29", static_cast<long long>(p.rows));
    return POVS_OK;
}

template <typename T, int EPL> void launch_route_of(const povs::RouteParams& p, int sms, cudaStream_t s)
{
    constexpr int V = EPL < 16 / static_cast<int>(sizeof(T)) ? EPL : 16 / static_cast<int>(sizeof(T));
    const bool vector = p.n_experts % V == 0 && p.row_stride % V == 0 && address(p.logits) % (V * sizeof(T)) == 0;
    const int grid = grid_for(p.rows, povs::ROUTE_WARPS, sms, 16);
    if (vector) povs::povs_route_kernel<T, EPL, true><<<grid, 32 * povs::ROUTE_WARPS, 0, s>>>(p);
    else povs::povs_route_kernel<T, EPL, false><<<grid, 32 * povs::ROUTE_WARPS, 0, s>>>(p);
}

// Up to 41 KB of shared memory (248 experts in 31 groups, float32).
template <typename T, int L, bool SIGMOID, bool BY_LOGIT, bool GROUPED> void launch_route_lanes(const povs::RouteParams& p, cudaStream_t s)
{
    constexpr int ROWS = 32 / L;
    const int floats = (BY_LOGIT ? 0 : p.n_experts) + (GROUPED ? 2 * ROWS * p.n_groups : 0);
    const int smem = ROWS * povs::route_pitch(p.n_experts * static_cast<int>(sizeof(T))) + 4 * floats;
    povs::povs_route_lanes_kernel<T, L, SIGMOID, BY_LOGIT, GROUPED>
        <<<static_cast<unsigned>((p.rows + ROWS - 1) / ROWS), 32, smem, s>>>(p);
}

template <typename T, int L> void launch_route_lanes_of(const povs::RouteParams& p, cudaStream_t s)
{
    const bool grouped = p.top_groups < p.n_groups, by_logit = p.bias == nullptr && !grouped;
    if (by_logit) p.sigmoid ? launch_route_lanes<T, L, true, true, false>(p, s) : launch_route_lanes<T, L, false, true, false>(p, s);
    else if (grouped) p.sigmoid ? launch_route_lanes<T, L, true, false, true>(p, s) : launch_route_lanes<T, L, false, false, true>(p, s);
    else p.sigmoid ? launch_route_lanes<T, L, true, false, false>(p, s) : launch_route_lanes<T, L, false, false, false>(p, s);
}

// Lanes per row: as many (1, 2, 4 or 8) as bring a warp's rows below 9 KB, in whole pieces of experts and groups.
int route_lanes(const povs::RouteParams& p, int element)
{
    int lanes = 1;
    while (lanes < 8 && 32 / lanes * p.n_experts * element > 9 * 1024 && p.n_experts / (2 * lanes) % 8 == 0 &&
           p.n_experts % (2 * lanes) == 0 && (p.top_groups == p.n_groups || p.n_groups % (2 * lanes) == 0))
        lanes *= 2;
    return lanes;
}

// Lanes where rows fill the GPU with them, eight choices or fewer are asked, and rows and groups come in
// whole pieces; else a warp per row.  B200, float32, top 8: 65536 x 256 with groups 57 us against 94 by warps,
// 16384 x 256 13 against 20, but 8192 x 256 20 against 14 and 16384 x 512 58 against 36.
bool route_by_lanes(const povs::RouteParams& p, int element, int sms)
{
    return p.rows >= 64 * static_cast<int64_t>(sms) && p.top_k <= povs::ROUTE_LIST && p.n_experts <= povs::ROUTE_LANES_EXPERTS && p.n_experts % 8 == 0 &&
           (p.top_groups == p.n_groups || p.n_experts / p.n_groups % 8 == 0) && p.n_experts * element % 16 == 0 &&
           p.row_stride * element % 16 == 0 && address(p.logits) % 16 == 0;
}

template <typename T> void launch_route(const povs::RouteParams& p, int sms, cudaStream_t s)
{
    if (route_by_lanes(p, sizeof(T), sms)) {
        switch (route_lanes(p, sizeof(T))) {
        case 8: return launch_route_lanes_of<T, 8>(p, s);
        case 4: return launch_route_lanes_of<T, 4>(p, s);
        case 2: return launch_route_lanes_of<T, 2>(p, s);
        default: return launch_route_lanes_of<T, 1>(p, s);
        }
    }
    const int epl = (p.n_experts + 31) / 32;
    if (epl <= 1) launch_route_of<T, 1>(p, sms, s);
    else if (epl <= 2) launch_route_of<T, 2>(p, sms, s);
    else if (epl <= 4) launch_route_of<T, 4>(p, sms, s);
    else if (epl <= 8) launch_route_of<T, 8>(p, sms, s);
    else if (epl <= 16) launch_route_of<T, 16>(p, sms, s);
    else launch_route_of<T, 32>(p, sms, s);
}

int check_rows(int64_t rows, int32_t top_k, int64_t n_slots)
{
    if (rows < 0 || n_slots < 0) return fail(POVS_ERR_INVALID_ARGUMENT, "rows and n_slots must not be negative");
    if (top_k < 1) return fail(POVS_ERR_INVALID_ARGUMENT, "top_k (%d) must be at least 1", top_k);
    if (rows > INT32_MAX / top_k || n_slots > INT32_MAX)
        return fail(POVS_ERR_UNSUPPORTED, "rows * top_k and n_slots must be below 2^31");
    return POVS_OK;
}

// Warps per row of the moving kernels, as a power of two: one for each run of the row, as long as all
// rows together have fewer than 64 per SM.
int split_of(int64_t rows, int64_t runs, int sms, int most_log2)
{
    int s = 0;
    while (s < most_log2 && (int64_t{1} << s) < runs && (rows << s) < 64 * static_cast<int64_t>(sms)) ++s;
    return s;
}

template <int BYTES> void launch_dispatch(povs::DispatchParams& p, int sms, cudaStream_t s)
{
    constexpr int UNROLL = BYTES == 16 ? 4 : BYTES == 8 ? 8 : 16;
    const int64_t runs = (p.row_bytes / BYTES + 32 * UNROLL - 1) / (32 * UNROLL);
    p.split_log2 = split_of(p.rows, runs, sms, 10);
    povs::povs_dispatch_kernel<BYTES, UNROLL>
        <<<grid_for(std::max(p.rows << p.split_log2, int64_t{1}), povs::MOVE_WARPS, sms, 8), 32 * povs::MOVE_WARPS, 0, s>>>(p);
}

template <typename T, int N, int UNROLL, int AT_ONCE> void launch_combine(povs::CombineParams& p, int sms, cudaStream_t s)
{
    const int64_t runs = (p.width / N + 32 * UNROLL - 1) / (32 * UNROLL);
    p.split_log2 = split_of(p.rows, runs, sms, 10);
    povs::povs_combine_kernel<T, N, UNROLL, AT_ONCE>
        <<<grid_for(p.rows << p.split_log2, povs::MOVE_WARPS, sms, 8), 32 * povs::MOVE_WARPS, 0, s>>>(p);
}

template <typename T, int N, int AT_ONCE> void launch_combine_backward(povs::CombineParams& p, int sms, cudaStream_t s)
{
    constexpr int UNROLL = N == 1 ? 4 : 1;
    p.split_log2 = split_of(p.rows, (p.width / N + 32 * UNROLL - 1) / (32 * UNROLL), sms, 3);
    povs::povs_combine_backward_kernel<T, N, UNROLL, AT_ONCE>
        <<<grid_for(std::max(p.rows << p.split_log2, int64_t{1}), povs::MOVE_WARPS, sms, 8), 32 * povs::MOVE_WARPS, 0, s>>>(p);
}

// 16 bytes per load where every row starts on a multiple of 16 bytes, else one element.  Eight loads in
// flight: four pieces of two slots, whatever top_k leaves over (184 us for 16384 rows of 4096 bfloat16
// from 8 slots, against 207 for two pieces of four slots), or two of four in rows shorter than that.
template <typename T> void launch_combine_by(int align, povs::CombineParams& p, int sms, cudaStream_t s)
{
    constexpr int N = 16 / sizeof(T);
    if (align < 16) launch_combine<T, 1, 4, 4>(p, sms, s);
    else if (p.top_k == 1) launch_combine<T, N, 2, 1>(p, sms, s);
    else if (p.width < 128 * N) launch_combine<T, N, 2, 4>(p, sms, s);
    else launch_combine<T, N, 4, 2>(p, sms, s);
}

template <typename T, int N> void launch_combine_backward_of(povs::CombineParams& p, int sms, cudaStream_t s)
{
    if (p.top_k <= 2) launch_combine_backward<T, N, 2>(p, sms, s);
    else if (p.top_k <= 4) launch_combine_backward<T, N, 4>(p, sms, s);
    else launch_combine_backward<T, N, 8>(p, sms, s);
}

template <typename T> void launch_combine_backward_by(int align, povs::CombineParams& p, int sms, cudaStream_t s)
{
    if (align >= 16) launch_combine_backward_of<T, 16 / sizeof(T)>(p, sms, s);
    else launch_combine_backward_of<T, 1>(p, sms, s);
}

int check_combine(const povs::CombineParams& p, int32_t dtype)
{
    int r = check_dtype(dtype);
    if (r != POVS_OK) return r;
    r = check_rows(p.rows, p.top_k, p.n_slots);
    if (r != POVS_OK) return r;
    if (p.width < 0 || p.data_stride < 0) return fail(POVS_ERR_INVALID_ARGUMENT, "width and data_stride must not be negative");
    if (p.rows > 0 && p.slots == nullptr) return fail(POVS_ERR_INVALID_ARGUMENT, "slots is NULL");
    return POVS_OK;
}

// Blocks per row: as many as the GPU holds at once for these rows (four per SM), of 2048 ids or more;
// two where a nucleus may be wide, which is read again (512 rows of 131072, top-p 0.9: 288 us against 384,
// but 90 against 75 for top-k 50).
int sample_cluster(int64_t rows, int64_t width, bool nucleus, int sms)
{
    int c = nucleus && rows < (1 << 29) && width >= 8192 ? 2 : 1;
    while (2 * c <= povs::SAMPLE_MAX_CLUSTER && rows * 2 * c <= 4 * static_cast<int64_t>(sms) && width / (2 * c) >= 2048) c *= 2;
    return c;
}

template <typename T> cudaError_t launch_sample(const povs::SampleParams& p, cudaStream_t s)
{
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(p.rows * p.cluster));
    config.blockDim = dim3(povs::SAMPLE_THREADS);
    config.stream = s;
    cudaLaunchAttribute attribute{};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = static_cast<unsigned>(p.cluster);
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = p.cluster > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&config, povs::povs_sample_kernel<T>, p);
}

} // namespace

extern "C" int povs_sample_v1(const void* logits, int32_t dtype, int64_t rows, int64_t width, int64_t row_stride,
                              const void* uniforms, int32_t uniform_bytes, const float* temperatures,
                              double temperature, const int32_t* top_ks, int64_t top_k, const float* top_ps,
                              double top_p, const float* min_ps, double min_p, int64_t* ids, int32_t device,
                              void* stream)
{
    g_err[0] = '\0';
    int r = check_dtype(dtype);
    if (r != POVS_OK) return r;
    if (rows < 0 || width < 1 || row_stride < 0)
        return fail(POVS_ERR_INVALID_ARGUMENT, "rows must not be negative, width at least 1, row_stride not negative");
    if (rows > INT32_MAX || width > INT32_MAX) return fail(POVS_ERR_UNSUPPORTED, "rows and width must be below 2^31");
    if (uniform_bytes != 4 && uniform_bytes != 8)
        return fail(POVS_ERR_INVALID_ARGUMENT, "uniform_bytes (%d) must be 4 or 8", uniform_bytes);
    if (rows > 0 && (logits == nullptr || uniforms == nullptr || ids == nullptr))
        return fail(POVS_ERR_INVALID_ARGUMENT, "logits, uniforms and ids must not be NULL");
    if (temperatures == nullptr && !(temperature >= 0.0 && std::isfinite(temperature)))
        return fail(POVS_ERR_INVALID_ARGUMENT, "temperature must be finite and not negative");
    if (top_ks == nullptr && top_k < 0) return fail(POVS_ERR_INVALID_ARGUMENT, "top_k must not be negative");
    if (top_ps == nullptr && !(top_p >= 0.0 && top_p <= 1.0)) return fail(POVS_ERR_INVALID_ARGUMENT, "top_p must be in [0, 1]");
    if (min_ps == nullptr && !(min_p >= 0.0 && min_p <= 1.0)) return fail(POVS_ERR_INVALID_ARGUMENT, "min_p must be in [0, 1]");
    r = check_aligned({{"logits", logits, element_bytes(dtype)}, {"uniforms", uniforms, uniform_bytes}, {"temperatures", temperatures, 4},
                       {"top_ks", top_ks, 4}, {"top_ps", top_ps, 4}, {"min_ps", min_ps, 4}, {"ids", ids, 8}});
    if (r != POVS_OK) return r;
    if (rows == 0) return POVS_OK;
    DeviceGuard dg;
    int sms = 0;
    r = enter(dg, device, &sms);
    if (r != POVS_OK) return r;
    povs::SampleParams p{};
    p.logits = logits;
    p.rows = rows;
    p.width = width;
    p.row_stride = row_stride;
    p.uniforms = uniforms;
    p.uniform_bytes = uniform_bytes;
    int log2 = 0;
    while ((int64_t{1} << log2) < width) ++log2;
    p.weight_bits = std::min(52, 62 - log2);
    p.temperatures = temperatures;
    p.top_ks = top_ks;
    p.top_ps = top_ps;
    p.min_ps = min_ps;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.ids = ids;
    // 2^r = 1 + r (poly[0] + r (poly[1] + ...)): Taylor terms (ln 2)^i / i!, the fifth economised for
    // |r| <= h: r^5 = 5/4 h^2 r^3 - 5/16 h^4 r, up to h^5 / 16.
    const double ln2 = 0.69314718055994530942, h2 = 1.0 / (64 * 64), fifth = ln2 * ln2 * ln2 * ln2 * ln2 / 120;
    p.poly[0] = ln2 - 0.3125 * h2 * h2 * fifth;
    p.poly[1] = ln2 * ln2 / 2;
    p.poly[2] = ln2 * ln2 * ln2 / 6 + 1.25 * h2 * fifth;
    p.poly[3] = ln2 * ln2 * ln2 * ln2 / 24;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    p.cluster = sample_cluster(rows, width, top_ps != nullptr || (top_p < 1.0 && top_ks == nullptr && top_k == 0), sms);
    cudaError_t e;
    if (dtype == POVS_FLOAT32) e = launch_sample<float>(p, s);
    else if (dtype == POVS_BFLOAT16) e = launch_sample<__nv_bfloat16>(p, s);
    else e = launch_sample<__half>(p, s);
    return e == cudaSuccess ? launched("sample kernel") : cuda_fail(e, "sample kernel");
}

extern "C" int povs_route_v1(const void* logits, int32_t dtype, int64_t rows, int32_t n_experts, int64_t row_stride,
                             const float* bias, int32_t top_k, int32_t scoring, int32_t n_groups, int32_t top_groups,
                             int32_t group_score, int32_t renormalize, float scale, int32_t* experts, float* weights,
                             int32_t device, void* stream)
{
    g_err[0] = '\0';
    povs::RouteParams p{};
    p.logits = logits;
    p.bias = bias;
    p.rows = rows;
    p.row_stride = row_stride;
    p.n_experts = n_experts;
    p.top_k = top_k;
    p.sigmoid = scoring == POVS_SCORE_SIGMOID;
    p.n_groups = n_groups;
    p.top_groups = top_groups;
    p.group_max = group_score == POVS_GROUP_MAX;
    p.renormalize = renormalize != 0;
    p.scale = scale;
    p.experts = experts;
    p.weights = weights;
    int r = check_route(p, dtype, scoring, group_score);
    if (r != POVS_OK) return r;
    if (rows == 0) return POVS_OK;
    if (experts == nullptr || weights == nullptr)
        return fail(POVS_ERR_INVALID_ARGUMENT, "experts and weights must not be NULL");
    r = check_aligned({{"logits", logits, element_bytes(dtype)}, {"bias", bias, 4}, {"experts", experts, 4}, {"weights", weights, 4}});
    if (r != POVS_OK) return r;
    DeviceGuard dg;
    int sms = 0;
    r = enter(dg, device, &sms);
    if (r != POVS_OK) return r;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == POVS_FLOAT32) launch_route<float>(p, sms, s);
    else if (dtype == POVS_BFLOAT16) launch_route<__nv_bfloat16>(p, sms, s);
    else launch_route<__half>(p, sms, s);
    return launched("route kernel");
}

extern "C" int povs_route_backward_v1(const void* logits, int32_t dtype, int64_t rows, int32_t n_experts,
                                      int64_t row_stride, int32_t top_k, int32_t scoring, int32_t renormalize,
                                      float scale, const int32_t* experts, const float* grad_weights,
                                      void* grad_logits, int32_t device, void* stream)
{
    g_err[0] = '\0';
    povs::RouteParams p{};
    p.logits = logits;
    p.rows = rows;
    p.row_stride = row_stride;
    p.n_experts = n_experts;
    p.top_k = top_k;
    p.sigmoid = scoring == POVS_SCORE_SIGMOID;
    p.n_groups = p.top_groups = 1;
    p.renormalize = renormalize != 0;
    p.scale = scale;
    p.chosen = experts;
    p.grad_weights = grad_weights;
    p.grad_logits = grad_logits;
    int r = check_route(p, dtype, scoring, POVS_GROUP_TOP2);
    if (r != POVS_OK) return r;
    if (rows == 0) return POVS_OK;
    if (experts == nullptr || grad_weights == nullptr || grad_logits == nullptr)
        return fail(POVS_ERR_INVALID_ARGUMENT, "experts, grad_weights and grad_logits must not be NULL");
    r = check_aligned({{"logits", logits, element_bytes(dtype)}, {"grad_logits", grad_logits, element_bytes(dtype)},
                       {"experts", experts, 4}, {"grad_weights", grad_weights, 4}});
    if (r != POVS_OK) return r;
    DeviceGuard dg;
    int sms = 0;
    r = enter(dg, device, &sms);
    if (r != POVS_OK) return r;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>((rows + 3) / 4);
    if (dtype == POVS_FLOAT32) povs::povs_route_backward_kernel<float><<<grid, 128, 0, s>>>(p);
    else if (dtype == POVS_BFLOAT16) povs::povs_route_backward_kernel<__nv_bfloat16><<<grid, 128, 0, s>>>(p);
    else povs::povs_route_backward_kernel<__half><<<grid, 128, 0, s>>>(p);
    return launched("route backward kernel");
}

namespace {

// Blocks and entries per block of the plan's kernels: one block (and one launch) up to 4096
// entries, then one per 2048 entries, at most one per SM.
constexpr int64_t PLAN_ONE_BLOCK = 4096, PLAN_ENTRIES_PER_BLOCK = 2048, PLAN_MAX_BLOCKS = 128;

int64_t plan_blocks(int64_t n)
{
    if (n <= PLAN_ONE_BLOCK) return 1;
    return std::min(PLAN_MAX_BLOCKS, (n + PLAN_ENTRIES_PER_BLOCK - 1) / PLAN_ENTRIES_PER_BLOCK);
}

// Warps that place entries: each holds one counter per expert in at most 128 KiB of shared memory.
int plan_warps(int32_t n_experts) { return std::min(povs::PLAN_WARPS, 32768 / n_experts); }

int check_plan(int64_t n_entries, int32_t n_experts)
{
    if (n_entries < 0) return fail(POVS_ERR_INVALID_ARGUMENT, "n_entries must not be negative");
    if (n_experts < 1) return fail(POVS_ERR_INVALID_ARGUMENT, "n_experts (%d) must be at least 1", n_experts);
    if (n_experts > POVS_MAX_PLAN_EXPERTS)
        return fail(POVS_ERR_UNSUPPORTED, "%d experts exceed the limit of %d", n_experts, POVS_MAX_PLAN_EXPERTS);
    if (n_entries > INT32_MAX) return fail(POVS_ERR_UNSUPPORTED, "n_entries must be below 2^31");
    return POVS_OK;
}

} // namespace

extern "C" int64_t povs_plan_rows_workspace_v1(int64_t n_entries, int32_t n_experts)
{
    g_err[0] = '\0';
    const int r = check_plan(n_entries, n_experts);
    if (r != POVS_OK) return r;
    const int64_t blocks = plan_blocks(n_entries);
    return blocks == 1 ? 0 : blocks * n_experts * static_cast<int64_t>(sizeof(int32_t));
}

extern "C" int povs_plan_rows_v1(const void* experts, int32_t id_bytes, int64_t n_entries, int32_t n_experts,
                                 int32_t* slots, int32_t* sources, int32_t* offsets, void* workspace,
                                 int64_t workspace_bytes, int32_t device, void* stream)
{
    g_err[0] = '\0';
    int r = check_plan(n_entries, n_experts);
    if (r != POVS_OK) return r;
    if (id_bytes != 4 && id_bytes != 8) return fail(POVS_ERR_INVALID_ARGUMENT, "id_bytes (%d) must be 4 or 8", id_bytes);
    if (offsets == nullptr || (n_entries > 0 && (experts == nullptr || slots == nullptr || sources == nullptr)))
        return fail(POVS_ERR_INVALID_ARGUMENT, "experts, slots, sources and offsets must not be NULL");
    const int64_t blocks = plan_blocks(n_entries);
    if (blocks > 1) {
        const int64_t need = blocks * n_experts * static_cast<int64_t>(sizeof(int32_t));
        if (workspace == nullptr || workspace_bytes < need)
            return fail(POVS_ERR_INVALID_ARGUMENT, "the workspace must hold %lld bytes", static_cast<long long>(need));
    }
    r = check_aligned({{"experts", experts, id_bytes}, {"slots", slots, 4}, {"sources", sources, 4}, {"offsets", offsets, 4},
                       {"workspace", blocks > 1 ? workspace : nullptr, 4}});
    if (r != POVS_OK) return r;
    DeviceGuard dg;
    int sms = 0;
    r = enter(dg, device, &sms);
    if (r != POVS_OK) return r;
    povs::PlanRowsParams p{};
    p.experts = experts;
    p.id_bytes = id_bytes;
    p.n_experts = n_experts;
    p.n = n_entries;
    p.chunk = (n_entries + blocks - 1) / blocks;
    p.counts = static_cast<int32_t*>(workspace);
    p.slots = slots;
    p.sources = sources;
    p.offsets = offsets;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const unsigned grid = static_cast<unsigned>(blocks);
    if (blocks > 1) povs::povs_plan_count_kernel<<<grid, povs::PLAN_THREADS, sizeof(int32_t) * n_experts, s>>>(p);
    const int warps = plan_warps(n_experts);
    const size_t smem = sizeof(int32_t) * static_cast<size_t>(n_experts) * (warps + 1);
    if (smem > 48 * 1024)
        POVS_CUDA_TRY(cudaFuncSetAttribute(reinterpret_cast<const void*>(povs::povs_plan_place_kernel),
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    povs::povs_plan_place_kernel<<<grid, povs::PLAN_THREADS, smem, s>>>(p, warps);
    return launched("plan kernels");
}

extern "C" int povs_dispatch_rows_v1(const void* data, int64_t rows, int64_t row_bytes, int64_t row_stride,
                                     const int32_t* slots, int32_t top_k, const int32_t* used, void* out,
                                     int64_t n_slots, int32_t device, void* stream)
{
    g_err[0] = '\0';
    int r = check_rows(rows, top_k, n_slots);
    if (r != POVS_OK) return r;
    if (row_bytes < 0 || row_stride < 0) return fail(POVS_ERR_INVALID_ARGUMENT, "row_bytes and row_stride must not be negative");
    if (row_bytes == 0 || n_slots == 0) return POVS_OK;
    if (out == nullptr || used == nullptr || (rows > 0 && (data == nullptr || slots == nullptr)))
        return fail(POVS_ERR_INVALID_ARGUMENT, "data, slots, used and out must not be NULL");
    r = check_aligned({{"slots", slots, 4}, {"used", used, 4}});
    if (r != POVS_OK) return r;
    DeviceGuard dg;
    int sms = 0;
    r = enter(dg, device, &sms);
    if (r != POVS_OK) return r;
    povs::DispatchParams p{};
    p.data = static_cast<const uint8_t*>(data);
    p.out = static_cast<uint8_t*>(out);
    p.slots = slots;
    p.used = used;
    p.rows = rows;
    p.row_bytes = row_bytes;
    p.row_stride = row_stride;
    p.n_slots = n_slots;
    p.top_k = top_k;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (common_alignment({address(data), address(out), static_cast<uint64_t>(row_bytes), static_cast<uint64_t>(row_stride)})) {
    case 16: launch_dispatch<16>(p, sms, s); break;
    case 8: launch_dispatch<8>(p, sms, s); break;
    case 4: launch_dispatch<4>(p, sms, s); break;
    case 2: launch_dispatch<2>(p, sms, s); break;
    default: launch_dispatch<1>(p, sms, s); break;
    }
    return launched("dispatch kernel");
}

extern "C" int povs_combine_rows_v1(const void* data, int32_t dtype, int64_t n_slots, int64_t width,
                                    int64_t data_stride, const int32_t* slots, int64_t rows, int32_t top_k,
                                    const float* weights, void* out, int32_t device, void* stream)
{
    g_err[0] = '\0';
    povs::CombineParams p{};
    p.data = data;
    p.slots = slots;
    p.weights = weights;
    p.out = out;
    p.rows = rows;
    p.width = width;
    p.data_stride = data_stride;
    p.n_slots = n_slots;
    p.top_k = top_k;
    int r = check_combine(p, dtype);
    if (r != POVS_OK) return r;
    if (rows == 0 || width == 0) return POVS_OK;
    if (out == nullptr || (n_slots > 0 && data == nullptr))
        return fail(POVS_ERR_INVALID_ARGUMENT, "data and out must not be NULL");
    const int64_t size = element_bytes(dtype);
    r = check_aligned({{"data", data, size}, {"slots", slots, 4}, {"weights", weights, 4}, {"out", out, size}});
    if (r != POVS_OK) return r;
    DeviceGuard dg;
    int sms = 0;
    r = enter(dg, device, &sms);
    if (r != POVS_OK) return r;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int align = common_alignment({address(data), address(out), static_cast<uint64_t>(width * size), static_cast<uint64_t>(data_stride * size)});
    if (dtype == POVS_FLOAT32) launch_combine_by<float>(align, p, sms, s);
    else if (dtype == POVS_BFLOAT16) launch_combine_by<__nv_bfloat16>(align, p, sms, s);
    else launch_combine_by<__half>(align, p, sms, s);
    return launched("combine kernel");
}

extern "C" int povs_combine_backward_v1(const void* grad, const void* data, int32_t dtype, int64_t n_slots,
                                        int64_t width, int64_t data_stride, const int32_t* slots, int64_t rows,
                                        int32_t top_k, const float* weights, const int32_t* used, void* grad_data,
                                        float* grad_weights, int32_t device, void* stream)
{
    g_err[0] = '\0';
    povs::CombineParams p{};
    p.data = data;
    p.slots = slots;
    p.weights = weights;
    p.rows = rows;
    p.width = width;
    p.data_stride = data_stride;
    p.n_slots = n_slots;
    p.top_k = top_k;
    p.used = used;
    p.grad = grad;
    p.grad_data = n_slots > 0 && width > 0 ? grad_data : nullptr;
    p.grad_weights = grad_weights;
    int r = check_combine(p, dtype);
    if (r != POVS_OK) return r;
    if (grad_data != nullptr && used == nullptr) return fail(POVS_ERR_INVALID_ARGUMENT, "grad_data needs used");
    if (p.grad_data == nullptr && (grad_weights == nullptr || rows == 0)) return POVS_OK;
    if ((rows > 0 && width > 0 && grad == nullptr) || (grad_weights != nullptr && n_slots > 0 && width > 0 && data == nullptr))
        return fail(POVS_ERR_INVALID_ARGUMENT, "grad and data must not be NULL");
    const int64_t size = element_bytes(dtype);
    r = check_aligned({{"grad", grad, size}, {"data", data, size}, {"slots", slots, 4}, {"weights", weights, 4}, {"used", used, 4},
                       {"grad_data", grad_data, size}, {"grad_weights", grad_weights, 4}});
    if (r != POVS_OK) return r;
    DeviceGuard dg;
    int sms = 0;
    r = enter(dg, device, &sms);
    if (r != POVS_OK) return r;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int align = common_alignment({address(grad), address(grad_weights != nullptr ? data : nullptr), address(p.grad_data),
                                        static_cast<uint64_t>(width * size), static_cast<uint64_t>(grad_weights != nullptr ? data_stride * size : 0)});
    if (dtype == POVS_FLOAT32) launch_combine_backward_by<float>(align, p, sms, s);
    else if (dtype == POVS_BFLOAT16) launch_combine_backward_by<__nv_bfloat16>(align, p, sms, s);
    else launch_combine_backward_by<__half>(align, p, sms, s);
    return launched("combine backward kernel");
}
