// Global norm over a list of gradients and the clipped gradients, for gfx950.
//
//     n = (sum over tensors and elements of g^2)^(1/2)   or   max |g|
//     c = max_norm * scale / (n + eps)                        (gradients carry the loss scale `scale`; n / scale is reported)
//     out = c < 1 ? g c : g
// Two passes over the gradients (the norm has to be known before the first output) and one workgroup between them; the
// factor never leaves the device.  Inputs are fp32, fp16 or bf16 and outputs any of the three: fp32 accumulators go
// straight into the 16-bit gradients an optimizer step takes.  Bound by HBM: 2 x 4 B read and 2 written per element for
// fp32 to 16 bits, 2 x 2 and 2 for 16 bits.
//
// Squares are formed and added in 64 bits: an fp32 or bf16 gradient's square may lie outside fp32's range.  Partial
// sums, one to a tile, are added in a fixed order: equal inputs give equal bits.
// Up to kBatch tensors of one pair of types travel in a launch's arguments; tiles are numbered through the tensors and
// a workgroup finds its tensor there.  The second pass goes through the gradients backwards, from what the first one
// read last, and both read and write past the caches (non-temporal).
// Measured on 45 fp32 tensors of 1.01 B elements into bf16: norm 0.59 ms (6.9 TB/s; 0.66 ms with temporal loads, 0.66
// with half the tile), scaling 0.91 ms (6.7 TB/s; 0.95 with one tile to an XCD in turn, 0.98 with three vectors to a
// lane); 202 M bf16 elements 64 + 128 us.  Leaving the first pass's last 128 to 240 MiB to the cache changed nothing, runs
// of tiles on one XCD made the norm pass slower (0.61 ms).
#include "bmt_vec.h"
#include "../../include/bmt_hip.h"

#include <algorithm>
#include <new>
#include <vector>

namespace bmt {
namespace {

constexpr int kThreads = 1024;           // norm pass: a tile is 8 vectors of 1,024 lanes, 128 KiB
constexpr int kUnroll = 8;
constexpr int kScaleThreads = 256;       // scaling pass: 2 vectors of 256 lanes, 8 KiB
constexpr int kScaleUnroll = 2;
constexpr uint32_t kScaleRun = 256;      // workgroups of consecutive tiles on one XCD
constexpr int kBatch = 96;

struct Batch {
    const void *src[kBatch];
    void *dst[kBatch];
    int64_t n[kBatch];
    uint32_t first[kBatch];              // number of a tensor's first tile; 0xFFFFFFFF behind the last tensor
};

// The tensor of tile `tile`: the last one that starts at or in front of it (a bisection over the arguments).
__device__ __forceinline__ int find_tensor(const Batch &b, uint32_t tile) {
    int low = 0, high = kBatch;          // first[low] <= tile < first[high]
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (b.first[mid] <= tile) low = mid;
        else high = mid;
    }
    return low;
}

template <bool MAX>
__device__ __forceinline__ void norm_add(double &acc, float &top, uint32_t &nan, float x) {
    if (MAX) {
        nan |= x != x ? 1u : 0u;
        top = fmaxf(top, fabsf(x));
    } else {
        acc = __builtin_fma((double)x, (double)x, acc);
    }
}

template <typename T, bool MAX>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(Batch batch, double *__restrict__ partials) {
    typedef Elem<T> E;
    constexpr int K = E::kVec;
    const int which = find_tensor(batch, blockIdx.x);
    const typename E::Bits *g = (const typename E::Bits *)batch.src[which];
    const int64_t n = batch.n[which];
    const uint32_t tile = blockIdx.x - batch.first[which];
    const int head = head_elements<T>(g, n < 64 ? (int)n : 64);
    const int64_t nvec = (n - head) / K;
    const u32x4 *body = (const u32x4 *)(g + head);
    const int64_t i0 = (int64_t)tile * (kThreads * kUnroll) + threadIdx.x;
    double acc = 0;
    float top = 0.f;
    uint32_t nan = 0;
    u32x4 w[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
        w[u] = u32x4{0u, 0u, 0u, 0u};
        if (i0 + u * kThreads < nvec) w[u] = __builtin_nontemporal_load(body + i0 + u * kThreads);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; u++) {
        float x[K];
        E::unpack(w[u], x);
#pragma unroll
        for (int k = 0; k < K; k++) norm_add<MAX>(acc, top, nan, x[k]);
    }
    if (tile == 0) {
        const int64_t tail_lo = head + nvec * K, edge = head + (n - tail_lo);
        if ((int64_t)threadIdx.x < edge)
            norm_add<MAX>(acc, top, nan, E::get(g[(int64_t)threadIdx.x < head ? (int64_t)threadIdx.x : tail_lo + threadIdx.x - head]));
    }
    if (MAX) acc = nan ? (double)__builtin_nanf("") : (double)top;
    __shared__ double slots[kThreads / kWave];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const double other = __shfl_xor(acc, off, kWave);
        acc = MAX ? (acc != acc ? acc : other > acc || other != other ? other : acc) : acc + other;
    }
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = acc;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kThreads / kWave; k++) {
            const double other = slots[k];
            acc = MAX ? (acc != acc ? acc : other > acc || other != other ? other : acc) : acc + other;
        }
        partials[blockIdx.x] = acc;
    }
}

// out: n / scale, then the factor c.
template <bool MAX>
__global__ __launch_bounds__(kThreads) void grad_norm_finish_kernel(const double *__restrict__ partials, int64_t count, double max_norm,
                                                                    double eps, double scale, float *__restrict__ out) {
    double acc = 0;
    for (int64_t i = threadIdx.x; i < count; i += kThreads) {
        const double other = partials[i];
        acc = MAX ? (acc != acc ? acc : other > acc || other != other ? other : acc) : acc + other;
    }
    __shared__ double lanes[kThreads];
    lanes[threadIdx.x] = acc;
    __syncthreads();
    for (int stride = kThreads / 2; stride > 0; stride >>= 1) {
        if ((int)threadIdx.x < stride) {
            const double other = lanes[threadIdx.x + stride];
            acc = MAX ? (acc != acc ? acc : other > acc || other != other ? other : acc) : acc + other;
            lanes[threadIdx.x] = acc;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        const double norm = MAX ? acc : sqrt(acc);
        out[0] = (float)(norm / scale);
        out[1] = (float)(max_norm * scale / (norm + eps));
    }
}

// K elements of type D, 8 or 16 bytes at a time, not kept in the cache.
template <typename D, int K>
__device__ __forceinline__ void store_past_cache(typename Elem<D>::Bits *to, const float *x) {
    if (sizeof(typename Elem<D>::Bits) * K == 8) {
        u32x2 w;
        w[0] = (uint32_t)Elem<D>::put(x[0]) | ((uint32_t)Elem<D>::put(x[1]) << 16);
        w[1] = (uint32_t)Elem<D>::put(x[2]) | ((uint32_t)Elem<D>::put(x[3]) << 16);
        __builtin_nontemporal_store(w, (u32x2_any2 *)to);
    } else {
#pragma unroll
        for (int k = 0; k < K; k += Elem<D>::kVec) __builtin_nontemporal_store(Elem<D>::pack(x + k), (typename Elem<D>::Vec *)(to + k));
    }
}

// The factor a tensor is multiplied by: c, or c rounded to the tensor's type (what torch's multiplication of a 16-bit
// tensor by a 0-dim fp32 tensor does); 1 where c is not below 1, a NaN among them.
template <typename S, typename D>
__global__ __launch_bounds__(kScaleThreads) void grad_scale_kernel(Batch batch, const float *__restrict__ coef, int32_t round_coef) {
    typedef Elem<S> E;
    constexpr int K = E::kVec;
    const float c = coef[0];
    const bool scales = c < 1.f;
    const uint32_t number = xcd_run<kScaleRun>(blockIdx.x, gridDim.x);
    const int which = find_tensor(batch, number);
    const typename E::Bits *g = (const typename E::Bits *)batch.src[which];
    typename Elem<D>::Bits *o = (typename Elem<D>::Bits *)batch.dst[which];
    if (!scales && (const void *)g == (const void *)o) return;
    const float f = !scales ? 1.f : round_coef ? E::get(E::put(c)) : c;
    const int64_t n = batch.n[which];
    constexpr int64_t kTile = (int64_t)kScaleThreads * kScaleUnroll;       // vectors
    const int64_t tile = (n + kTile * K - 1) / (kTile * K) - 1 - (number - batch.first[which]);      // last tile first
    const int head = head_elements<S>(g, n < 64 ? (int)n : 64);
    const int64_t nvec = (n - head) / K;
    const u32x4 *body = (const u32x4 *)(g + head);
    const int64_t i0 = tile * kTile + threadIdx.x;
    u32x4 w[kScaleUnroll];
#pragma unroll
    for (int u = 0; u < kScaleUnroll; u++)
        if (i0 + u * kScaleThreads < nvec) w[u] = __builtin_nontemporal_load(body + i0 + u * kScaleThreads);
#pragma unroll
    for (int u = 0; u < kScaleUnroll; u++) {
        const int64_t i = i0 + u * kScaleThreads;
        if (i >= nvec) break;
        float x[K];
        E::unpack(w[u], x);
#pragma unroll
        for (int k = 0; k < K; k++) x[k] = x[k] * f;
        store_past_cache<D, K>(o + head + i * K, x);
    }
    if (tile == 0) {
        const int64_t tail_lo = head + nvec * K, edge = head + (n - tail_lo);
        if ((int64_t)threadIdx.x < edge) {
            const int64_t j = (int64_t)threadIdx.x < head ? (int64_t)threadIdx.x : tail_lo + threadIdx.x - head;
            o[j] = Elem<D>::put(E::get(g[j]) * f);
        }
    }
}

uintptr_t size_of(int32_t type) { return type == kFp32 ? 4 : 2; }
bool known(int32_t type) { return type == kFp32 || type == kFp16 || type == kBf16; }
// Tiles of `vectors` 16-byte vectors.
int64_t tiles_of(const bmt_clip_tensor &t, int64_t vectors) {
    const int64_t tile = vectors * 16 / (int64_t)size_of(t.src_type);
    return t.n <= 0 ? 0 : (t.n + tile - 1) / tile;
}
constexpr int64_t kNormTile = (int64_t)kThreads * kUnroll, kScaleTile = (int64_t)kScaleThreads * kScaleUnroll;

// Calls launch(batch, tiles) for batches of the tensors with these types (dst_type < 0: any), in order or backwards.
template <typename F>
hipError_t in_batches(int32_t count, const bmt_clip_tensor *tensors, int32_t src_type, int32_t dst_type, int64_t vectors, int threads,
                      bool backwards, F launch) {
    Batch b;
    int held = 0;
    int64_t tiles = 0;
    auto flush = [&]() -> hipError_t {
        if (!held) return hipSuccess;
        for (int k = held; k < kBatch; k++) b.src[k] = nullptr, b.dst[k] = nullptr, b.n[k] = 0, b.first[k] = 0xFFFFFFFFu;
        launch(b, (uint32_t)tiles);
        held = 0, tiles = 0;
        return hipGetLastError();
    };
    for (int32_t j = 0; j < count; j++) {
        const bmt_clip_tensor &t = tensors[backwards ? count - 1 - j : j];
        if (t.n <= 0 || t.src_type != src_type || (dst_type >= 0 && t.dst_type != dst_type)) continue;
        const int64_t more = tiles_of(t, vectors);
        if (held == kBatch || !launch_fits(tiles + more, threads)) {
            const hipError_t e = flush();
            if (e != hipSuccess) return e;
        }
        b.src[held] = t.src, b.dst[held] = t.dst, b.n[held] = t.n, b.first[held] = (uint32_t)tiles;
        tiles += more;
        held++;
    }
    return flush();
}

const char *check_table(int32_t count, const bmt_clip_tensor *tensors, bool with_dst) {
    if (count > 0 && !tensors) return "null tensor table";
    for (int32_t k = 0; k < count; k++) {
        const bmt_clip_tensor &t = tensors[k];
        if (t.n <= 0) continue;
        if (!known(t.src_type) || (with_dst && !known(t.dst_type))) return "unknown type code";
        if (!t.src || (with_dst && !t.dst)) return "null pointer";
        if ((uintptr_t)t.src % size_of(t.src_type) || (with_dst && (uintptr_t)t.dst % size_of(t.dst_type)))
            return "tensor is not aligned to its elements";
        if (!launch_fits(tiles_of(t, kScaleTile), kScaleThreads)) return "tensor too large for one launch";
    }
    return nullptr;
}

// No output may share memory with another entry's input or output, nor with its own input other than as that input
// itself (same address, same type): workgroups write outputs while others still read inputs.
const char *check_overlap(int32_t count, const bmt_clip_tensor *tensors) {
    struct Span {
        uintptr_t begin, end;
        bool out;
    };
    // inputs and outputs apart: gradients are often allocated in order, as are the places they go to
    std::vector<Span> spans, outs;
    spans.reserve(2 * (size_t)count), outs.reserve((size_t)count);
    for (int32_t k = 0; k < count; k++) {
        const bmt_clip_tensor &t = tensors[k];
        if (t.n <= 0) continue;
        const uintptr_t s = (uintptr_t)t.src, d = (uintptr_t)t.dst;
        if (s != d || t.src_type != t.dst_type) spans.push_back({s, s + (uintptr_t)t.n * size_of(t.src_type), false});
        outs.push_back({d, d + (uintptr_t)t.n * size_of(t.dst_type), true});
    }
    auto before = [](const Span &a, const Span &b) { return a.begin < b.begin; };
    if (!std::is_sorted(spans.begin(), spans.end(), before)) std::sort(spans.begin(), spans.end(), before);
    if (!std::is_sorted(outs.begin(), outs.end(), before)) std::sort(outs.begin(), outs.end(), before);
    const size_t inputs = spans.size();
    spans.insert(spans.end(), outs.begin(), outs.end());
    std::inplace_merge(spans.begin(), spans.begin() + (std::ptrdiff_t)inputs, spans.end(), before);
    uintptr_t out_end = 0, any_end = 0;                  // how far outputs / anything in front of here reach
    for (const Span &s : spans) {
        if (s.begin < out_end || (s.out && s.begin < any_end)) return "an output shares memory with another tensor of the call";
        if (s.out) out_end = std::max(out_end, s.end);
        any_end = std::max(any_end, s.end);
    }
    return nullptr;
}

template <typename S>
hipError_t norm_passes(int32_t count, const bmt_clip_tensor *tensors, int32_t type, bool max, double *partials, int64_t *used,
                       hipStream_t s) {
    return in_batches(count, tensors, type, -1, kNormTile, kThreads, false, [&](const Batch &b, uint32_t tiles) {
        if (max) hipLaunchKernelGGL((grad_norm_kernel<S, true>), dim3(tiles), dim3(kThreads), 0, s, b, partials + *used);
        else hipLaunchKernelGGL((grad_norm_kernel<S, false>), dim3(tiles), dim3(kThreads), 0, s, b, partials + *used);
        *used += tiles;
    });
}

template <typename S, typename D>
hipError_t scale_passes(int32_t count, const bmt_clip_tensor *tensors, int32_t src_type, int32_t dst_type, const float *coef,
                        int32_t round_coef, hipStream_t s) {
    return in_batches(count, tensors, src_type, dst_type, kScaleTile, kScaleThreads, true, [&](const Batch &b, uint32_t tiles) {
        hipLaunchKernelGGL((grad_scale_kernel<S, D>), dim3(tiles), dim3(kScaleThreads), 0, s, b, coef, round_coef);
    });
}
template <typename S>
hipError_t scale_from(int32_t count, const bmt_clip_tensor *tensors, int32_t src_type, const float *coef, int32_t round_coef, hipStream_t s) {
    hipError_t e = scale_passes<S, Single>(count, tensors, src_type, kFp32, coef, round_coef, s);
    if (e == hipSuccess) e = scale_passes<S, Half>(count, tensors, src_type, kFp16, coef, round_coef, s);
    if (e == hipSuccess) e = scale_passes<S, BFloat16>(count, tensors, src_type, kBf16, coef, round_coef, s);
    return e;
}

}  // namespace
}  // namespace bmt

extern "C" int64_t grad_norm_workspace_doubles(int32_t count, const bmt_clip_tensor *tensors) {
    int64_t tiles = 1;
    if (tensors)
        for (int32_t k = 0; k < count; k++) tiles += bmt::tiles_of(tensors[k], bmt::kNormTile);
    return tiles;
}

extern "C" int grad_norm_multi_launcher(int32_t count, const bmt_clip_tensor *tensors, int32_t use_max, double max_norm, double eps,
                                        double scale, void *workspace, void *out, void *stream) {
    using namespace bmt;
    const char *who = "grad_norm_multi_launcher";
    if (const char *why = check_table(count, tensors, false)) return refuse(who, why);
    if (!workspace || !out) return refuse(who, "null pointer");
    if ((uintptr_t)workspace % 8 || (uintptr_t)out % 4) return refuse(who, "misaligned output");
    if (!(scale > 0)) return refuse(who, "scale must be positive");
    hipStream_t s = (hipStream_t)stream;
    double *partials = (double *)workspace;
    int64_t used = 0;
    hipError_t e = norm_passes<Single>(count, tensors, kFp32, use_max != 0, partials, &used, s);
    if (e == hipSuccess) e = norm_passes<Half>(count, tensors, kFp16, use_max != 0, partials, &used, s);
    if (e == hipSuccess) e = norm_passes<BFloat16>(count, tensors, kBf16, use_max != 0, partials, &used, s);
    if (e != hipSuccess) return fail((int)e, who, e);
    if (use_max)
        hipLaunchKernelGGL((grad_norm_finish_kernel<true>), dim3(1), dim3(kThreads), 0, s, partials, used, max_norm, eps, scale, (float *)out);
    else
        hipLaunchKernelGGL((grad_norm_finish_kernel<false>), dim3(1), dim3(kThreads), 0, s, partials, used, max_norm, eps, scale, (float *)out);
    e = hipGetLastError();
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}

extern "C" int grad_scale_multi_launcher(int32_t count, const bmt_clip_tensor *tensors, const void *coef, int32_t round_coef,
                                         void *stream) {
    using namespace bmt;
    const char *who = "grad_scale_multi_launcher";
    if (count <= 0) return 0;
    if (const char *why = check_table(count, tensors, true)) return refuse(who, why);
    if (!coef) return refuse(who, "null pointer");
    if ((uintptr_t)coef % 4) return refuse(who, "misaligned coefficient");
    try {
        if (const char *why = check_overlap(count, tensors)) return refuse(who, why);
    } catch (const std::bad_alloc &) {
        return refuse(who, "out of host memory");
    }
    hipStream_t s = (hipStream_t)stream;
    hipError_t e = scale_from<BFloat16>(count, tensors, kBf16, (const float *)coef, round_coef, s);     // backwards here too
    if (e == hipSuccess) e = scale_from<Half>(count, tensors, kFp16, (const float *)coef, round_coef, s);
    if (e == hipSuccess) e = scale_from<Single>(count, tensors, kFp32, (const float *)coef, round_coef, s);
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}
