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
// Up to kBatch tensors travel in a launch's arguments, whatever their types; tiles are numbered through the tensors and
// a workgroup finds its tensor and its types there.  The second pass goes through the gradients backwards, from what the
// first one read last, and both read and write past the caches (non-temporal).
// Measured on 45 fp32 tensors of 1.01 B elements into bf16: norm 0.59 ms (6.9 TB/s; 0.66 ms with temporal loads, 0.66
// with half the tile), scaling 0.91 ms (6.7 TB/s; 0.95 with one tile to an XCD in turn, 0.98 with three vectors to a
// lane); 202 M bf16 elements 64 + 128 us.  Leaving the first pass's last 128 to 240 MiB to the cache changed nothing, runs
// of tiles on one XCD made the norm pass slower (0.61 ms).
#include "bmt_vec.h"
#include "../../include/bmt_hip.h"

#include <algorithm>
#include <new>
#include <utility>
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
    uint8_t types[kBatch];               // src_type + 4 * dst_type
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

// The sum, or the larger one; a NaN stays.
template <bool MAX>
__device__ __forceinline__ double join(double a, double b) {
    return MAX ? a != a ? a : b > a || b != b ? b : a : a + b;
}
// Over a workgroup of kThreads, in a fixed order; thread 0 has it.
template <bool MAX>
__device__ __forceinline__ double workgroup_join(double acc) {
    __shared__ double slots[kThreads / kWave];
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) acc = join<MAX>(acc, __shfl_xor(acc, off, kWave));
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = acc;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int k = 1; k < kThreads / kWave; k++) acc = join<MAX>(acc, slots[k]);
    return acc;
}

// The tensor's tile into the thread's sum, or largest magnitude (NaN where there is one).
template <typename T, bool MAX>
__device__ __forceinline__ double norm_tile(const void *src, int64_t n, uint32_t tile) {
    typedef Elem<T> E;
    constexpr int K = E::kVec;
    const typename E::Bits *g = (const typename E::Bits *)src;
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
    return MAX ? nan ? (double)__builtin_nanf("") : (double)top : acc;
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void grad_norm_kernel(Batch batch, double *__restrict__ partials) {
    const int which = find_tensor(batch, blockIdx.x);
    const uint32_t tile = blockIdx.x - batch.first[which];
    const int type = batch.types[which] & 3;
    double acc = type == kFp32   ? norm_tile<Single, MAX>(batch.src[which], batch.n[which], tile)
                 : type == kFp16 ? norm_tile<Half, MAX>(batch.src[which], batch.n[which], tile)
                                 : norm_tile<BFloat16, MAX>(batch.src[which], batch.n[which], tile);
    acc = workgroup_join<MAX>(acc);
    if (threadIdx.x == 0) partials[blockIdx.x] = acc;
}

// out: n / scale, then the factor c.
template <bool MAX>
__global__ __launch_bounds__(kThreads) void grad_norm_finish_kernel(const double *__restrict__ partials, int64_t count, double max_norm,
                                                                    double eps, double scale, float *__restrict__ out) {
    double acc = 0;
    for (int64_t i = threadIdx.x; i < count; i += kThreads) acc = join<MAX>(acc, partials[i]);
    acc = workgroup_join<MAX>(acc);
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

// The tensor's tile times f.
template <typename S, typename D>
__device__ __forceinline__ void scale_tile(const void *src, void *dst, int64_t n, int64_t number, float c, int32_t round_coef) {
    typedef Elem<S> E;
    constexpr int K = E::kVec;
    const typename E::Bits *g = (const typename E::Bits *)src;
    typename Elem<D>::Bits *o = (typename Elem<D>::Bits *)dst;
    const float f = !(c < 1.f) ? 1.f : round_coef ? E::get(E::put(c)) : c;
    constexpr int64_t kTile = (int64_t)kScaleThreads * kScaleUnroll;       // vectors
    const int64_t tile = (n + kTile * K - 1) / (kTile * K) - 1 - number;   // last tile first
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

template <typename S>
__device__ __forceinline__ void scale_tile_into(int dst_type, const void *src, void *dst, int64_t n, int64_t number, float c,
                                                int32_t round_coef) {
    if (dst_type == kFp32) scale_tile<S, Single>(src, dst, n, number, c, round_coef);
    else if (dst_type == kFp16) scale_tile<S, Half>(src, dst, n, number, c, round_coef);
    else scale_tile<S, BFloat16>(src, dst, n, number, c, round_coef);
}

// The factor a tensor is multiplied by: c, or c rounded to the tensor's type (what torch's multiplication of a 16-bit
// tensor by a 0-dim fp32 tensor does); 1 where c is not below 1, a NaN among them.  TYPES: those of all tensors of the
// launch, or kMixed (one launch instead of up to nine: a call on 36 small tensors of three types into three types 16 us
// instead of 56; where all are alike the types are the compiler's, 1.01 B fp32 elements into bf16 0.91 ms instead of 0.94).
constexpr int kMixed = -1;
template <int TYPES>
__global__ __launch_bounds__(kScaleThreads) void grad_scale_kernel(Batch batch, const float *__restrict__ coef, int32_t round_coef) {
    const float c = coef[0];
    const uint32_t unit = xcd_run<kScaleRun>(blockIdx.x, gridDim.x);
    const int which = find_tensor(batch, unit);
    const void *src = batch.src[which];
    void *dst = batch.dst[which];
    if (!(c < 1.f) && src == (const void *)dst) return;
    const int types = TYPES == kMixed ? batch.types[which] : TYPES, src_type = types & 3, dst_type = types >> 2;
    const int64_t n = batch.n[which], number = unit - batch.first[which];
    if (src_type == kFp32) scale_tile_into<Single>(dst_type, src, dst, n, number, c, round_coef);
    else if (src_type == kFp16) scale_tile_into<Half>(dst_type, src, dst, n, number, c, round_coef);
    else scale_tile_into<BFloat16>(dst_type, src, dst, n, number, c, round_coef);
}

template <int... TYPES>
void scale_launch(std::integer_sequence<int, TYPES...>, const Batch &b, uint32_t tiles, int types, const float *coef, int32_t round_coef,
                  hipStream_t s) {
    auto one = [&](auto t) {
        constexpr int kTypes = decltype(t)::value;
        if (types != kTypes) return false;
        hipLaunchKernelGGL((grad_scale_kernel<kTypes>), dim3(tiles), dim3(kScaleThreads), 0, s, b, coef, round_coef);
        return true;
    };
    (one(std::integral_constant<int, TYPES>()) || ...);
}

uintptr_t size_of(int32_t type) { return type == kFp32 ? 4 : 2; }
bool known(int32_t type) { return type == kFp32 || type == kFp16 || type == kBf16; }
// Tiles of `vectors` 16-byte vectors.
int64_t tiles_of(const bmt_clip_tensor &t, int64_t vectors) {
    const int64_t tile = vectors * 16 / (int64_t)size_of(t.src_type);
    return t.n <= 0 ? 0 : (t.n + tile - 1) / tile;
}
constexpr int64_t kNormTile = (int64_t)kThreads * kUnroll, kScaleTile = (int64_t)kScaleThreads * kScaleUnroll;

// Calls launch(batch, tiles, the types of all its tensors or kMixed) for batches of the tensors, in order or backwards.
template <typename F>
hipError_t in_batches(int32_t count, const bmt_clip_tensor *tensors, int64_t vectors, int threads, bool backwards, F launch) {
    Batch b;
    int held = 0, types = kMixed;
    int64_t tiles = 0;
    auto flush = [&]() -> hipError_t {
        if (!held) return hipSuccess;
        for (int k = held; k < kBatch; k++) b.src[k] = nullptr, b.dst[k] = nullptr, b.n[k] = 0, b.first[k] = 0xFFFFFFFFu, b.types[k] = 0;
        launch(b, (uint32_t)tiles, types);
        held = 0, tiles = 0;
        return hipGetLastError();
    };
    for (int32_t j = 0; j < count; j++) {
        const bmt_clip_tensor &t = tensors[backwards ? count - 1 - j : j];
        if (t.n <= 0) continue;
        const int64_t more = tiles_of(t, vectors);
        if (held == kBatch || !launch_fits(tiles + more, threads)) {
            const hipError_t e = flush();
            if (e != hipSuccess) return e;
        }
        b.src[held] = t.src, b.dst[held] = t.dst, b.n[held] = t.n, b.first[held] = (uint32_t)tiles;
        b.types[held] = (uint8_t)(t.src_type + 4 * (t.dst_type & 3));
        types = held == 0 || types == b.types[held] ? b.types[held] : kMixed;
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
    hipError_t e = in_batches(count, tensors, kNormTile, kThreads, false, [&](const Batch &b, uint32_t tiles, int) {
        if (use_max) hipLaunchKernelGGL((grad_norm_kernel<true>), dim3(tiles), dim3(kThreads), 0, s, b, partials + used);
        else hipLaunchKernelGGL((grad_norm_kernel<false>), dim3(tiles), dim3(kThreads), 0, s, b, partials + used);
        used += tiles;
    });
    if (e != hipSuccess) return fail((int)e, who, e);
    if (use_max)
        hipLaunchKernelGGL((grad_norm_finish_kernel<true>), dim3(1), dim3(kThreads), 0, s, partials, used, max_norm, eps, scale,
                           (float *)out);
    else
        hipLaunchKernelGGL((grad_norm_finish_kernel<false>), dim3(1), dim3(kThreads), 0, s, partials, used, max_norm, eps, scale,
                           (float *)out);
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
    const hipError_t e = in_batches(count, tensors, kScaleTile, kScaleThreads, true, [&](const Batch &b, uint32_t tiles, int types) {
        scale_launch(std::integer_sequence<int, kMixed, 0, 1, 2, 4, 5, 6, 8, 9, 10>(), b, tiles, types, (const float *)coef,
                     round_coef, s);
    });
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}
