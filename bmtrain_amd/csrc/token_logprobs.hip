// Log-probabilities (and entropies) of given tokens under logits, and the logits' gradient, for gfx950.
//
// Row r of the logits holds x_0 .. x_{V-1}; with temperature T, z_j = (x_j - max x) / T and L = log sum_j e^{z_j}:
//     logprob = z_target - L                 entropy H = L - (sum_j e^{z_j} z_j) / (sum_j e^{z_j})
// and with upstream gradients g (of logprob) and h (of entropy), p_j = e^{z_j - L}:
//     dx_j = ( g (1[j = target] - p_j) - h p_j (z_j - L + H) ) / T
// The softmax is not stored: the forward pass reads the logits once and keeps {max, L, H} per row; the backward pass
// reads the logits once more and writes the gradient.  Both are bound by HBM (2 or 4 bytes per element read, and as
// many written on the way back).
//
// The target is left out of the running sums and joins at the end: where it is the largest logit, logprob =
// -log(1 + sum_{j != target} e^{z_j}) keeps its digits however near to 0 it is (as 1 - p does in the gradient), which a sum
// of everything rounded at 1 would not.
// (x_j - max) is formed before it is scaled: it is exact for neighbouring values, so rows of large magnitude lose
// nothing, and a row of the type's lowest value gives z = 0 instead of inf - inf.  All sums and exponents are fp32; the
// gradient is rounded once, to the logits' type.
//
// A row is a workgroup's, or a wave's where rows are short.  Vectors are 16 bytes from the row's first 16-byte boundary,
// the few elements in front of it and behind the last vector go one to a lane.
#include "bmt_host.h"
#include "bmt_vec.h"
#include "../../include/bmt_hip.h"

namespace bmt {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// exponent behind which a probability is 0 in fp32 (the smallest subnormal is 2^-149): keeps 0 * -inf out of the entropy's
// sums and gradients
constexpr float kFar = -1000.f;

struct RowStats {       // what the backward pass needs of a row
    float max, log_sum, entropy, unused;
};

struct LogitRows {      // row r starts at element (r / inner) * outer_stride + (r % inner) * inner_stride
    const void *x;
    int64_t outer_stride, inner_stride;
    int32_t rows, inner, n;
    __device__ __forceinline__ int64_t start(int32_t r) const {
        if (inner >= rows) return (int64_t)r * inner_stride;
        const int32_t o = r / inner;
        return (int64_t)o * outer_stride + (int64_t)(r - o * inner) * inner_stride;
    }
};

struct Targets {
    const void *t;
    int32_t is_64;
    int64_t ignore;
    __device__ __forceinline__ int64_t at(int32_t r) const {
        return is_64 ? ((const int64_t *)t)[r] : (int64_t)((const int32_t *)t)[r];
    }
};

template <bool PAST>
__device__ __forceinline__ u32x4 load_vector(const u32x4 *p) {
    return PAST ? __builtin_nontemporal_load(p) : *p;
}

// Running maximum m, s = sum 2^z and w = sum 2^z z with z = (x - m) * c in units of log 2.
struct Online {
    float m, s, w;
};
template <bool ENTROPY>
__device__ __forceinline__ void online_join(Online &a, float m, float s, float w, float c) {
    const float top = fmaxf(a.m, m);
    const float da = (a.m - top) * c, db = (m - top) * c;
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    if (ENTROPY) {      // the sums move by the shift of z: sum 2^(z+d) (z+d)
        const float wa = __builtin_fmaf(fmaxf(da, kFar), a.s, a.w), wb = __builtin_fmaf(fmaxf(db, kFar), s, w);
        a.w = wa * fa + wb * fb;
    }
    a.s = a.s * fa + s * fb;
    a.m = top;
}

// Element `at` of the vector becomes -inf.  And-or masks on whole words: written as a choice of elements it becomes an
// indexed store to memory, which costs the kernel two fifths of its speed.
template <typename T>
__device__ __forceinline__ void leave_out(u32x4 &w, int at) {
    constexpr int kPerWord = Elem<T>::kVec / 4;
    const uint32_t shift = kPerWord == 2 ? 16u * (uint32_t)(at & 1) : 0u;
    const uint32_t gone = (kPerWord == 2 ? 0xFFFFu : 0xFFFFFFFFu) << shift, put = (uint32_t)Elem<T>::put(-INFINITY) << shift;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t here = k == at / kPerWord ? 0xFFFFFFFFu : 0u;
        w[k] = (w[k] & ~(gone & here)) | (put & here);
    }
}

// K values x[0..K) into the running sums.
template <bool ENTROPY, int K>
__device__ __forceinline__ void online_add(Online &a, const float *x, float c) {
    float top = x[0];
#pragma unroll
    for (int k = 1; k < K; k++) top = fmaxf(top, x[k]);
    top = fmaxf(a.m, top);
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const float z = (x[k] - top) * c;
        const float e = __builtin_amdgcn_exp2f(z);
        s += e;
        if (ENTROPY) w = __builtin_fmaf(e, fmaxf(z, kFar), w);
    }
    const float d = (a.m - top) * c;
    const float f = __builtin_amdgcn_exp2f(d);
    if (ENTROPY) a.w = __builtin_fmaf(__builtin_fmaf(fmaxf(d, kFar), a.s, a.w), f, w);
    a.s = __builtin_fmaf(a.s, f, s);
    a.m = top;
}

// ROW: threads to a row (64: the workgroup's four waves take a row each); UNROLL: vectors of a lane in flight; PAST: the
// logits are read past the caches.
template <typename T, int ROW, int UNROLL, bool ENTROPY, bool PAST>
__global__ __launch_bounds__(ROW < 256 ? 256 : ROW) void token_logprobs_kernel(
    LogitRows in, Targets target, float inv_t, float *__restrict__ logprob, float *__restrict__ entropy,
    RowStats *__restrict__ stats) {
    typedef Elem<T> E;
    constexpr int PER = ROW < 256 ? 256 / ROW : 1;      // rows of a workgroup
    const int lane = threadIdx.x % ROW;
    const int32_t r = (int32_t)(blockIdx.x * PER + threadIdx.x / ROW);
    if (PER > 1 && r >= in.rows) return;
    const int64_t t = target.at(r);
    if (t == target.ignore) {
        if (lane == 0) {
            logprob[r] = 0.f;
            if (ENTROPY) entropy[r] = 0.f;
        }
        return;
    }
    const typename E::Bits *x = (const typename E::Bits *)in.x + in.start(r);
    const int n = in.n;
    const int head = head_elements<T>(x, n);
    const int nvec = (n - head) / E::kVec;
    const u32x4 *body = (const u32x4 *)(x + head);
    const float c = inv_t * kLog2e;
    constexpr int K = E::kVec;
    const bool inside = (uint64_t)t < (uint64_t)n;
    float xt = 0.f;
    if (lane == 0 && inside) xt = E::get(x[t]);
    // the vector that holds the target, in the lane that reads it, and the target's place in it; none in every other lane
    const int body_t = inside ? (int)t - head : -1;
    const int target_vec = body_t >= 0 && body_t / K < nvec && body_t / K % ROW == lane ? body_t / K : INT32_MIN, target_at = body_t % K;

    Online a = {-__FLT_MAX__, 0.f, 0.f};
    int i = lane;
    for (; i + (UNROLL - 1) * ROW < nvec; i += UNROLL * ROW) {
        u32x4 w[UNROLL];
        float v[UNROLL * K];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) w[u] = load_vector<PAST>(body + i + u * ROW);
        if ((uint32_t)target_vec - (uint32_t)i < (uint32_t)(UNROLL * ROW)) {
#pragma unroll
            for (int u = 0; u < UNROLL; u++)
                if (target_vec == i + u * ROW) leave_out<T>(w[u], target_at);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) E::unpack(w[u], v + u * K);
        online_add<ENTROPY, UNROLL * K>(a, v, c);
    }
    {       // fewer than UNROLL vectors are left to this lane: all are requested before the first is used
        u32x4 w[UNROLL - 1];
#pragma unroll
        for (int u = 0; u < UNROLL - 1; u++)
            if (i + u * ROW < nvec) w[u] = load_vector<PAST>(body + i + u * ROW);
        if ((uint32_t)target_vec - (uint32_t)i < (uint32_t)((UNROLL - 1) * ROW)) {
#pragma unroll
            for (int u = 0; u < UNROLL - 1; u++)
                if (target_vec == i + u * ROW) leave_out<T>(w[u], target_at);
        }
#pragma unroll
        for (int u = 0; u < UNROLL - 1; u++) {
            if (i + u * ROW >= nvec) break;
            float v[K];
            E::unpack(w[u], v);
            online_add<ENTROPY, K>(a, v, c);
        }
    }
    const int tail_lo = head + nvec * K, edge = head + (n - tail_lo);      // fewer than 2 * kVec elements
    if (lane < edge) {
        const int j = lane < head ? lane : tail_lo + (lane - head);
        const float v = j == t ? -INFINITY : E::get(x[j]);
        online_add<ENTROPY, 1>(a, &v, c);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
        online_join<ENTROPY>(a, __shfl_xor(a.m, off, kWave), __shfl_xor(a.s, off, kWave),
                             ENTROPY ? __shfl_xor(a.w, off, kWave) : 0.f, c);
    if (ROW > kWave) {
        constexpr int WAVES = ROW / kWave > 0 ? ROW / kWave : 1;
        __shared__ Online part[WAVES];
        if (lane % kWave == 0) part[lane / kWave] = a;
        __syncthreads();
        if (lane != 0) return;
        for (int k = 1; k < WAVES; k++) online_join<ENTROPY>(a, part[k].m, part[k].s, part[k].w, c);
    }
    if (lane == 0) {
        float log_sum, lp = __builtin_nanf("");
        if (inside && xt >= a.m) {                        // z = 0 for the target, all others together weigh `rest`
            const float d = (a.m - xt) * c, f = __builtin_amdgcn_exp2f(d), rest = a.s * f;
            if (ENTROPY) a.w = __builtin_fmaf(fmaxf(d, kFar), a.s, a.w) * f;
            a.m = xt, a.s = 1.f + rest;
            log_sum = log1pf(rest) + (xt - xt);           // NaN for an infinite logit, and with it the entropy and the gradient
            lp = 0.f - log_sum;
        } else {
            if (inside) online_join<ENTROPY>(a, xt, 1.f, 0.f, c);
            log_sum = logf(a.s);
            if (inside) lp = (xt - a.m) * inv_t - log_sum;
        }
        const float h = ENTROPY ? log_sum - kLn2 * (a.w / a.s) : 0.f;
        logprob[r] = lp;
        if (ENTROPY) entropy[r] = h;
        if (stats) stats[r] = RowStats{a.m, log_sum, h, 0.f};
    }
}

// A tile is UNROLL vectors of ROW lanes; tiles are numbered through the rows, and every XCD works on runs of consecutive
// ones, 32 workgroups of 256 or 8 of 1,024.
template <typename T, int ROW, int UNROLL, bool ENTROPY>
__global__ __launch_bounds__(ROW < 256 ? 256 : ROW) void token_logprobs_backward_kernel(
    LogitRows in, Targets target, float inv_t, const RowStats *__restrict__ stats, const float *__restrict__ grad_logprob,
    const float *__restrict__ grad_entropy, typename Elem<T>::Bits *__restrict__ grad, int32_t tiles) {
    typedef Elem<T> E;
    constexpr int PER = ROW < 256 ? 256 / ROW : 1, K = E::kVec;
    const int lane = threadIdx.x % ROW;
    const uint32_t unit = xcd_run<(ROW > 256 ? 8 : 32)>(blockIdx.x, gridDim.x) * PER + threadIdx.x / ROW;
    const int32_t r = (int32_t)(unit / (uint32_t)tiles), tile = (int32_t)(unit - (uint32_t)r * (uint32_t)tiles);
    if (PER > 1 && r >= in.rows) return;
    const int64_t t = target.at(r);
    const bool counted = t != target.ignore;
    const float g = grad_logprob && counted ? grad_logprob[r] : 0.f;
    const float h = ENTROPY && counted ? grad_entropy[r] : 0.f;
    const bool live = !(g == 0.f && h == 0.f);          // nothing comes back through this row: its logits are not read
    const typename E::Bits *x = (const typename E::Bits *)in.x + in.start(r);
    typename E::Bits *d = grad + (int64_t)r * in.n;
    const int n = in.n;
    const int head = head_elements<T>(x, n);
    const int nvec = (n - head) / K;
    const u32x4 *body = (const u32x4 *)(x + head);
    typename E::Vec *out = (typename E::Vec *)(d + head);
    const RowStats st = live ? stats[r] : RowStats{0.f, 0.f, 0.f, 0.f};
    // p = 2^y with y = (x - max) * c - log2(sum), log p = y ln 2:  dx = p (a + b y), a = -(g + h H) / T, b = -h ln 2 / T
    const float c = inv_t * kLog2e, log2_sum = st.log_sum * kLog2e;
    const float hot = g * inv_t, b = -h * inv_t * kLn2, a_rest = -h * st.entropy * inv_t, a = a_rest - hot;
    auto one = [&](float v) {
        const float y = __builtin_fmaf(v - st.max, c, -log2_sum);
        const float p = __builtin_amdgcn_exp2f(y);
        return p * (ENTROPY ? __builtin_fmaf(b, fmaxf(y, kFar), a) : a);
    };
    auto target_one = [&](float v) {                      // the same with (1 - p) g / T in the place of g / T - p g / T
        const float y = __builtin_fmaf(v - st.max, c, -log2_sum);
        return __builtin_fmaf(__builtin_amdgcn_exp2f(y), __builtin_fmaf(b, fmaxf(y, kFar), a_rest), -expm1f(y * kLn2) * hot);
    };
    const int i0 = tile * (ROW * UNROLL) + lane;
    u32x4 w[UNROLL];
    if (live) {
#pragma unroll
        for (int u = 0; u < UNROLL; u++)
            if (i0 + u * ROW < nvec) w[u] = __builtin_nontemporal_load(body + i0 + u * ROW);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
        const int i = i0 + u * ROW;
        if (i >= nvec) break;
        u32x4 packed = {0u, 0u, 0u, 0u};
        if (live) {
            float v[K], x_target = 0.f;
            E::unpack(w[u], v);
            const int64_t at = t - (head + (int64_t)i * K);
            const bool has_target = (uint64_t)at < (uint64_t)K;
            if (has_target) {
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (k == (int)at) x_target = v[k];
            }
#pragma unroll
            for (int k = 0; k < K; k++) v[k] = one(v[k]);
            if (has_target) {
                x_target = target_one(x_target);
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (k == (int)at) v[k] = x_target;
            }
            packed = E::pack(v);
        }
        __builtin_nontemporal_store(packed, out + i);
    }
    const int tail_lo = head + nvec * K, edge = head + (n - tail_lo);
    if (tile == 0 && lane < edge) {
        const int j = lane < head ? lane : tail_lo + (lane - head);
        float v = 0.f;
        if (live) {
            v = E::get(x[j]);
            v = j == t ? target_one(v) : one(v);
        }
        d[j] = E::put(v);
    }
}

// Rows of up to this many elements go one to a wave: a workgroup's meeting point and its idle lanes cost more there.
constexpr int32_t kWaveRow = 4096;

static const char *check_rows(int64_t rows, int64_t inner, int64_t n, const void *x, int32_t type, const void *target,
                              int32_t target_bits, float temperature) {
    if (type != kFp32 && type != kFp16 && type != kBf16) return "unknown type code";
    if (rows > 0x7FFFFFFF || n > 0x7FFFFFF0 || inner > 0x7FFFFFFF || inner < 1) return "too many rows or classes";
    if (!x || !target) return "null pointer";
    if ((uintptr_t)x % (type == kFp32 ? 4 : 2)) return "logits are not aligned to their elements";
    if (target_bits != 32 && target_bits != 64) return "targets have 32 or 64 bits";
    if ((uintptr_t)target % (uintptr_t)(target_bits / 8)) return "targets are not aligned to their elements";
    if (!(temperature > 0.f) || !(kLog2e / temperature <= __FLT_MAX__) || !(temperature <= __FLT_MAX__))
        return "temperature must be positive and finite";
    return nullptr;
}

template <typename T, int ROW, int UNROLL, bool ENTROPY, bool PAST>
static const char *forward_launch(const LogitRows &in, const Targets &t, float inv_t, float *logprob, float *entropy, RowStats *stats,
                           hipStream_t stream) {
    constexpr int PER = ROW < 256 ? 256 / ROW : 1;
    const unsigned grid = (unsigned)((in.rows + (int64_t)PER - 1) / PER);
    if (!launch_fits(grid, ROW < 256 ? 256 : ROW)) return "too many rows for one launch";
    hipLaunchKernelGGL((token_logprobs_kernel<T, ROW, UNROLL, ENTROPY, PAST>), dim3(grid), dim3(ROW < 256 ? 256 : ROW), 0, stream,
                       in, t, inv_t, logprob, entropy, stats);
    return nullptr;
}
// Logits of up to this many bytes go through the caches on the way forward: what the 256 MiB of the last level keep of
// them is there when the backward pass reads them again.  Both passes, through / past the caches: 412 MB of fp32 196 / 203
// us, 154 MB of bf16 77 / 81; 1.05 GB of fp16 508 / 498, 2.1 GB of bf16 1,021 / 995.
constexpr int64_t kKeepBytes = (int64_t)512 << 20;

template <typename T, int ROW, int UNROLL>
static const char *forward_rows(const LogitRows &in, const Targets &t, float inv_t, float *logprob, float *entropy, RowStats *stats,
                         hipStream_t stream) {
    const bool past = (int64_t)in.rows * in.n * (int64_t)sizeof(typename Elem<T>::Bits) > kKeepBytes;
    if (entropy && past) return forward_launch<T, ROW, UNROLL, true, true>(in, t, inv_t, logprob, entropy, stats, stream);
    if (entropy) return forward_launch<T, ROW, UNROLL, true, false>(in, t, inv_t, logprob, entropy, stats, stream);
    if (past) return forward_launch<T, ROW, UNROLL, false, true>(in, t, inv_t, logprob, entropy, stats, stream);
    return forward_launch<T, ROW, UNROLL, false, false>(in, t, inv_t, logprob, entropy, stats, stream);
}
// Threads to a row by its vectors: eight or more to a lane.  Measured (us, 256 / 512 / 1,024 threads): 16,384 x 32,000 fp16
// 156 / 147 / 190, 8,192 x 128,256 bf16 with entropies 314 / 309 / 304, 20,000 x 5,000 fp16 46 / 63 / 103, one row of
// 128,256 17.7 / 12.0 / 11.8.  Vectors of a lane in flight, 2 / 3 / 4 / 8: 311 / 300 / 306 / 387 on 8,192 x 128,256 and
// 45 / 41 / 51 / 67 on 30,000 x 4,000.
template <typename T>
static const char *forward_pick(const LogitRows &in, const Targets &t, float inv_t, float *logprob, float *entropy, RowStats *stats,
                         hipStream_t stream) {
    const int32_t vectors = in.n / Elem<T>::kVec;
    if (in.n <= kWaveRow) return forward_rows<T, 64, 3>(in, t, inv_t, logprob, entropy, stats, stream);
    if (vectors < 2048) return forward_rows<T, 256, 3>(in, t, inv_t, logprob, entropy, stats, stream);
    if (vectors < 12288) return forward_rows<T, 512, 3>(in, t, inv_t, logprob, entropy, stats, stream);
    return forward_rows<T, 1024, 3>(in, t, inv_t, logprob, entropy, stats, stream);
}

template <typename T, int ROW, int UNROLL>
static const char *backward_launch(const LogitRows &in, const Targets &t, float inv_t, const RowStats *stats, const float *gl,
                                   const float *ge, void *grad, hipStream_t stream) {
    constexpr unsigned threads = ROW < 256 ? 256 : ROW;
    const int64_t per_tile = (int64_t)ROW * UNROLL * Elem<T>::kVec;
    const int64_t tiles = (in.n + per_tile - 1) / per_tile, per = ROW < 256 ? 256 / ROW : 1;
    const int64_t grid = (in.rows * tiles + per - 1) / per;
    if (in.rows * tiles > 0x7FFFFFFF || !launch_fits(grid, threads)) return "too many elements for one launch";
    typedef typename Elem<T>::Bits Bits;
    if (ge)
        hipLaunchKernelGGL((token_logprobs_backward_kernel<T, ROW, UNROLL, true>), dim3((unsigned)grid), dim3(threads), 0, stream,
                           in, t, inv_t, stats, gl, ge, (Bits *)grad, (int32_t)tiles);
    else
        hipLaunchKernelGGL((token_logprobs_backward_kernel<T, ROW, UNROLL, false>), dim3((unsigned)grid), dim3(threads), 0, stream,
                           in, t, inv_t, stats, gl, ge, (Bits *)grad, (int32_t)tiles);
    return nullptr;
}
template <typename T>
static const char *backward_pick(const LogitRows &in, const Targets &t, float inv_t, const RowStats *stats, const float *gl,
                                 const float *ge, void *grad, hipStream_t stream) {
    if (in.n <= kWaveRow) return backward_launch<T, 64, 4>(in, t, inv_t, stats, gl, ge, grad, stream);
    // Tiles of 2,048 vectors where they leave at most 15 % of a row's last one idle, of 512 where a row has four of those, of
    // 1,024 in rows shorter than that.  Measured (us; 2,048 / 512 / 1,024): 8,192 x 128,256 bf16 with entropies 661 / 692 /
    // 710, 16,384 x 32,000 fp16 329 / 344 / 365, 2,049 x 50,257 fp32 129 / 137 / 138; 5,000 x 20,000 bf16 (61 % full) 76 /
    // 67; 20,000 x 5,000 fp16 - / 83 / 67.  Without runs of tiles on one XCD 697 and 334 (tiles of 512).
    const int64_t vectors = in.n / Elem<T>::kVec, large = (vectors + 2047) / 2048 * 2048;
    if (vectors * 100 >= large * 85) return backward_launch<T, 1024, 2>(in, t, inv_t, stats, gl, ge, grad, stream);
    if (vectors > 4 * 512) return backward_launch<T, 256, 2>(in, t, inv_t, stats, gl, ge, grad, stream);
    return backward_launch<T, 256, 4>(in, t, inv_t, stats, gl, ge, grad, stream);
}

}  // namespace bmt

extern "C" int token_logprobs_forward_launcher(int64_t rows, int64_t n, int64_t inner, int64_t outer_stride, int64_t inner_stride,
                                               const void *logits, int32_t type, const void *target, int32_t target_bits,
                                               int64_t ignore_index, float temperature, void *logprob, void *entropy, void *stats,
                                               void *stream) {
    using namespace bmt;
    if (rows <= 0 || n <= 0) return 0;
    const char *who = "token_logprobs_forward_launcher";
    if (const char *why = check_rows(rows, inner, n, logits, type, target, target_bits, temperature)) return refuse(who, why);
    if (!logprob) return refuse(who, "null pointer");
    if (((uintptr_t)logprob | (uintptr_t)entropy) % 4 || (uintptr_t)stats % 16) return refuse(who, "misaligned output");
    const LogitRows in = {logits, outer_stride, inner_stride, (int32_t)rows, (int32_t)inner, (int32_t)n};
    const Targets t = {target, target_bits == 64, ignore_index};
    const float inv_t = 1.f / temperature;
    hipStream_t s = (hipStream_t)stream;
    float *lp = (float *)logprob, *h = (float *)entropy;
    RowStats *st = (RowStats *)stats;
    const char *why = type == kFp32   ? forward_pick<Single>(in, t, inv_t, lp, h, st, s)
                      : type == kFp16 ? forward_pick<Half>(in, t, inv_t, lp, h, st, s)
                                      : forward_pick<BFloat16>(in, t, inv_t, lp, h, st, s);
    if (why) return refuse(who, why);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}

extern "C" int token_logprobs_backward_launcher(int64_t rows, int64_t n, int64_t inner, int64_t outer_stride, int64_t inner_stride,
                                                const void *logits, int32_t type, const void *target, int32_t target_bits,
                                                int64_t ignore_index, float temperature, const void *stats,
                                                const void *grad_logprob, const void *grad_entropy, void *grad, void *stream) {
    using namespace bmt;
    if (rows <= 0 || n <= 0) return 0;
    const char *who = "token_logprobs_backward_launcher";
    if (const char *why = check_rows(rows, inner, n, logits, type, target, target_bits, temperature)) return refuse(who, why);
    if (!stats || !grad) return refuse(who, "null pointer");
    if (((uintptr_t)grad_logprob | (uintptr_t)grad_entropy) % 4 || (uintptr_t)stats % 16 || (uintptr_t)grad % (type == kFp32 ? 4 : 2))
        return refuse(who, "misaligned pointer");
    const LogitRows in = {logits, outer_stride, inner_stride, (int32_t)rows, (int32_t)inner, (int32_t)n};
    const Targets t = {target, target_bits == 64, ignore_index};
    const float inv_t = 1.f / temperature;
    const RowStats *st = (const RowStats *)stats;
    const float *gl = (const float *)grad_logprob, *ge = (const float *)grad_entropy;
    hipStream_t s = (hipStream_t)stream;
    const char *why = type == kFp32   ? backward_pick<Single>(in, t, inv_t, st, gl, ge, grad, s)
                      : type == kFp16 ? backward_pick<Half>(in, t, inv_t, st, gl, ge, grad, s)
                                      : backward_pick<BFloat16>(in, t, inv_t, st, gl, ge, grad, s);
    if (why) return refuse(who, why);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}
