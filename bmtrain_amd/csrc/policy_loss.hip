// Clipped policy loss with KL and entropy terms over a padded batch of answers, and its gradients, for gfx950.
//
// Per token with new / old / reference log-probabilities l, o, f, advantage A and entropy E, where the mask is set:
//     d = l - o,  r = e^d                 policy = -min(r A, clip(r, 1 - lo, 1 + hi) A), for A < 0 at most -c A (dual clip)
//     q = f - l                           kl     = e^q - 1 - q           old_kl = e^d - 1 - d
//     loss = R(policy) + beta R(kl) - alpha R(E)
// R is the masked mean over all tokens, the mean over the sequences that have tokens of their own masked means, or the
// masked sum.  Back, with w the token's weight in R:
//     dl = w ( [not clipped] (-A r) + beta (1 - e^q) ),      dE = -alpha w
// Which side of a clip a token falls is decided on d in 64 bits against the logarithm of the border, so it does not
// depend on the rounding of e^d; e^x - 1 - x is a power series near 0, where the difference would leave no digits.
// Values under an unset mask are read but never used: whatever stands there leaves no trace.
//
// A unit is a row's part of up to 4,096 tokens; 8, 64 or 256 lanes work on one, four tokens to a lane at a time.  The
// loss pass writes the six sums of a unit (or, where rows are not split, of a workgroup) and the token's unweighted
// derivative; one workgroup adds the sums in a fixed order; the backward pass multiplies by weight and upstream.  All
// sums are held in 64 bits.  Bound by HBM for large batches (fp32 with a reference: 13 B read and 4 written per token
// forward, 4 read and 4 written back), by launches for small ones.
#include "bmt_vec.h"
#include "../../include/bmt_hip.h"

namespace bmt {

constexpr int kSums = 6;             // policy, kl, entropy, clipped, old_kl, tokens (or sequences) counted
constexpr int kUnitTokens = 4096;
constexpr int kLossThreads = 256;
constexpr int kFinishThreads = 1024;
constexpr int64_t kMaxWorkgroups = 2048;

enum : int32_t { kMean = 0, kSequence = 1, kSum = 2 };

struct PolicyIn {
    const void *logprob, *old, *ref, *entropy;       // ref, entropy: null where absent
    const float *advantage;
    const uint8_t *mask;                             // null: every token counts
    int64_t logprob_row, old_row, ref_row, entropy_row, advantage_row, mask_row;   // elements between rows
    int32_t advantage_col;                           // 0: one advantage for a whole row; 1: one for each token
    int32_t rows, time, chunks, reduction;
    double high, low, far;                           // log(1 + hi), log(1 - lo), log(c); far = inf: no dual clip
    float ratio_high, ratio_low, ratio_far, kl_coef;
};

// e^x - 1 - x
__device__ __forceinline__ float exp_minus_linear(float x) {
    if (fabsf(x) < 0.5f) {           // x^2 (1/2 + x/6 + ... + x^7/9!): the first term left out is below 2^-29 of the sum
        float s = 1.f / 362880.f;
        s = __builtin_fmaf(s, x, 1.f / 40320.f);
        s = __builtin_fmaf(s, x, 1.f / 5040.f);
        s = __builtin_fmaf(s, x, 1.f / 720.f);
        s = __builtin_fmaf(s, x, 1.f / 120.f);
        s = __builtin_fmaf(s, x, 1.f / 24.f);
        s = __builtin_fmaf(s, x, 1.f / 6.f);
        s = __builtin_fmaf(s, x, 0.5f);
        return x * x * s;
    }
    return expm1f(x) - x;
}

template <typename T, int LANES>
__global__ __launch_bounds__(kLossThreads) void policy_loss_kernel(PolicyIn in, int64_t units, float *__restrict__ saved,
                                                                   float *__restrict__ weights, double *__restrict__ sums) {
    typedef typename Elem<T>::Bits Bits;
    constexpr int GROUPS = kLossThreads / LANES, WAVES = kLossThreads / kWave;
    const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
    const bool split = in.chunks > 1;
    __shared__ double slots[WAVES][kSums];
    double total[kSums] = {0, 0, 0, 0, 0, 0};
    for (int64_t first = (int64_t)blockIdx.x * GROUPS; first < units; first += (int64_t)gridDim.x * GROUPS) {
        const int64_t unit = first + group;
        double acc[kSums] = {0, 0, 0, 0, 0, 0};
        const bool there = unit < units;
        const int32_t row = there ? (int32_t)(unit / in.chunks) : 0;
        const int begin = there ? (int)(unit - (int64_t)row * in.chunks) * kUnitTokens : in.time;
        const int end = there ? (in.time - begin < kUnitTokens ? in.time : begin + kUnitTokens) : 0;
        const Bits *lp = (const Bits *)in.logprob + row * in.logprob_row;
        const Bits *op = (const Bits *)in.old + row * in.old_row;
        const Bits *fp = (const Bits *)in.ref + (in.ref ? row * in.ref_row : 0);
        const Bits *ep = (const Bits *)in.entropy + (in.entropy ? row * in.entropy_row : 0);
        const uint8_t *mp = in.mask ? in.mask + row * in.mask_row : nullptr;
        const float *ap = in.advantage + row * in.advantage_row;
        for (int i = begin + lane * 4; i < end; i += LANES * 4) {
            const int count = end - i;
            float l[4], o[4], f[4] = {0, 0, 0, 0}, e[4] = {0, 0, 0, 0}, a[4], g[4];
            const uint32_t m = mask4(mp ? mp + i : nullptr, count);
            load4<T>(lp + i, count, l);
            load4<T>(op + i, count, o);
            if (in.ref) load4<T>(fp + i, count, f);
            if (in.entropy) load4<T>(ep + i, count, e);
            if (in.advantage_col) load4<Single>((const uint32_t *)ap + i, count, a);
            else a[0] = a[1] = a[2] = a[3] = ap[0];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const double wide = (double)l[k] - (double)o[k];
                const float d = (float)wide, r = expf(d), A = a[k];
                float policy = -r * A, slope = -r * A;
                bool clipped = false;
                if (A > 0.f) {
                    if (wide > in.high) clipped = true, policy = -in.ratio_high * A;
                } else if (A < 0.f) {
                    if (wide < in.low) clipped = true, policy = -in.ratio_low * A;
                    else if (wide > in.far) clipped = true, policy = -in.ratio_far * A;
                }
                if (clipped) slope = 0.f;
                float kl = 0.f;
                if (in.ref) {
                    const float q = (float)((double)f[k] - (double)l[k]);
                    kl = exp_minus_linear(q);
                    slope = __builtin_fmaf(-in.kl_coef, expm1f(q), slope);
                }
                const bool on = m >> k & 1u;
                g[k] = on ? slope : 0.f;
                if (on) {
                    acc[0] += (double)policy;
                    acc[1] += (double)kl;
                    acc[2] += (double)e[k];
                    acc[3] += clipped ? 1.0 : 0.0;
                    acc[4] += (double)exp_minus_linear(d);
                    acc[5] += 1.0;
                }
            }
            if (saved) store4<Single>((uint32_t *)saved + (int64_t)row * in.time + i, count, g);
        }
        if (!split && in.reduction == kSequence) {        // the row is this group's: its own mean
#pragma unroll
            for (int k = 0; k < kSums; k++) acc[k] = lanes_sum(acc[k], LANES < kWave ? LANES : kWave);
            if (LANES > kWave) {
                __syncthreads();
                if (threadIdx.x % kWave == 0)
                    for (int k = 0; k < kSums; k++) slots[threadIdx.x / kWave][k] = acc[k];
                __syncthreads();
                for (int k = 0; k < kSums; k++) {
                    acc[k] = 0;
                    for (int w = 0; w < WAVES; w++) acc[k] += slots[w][k];
                }
            }
            const double weight = acc[5] > 0 ? 1.0 / acc[5] : 0.0;
            if (lane == 0 && there) {
                weights[1 + row] = (float)weight;
                for (int k = 0; k < 5; k++) total[k] += acc[k] * weight;
                total[5] += acc[5] > 0 ? 1.0 : 0.0;
            }
        } else {
#pragma unroll
            for (int k = 0; k < kSums; k++) total[k] += acc[k];
        }
        if (split) break;                                 // one unit to a workgroup: its sums are joined by row
    }
#pragma unroll
    for (int k = 0; k < kSums; k++) total[k] = lanes_sum(total[k], kWave);
    __syncthreads();
    if (threadIdx.x % kWave == 0)
        for (int k = 0; k < kSums; k++) slots[threadIdx.x / kWave][k] = total[k];
    __syncthreads();
    if (threadIdx.x < kSums) {
        double v = 0;
        for (int w = 0; w < WAVES; w++) v += slots[w][threadIdx.x];
        sums[(int64_t)blockIdx.x * kSums + threadIdx.x] = v;
    }
}

// Adds the sums of all workgroups.  by_row: `parts` = rows x chunks, and every row's mean is formed first.
// stats: R(policy), R(kl), R(entropy), R(clipped), R(old_kl).  weights[0]: 1 / (tokens or sequences counted), behind it
// the rows' own weights (sequence mean only).
__global__ __launch_bounds__(kFinishThreads) void policy_finish_kernel(const double *__restrict__ sums, int64_t parts,
                                                                       int32_t chunks, int32_t reduction, float kl_coef,
                                                                       float entropy_coef, float *__restrict__ weights,
                                                                       float *__restrict__ loss, float *__restrict__ stats) {
    const bool by_row = reduction == kSequence && chunks > 1;
    double acc[kSums] = {0, 0, 0, 0, 0, 0};
    if (by_row) {
        const int64_t rows = parts / chunks;
        for (int64_t r = threadIdx.x; r < rows; r += kFinishThreads) {
            double row[kSums] = {0, 0, 0, 0, 0, 0};
            for (int32_t c = 0; c < chunks; c++)
                for (int k = 0; k < kSums; k++) row[k] += sums[(r * chunks + c) * kSums + k];
            const double weight = row[5] > 0 ? 1.0 / row[5] : 0.0;
            weights[1 + r] = (float)weight;
            for (int k = 0; k < 5; k++) acc[k] += row[k] * weight;
            acc[5] += row[5] > 0 ? 1.0 : 0.0;
        }
    } else {
        for (int64_t p = threadIdx.x; p < parts; p += kFinishThreads)
            for (int k = 0; k < kSums; k++) acc[k] += sums[p * kSums + k];
    }
    __shared__ double slots[kFinishThreads / kWave][kSums];
#pragma unroll
    for (int k = 0; k < kSums; k++) acc[k] = lanes_sum(acc[k], kWave);
    if (threadIdx.x % kWave == 0)
        for (int k = 0; k < kSums; k++) slots[threadIdx.x / kWave][k] = acc[k];
    __syncthreads();
    __shared__ double all[kSums];
    if (threadIdx.x < kSums) {
        double v = 0;
        for (int w = 0; w < kFinishThreads / kWave; w++) v += slots[w][threadIdx.x];
        all[threadIdx.x] = v;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const double share = reduction == kSum ? 1.0 : all[5] > 0 ? 1.0 / all[5] : 0.0;     // nothing counts: loss 0
        for (int k = 0; k < 5; k++) all[k] *= share;
        loss[0] = (float)(all[0] + (double)kl_coef * all[1] - (double)entropy_coef * all[2]);
        for (int k = 0; k < 5; k++) stats[k] = (float)all[k];
        weights[0] = (float)share;
    }
}

// grad = saved * weight * upstream and, where asked for, grad_entropy = -alpha * weight * upstream under the mask.
template <typename T>
__global__ __launch_bounds__(kLossThreads) void policy_backward_kernel(
    int32_t time, int64_t quads_per_row, int64_t quads, const float *__restrict__ saved, const float *__restrict__ weights,
    int32_t by_row, const float *__restrict__ upstream, const uint8_t *__restrict__ mask, int64_t mask_row,
    float entropy_coef, typename Elem<T>::Bits *__restrict__ grad, typename Elem<T>::Bits *__restrict__ grad_entropy) {
    const int64_t q = (int64_t)blockIdx.x * kLossThreads + threadIdx.x;
    if (q >= quads) return;
    const int64_t row = q / quads_per_row;
    const int i = (int)(q - row * quads_per_row) * 4, count = time - i;
    const float scale = upstream[0] * weights[0] * (by_row ? weights[1 + row] : 1.f);
    const int64_t at = row * time + i;
    if (grad) {
        float g[4];
        load4<Single>((const uint32_t *)saved + at, count, g);
#pragma unroll
        for (int k = 0; k < 4; k++) g[k] = g[k] == 0.f ? 0.f : g[k] * scale;      // 0 also under an infinite upstream
        store4<T>(grad + at, count, g);
    }
    if (grad_entropy) {
        const uint32_t m = mask4(mask ? mask + row * mask_row + i : nullptr, count);
        float g[4];
#pragma unroll
        for (int k = 0; k < 4; k++) g[k] = m >> k & 1u ? -entropy_coef * scale : 0.f;
        store4<T>(grad_entropy + at, count, g);
    }
}

struct Shape {
    int lanes;
    int32_t chunks;
    int64_t units, grid;
};
// Lanes to a unit: a row of up to 32 tokens is eight lanes' (four tokens each), one of up to 1,024 a wave's, anything
// longer a workgroup's.  Rows that are split get a workgroup for every part.
static Shape shape_of(int64_t rows, int64_t time) {
    Shape s;
    s.chunks = (int32_t)((time + kUnitTokens - 1) / kUnitTokens);
    s.lanes = time <= 32 ? 8 : time <= 1024 ? 64 : 256;
    s.units = rows * s.chunks;
    const int64_t groups = kLossThreads / s.lanes;
    s.grid = (s.units + groups - 1) / groups;
    if (s.chunks == 1 && s.grid > kMaxWorkgroups) s.grid = kMaxWorkgroups;
    return s;
}

template <typename T>
static void loss_launch(const PolicyIn &in, const Shape &s, float *saved, float *weights, double *sums, hipStream_t stream) {
    if (s.lanes == 8)
        hipLaunchKernelGGL((policy_loss_kernel<T, 8>), dim3((unsigned)s.grid), dim3(kLossThreads), 0, stream, in, s.units, saved,
                           weights, sums);
    else if (s.lanes == 64)
        hipLaunchKernelGGL((policy_loss_kernel<T, 64>), dim3((unsigned)s.grid), dim3(kLossThreads), 0, stream, in, s.units, saved,
                           weights, sums);
    else
        hipLaunchKernelGGL((policy_loss_kernel<T, 256>), dim3((unsigned)s.grid), dim3(kLossThreads), 0, stream, in, s.units, saved,
                           weights, sums);
}

static bool fits(int64_t rows, int64_t time) {
    return rows <= 0x7FFFFFFF && time <= 0x3FFFFFFF && (rows * ((time + 3) / 4)) / kLossThreads < 0x7FFFFFFF &&
           rows * ((time + kUnitTokens - 1) / kUnitTokens) < 0x7FFFFFFF;
}

}  // namespace bmt

extern "C" int64_t policy_loss_workspace_doubles(int64_t rows, int64_t time) {
    if (rows <= 0 || time <= 0 || !bmt::fits(rows, time)) return 1;
    return bmt::shape_of(rows, time).grid * bmt::kSums;
}

extern "C" int policy_loss_forward_launcher(int64_t rows, int64_t time, int32_t type, const void *logprob, int64_t logprob_row,
                                            const void *old_logprob, int64_t old_row, const void *ref_logprob, int64_t ref_row,
                                            const void *entropy, int64_t entropy_row, const void *advantage,
                                            int64_t advantage_row, int32_t advantage_col, const void *mask, int64_t mask_row,
                                            double clip_low, double clip_high, double dual_clip, float kl_coef,
                                            float entropy_coef, int32_t reduction, void *saved, void *weights,
                                            void *workspace, void *loss, void *stats, void *stream) {
    using namespace bmt;
    const char *who = "policy_loss_forward_launcher";
    if (rows < 0 || time < 0) return refuse(who, "negative size");
    if (!loss || !stats || !weights || !workspace) return refuse(who, "null pointer");
    if (reduction < kMean || reduction > kSum) return refuse(who, "unknown reduction");
    if (type != kFp32 && type != kFp16 && type != kBf16) return refuse(who, "unknown type code");
    if (!(clip_low >= 0) || !(clip_high >= 0) || clip_low > 1) return refuse(who, "clip range must be in [0, 1] and [0, inf)");
    if (dual_clip != 0 && !(dual_clip > 1)) return refuse(who, "dual_clip must be above 1, or 0 for none");
    if ((uintptr_t)workspace % 8 || ((uintptr_t)loss | (uintptr_t)stats | (uintptr_t)saved | (uintptr_t)weights) % 4)
        return refuse(who, "misaligned output");
    hipStream_t s = (hipStream_t)stream;
    Shape shape = {64, 1, 0, 0};
    if (rows > 0 && time > 0) {
        if (!fits(rows, time)) return refuse(who, "too many tokens for one launch");
        if (!logprob || !old_logprob || !advantage) return refuse(who, "null pointer");
        if (advantage_col != 0 && advantage_col != 1) return refuse(who, "advantages are one to a row or one to a token");
        const uintptr_t size = type == kFp32 ? 4 : 2;
        if (((uintptr_t)logprob | (uintptr_t)old_logprob | (uintptr_t)ref_logprob | (uintptr_t)entropy) % size ||
            (uintptr_t)advantage % 4)
            return refuse(who, "misaligned input");
        shape = shape_of(rows, time);
        PolicyIn in;
        in.logprob = logprob, in.old = old_logprob, in.ref = ref_logprob, in.entropy = entropy;
        in.advantage = (const float *)advantage, in.mask = (const uint8_t *)mask;
        in.logprob_row = logprob_row, in.old_row = old_row, in.ref_row = ref_row, in.entropy_row = entropy_row;
        in.advantage_row = advantage_row, in.mask_row = mask_row, in.advantage_col = advantage_col;
        in.rows = (int32_t)rows, in.time = (int32_t)time, in.chunks = shape.chunks, in.reduction = reduction;
        in.high = log1p(clip_high), in.low = log1p(-clip_low);          // clip_low = 1: log 0 = -inf, never below it
        in.far = dual_clip != 0 ? log(dual_clip) : (double)INFINITY;
        in.ratio_high = (float)(1 + clip_high), in.ratio_low = (float)(1 - clip_low), in.ratio_far = (float)dual_clip;
        in.kl_coef = kl_coef;
        if (type == kFp32) loss_launch<Single>(in, shape, (float *)saved, (float *)weights, (double *)workspace, s);
        else if (type == kFp16) loss_launch<Half>(in, shape, (float *)saved, (float *)weights, (double *)workspace, s);
        else loss_launch<BFloat16>(in, shape, (float *)saved, (float *)weights, (double *)workspace, s);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return fail((int)e, who, e);
    }
    hipLaunchKernelGGL(policy_finish_kernel, dim3(1), dim3(kFinishThreads), 0, s, (const double *)workspace, shape.grid, shape.chunks,
                       reduction, kl_coef, entropy_coef, (float *)weights, (float *)loss, (float *)stats);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}

extern "C" int policy_loss_backward_launcher(int64_t rows, int64_t time, int32_t type, int32_t reduction, const void *saved,
                                             const void *weights, const void *upstream, const void *mask, int64_t mask_row,
                                             float entropy_coef, void *grad_logprob, void *grad_entropy, void *stream) {
    using namespace bmt;
    const char *who = "policy_loss_backward_launcher";
    if (rows <= 0 || time <= 0 || (!grad_logprob && !grad_entropy)) return 0;
    if (!fits(rows, time)) return refuse(who, "too many tokens for one launch");
    if (type != kFp32 && type != kFp16 && type != kBf16) return refuse(who, "unknown type code");
    if (!weights || !upstream || (grad_logprob && !saved)) return refuse(who, "null pointer");
    if (((uintptr_t)grad_logprob | (uintptr_t)grad_entropy) % (type == kFp32 ? 4 : 2) ||
        ((uintptr_t)saved | (uintptr_t)weights | (uintptr_t)upstream) % 4)
        return refuse(who, "misaligned pointer");
    const int64_t per_row = (time + 3) / 4, quads = rows * per_row;
    const dim3 grid((unsigned)((quads + kLossThreads - 1) / kLossThreads));
    hipStream_t s = (hipStream_t)stream;
#define BMT_LAUNCH(T)                                                                                                          \
    hipLaunchKernelGGL((policy_backward_kernel<T>), grid, dim3(kLossThreads), 0, s, (int32_t)time, per_row, quads,             \
                       (const float *)saved, (const float *)weights, (int32_t)(reduction == kSequence),                        \
                       (const float *)upstream, (const uint8_t *)mask, mask_row, entropy_coef, (Elem<T>::Bits *)grad_logprob,  \
                       (Elem<T>::Bits *)grad_entropy)
    if (type == kFp32) BMT_LAUNCH(Single);
    else if (type == kFp16) BMT_LAUNCH(Half);
    else BMT_LAUNCH(BFloat16);
#undef BMT_LAUNCH
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}
