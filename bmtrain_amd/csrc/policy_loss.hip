// Clipped policy loss with KL and entropy terms over a padded batch of answers, and its gradients, for gfx950.
//
// Per token with new / old / reference log-probabilities l, o, f, advantage A and entropy E, where the mask is set:
//     d = l - o,  r = e^d                 policy = -min(r A, clip(r, 1 - lo, 1 + hi) A), for A < 0 at most -c A (dual clip)
//     q = f - l                           kl     = e^q - 1 - q           old_kl = e^d - 1 - d
//     loss = R(policy) + beta R(kl) - alpha R(E)
// R is the masked mean over all tokens, the mean over the sequences that have tokens of their own masked means, or the
// masked sum.  Back, with w the token's weight in R:
//     dl = w ( [not clipped] (-A r) + beta (1 - e^q) ),      dE = -alpha w
// Which side of a clip a token falls is decided on the exact d against the logarithm of the border in 64 bits, so it does
// not depend on the rounding of e^d; e^x - 1 - x is a power series for |x| < 1, where the difference would leave few
// digits, and e^x comes from the same series.
// Values under an unset mask are read but never used: whatever stands there leaves no trace.
//
// A unit is a row's part of 1,024 to 16,384 tokens, fewer in large batches; 8 to 256 lanes work on one, four tokens to a
// lane at a time.  The loss pass writes the six sums of a unit (or, where rows are not split, of a workgroup) and the
// token's unweighted derivative; one workgroup adds the sums in a fixed order; the backward pass multiplies by weight and
// upstream.  Four neighbouring tokens are added in fp32, everything above in 64 bits.  All of a quad's loads are asked for
// before the first value is used; values that few tokens need (|x| >= 1, ties at a border) are computed behind a branch
// of the whole wave.  A masked token counts as d = q = A = 0, which adds nothing anywhere; the borders and the ratios they
// cut to are picked by the advantage's sign, once for a row with one advantage.  Bound by HBM and the latency of its loads
// for large batches (1,024 x 8,192 fp32 with reference and entropy: 176 MB in 35.5 us, 5.0 TB/s; 95 to 111 registers leave
// four waves to a SIMD, a cap for five makes them spill: 50 us for both launches instead of 40.6), by launches for small.
#include "bmt_vec.h"
#include "../../include/bmt_hip.h"

namespace bmt {

constexpr int kSums = 6;             // policy, kl, entropy, clipped, old_kl, tokens (or sequences) counted
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
    int32_t rows, time, chunks, unit, lanes, reduction;
    double high, low, far;                           // log(1 + hi), log(1 - lo), log(c); far = inf: no dual clip
    float ratio_high, ratio_low, ratio_far, kl_coef;
};

// e^x - 1 - x for |x| < 1: x^2 (1/2 + x/6 + ... + x^9/11!), what is left out is below 2^-27 of the sum.
__device__ __forceinline__ float exp_tail_series(float x) {
    float s = 1.f / 39916800.f;
    s = __builtin_fmaf(s, x, 1.f / 3628800.f);
    s = __builtin_fmaf(s, x, 1.f / 362880.f);
    s = __builtin_fmaf(s, x, 1.f / 40320.f);
    s = __builtin_fmaf(s, x, 1.f / 5040.f);
    s = __builtin_fmaf(s, x, 1.f / 720.f);
    s = __builtin_fmaf(s, x, 1.f / 120.f);
    s = __builtin_fmaf(s, x, 1.f / 24.f);
    s = __builtin_fmaf(s, x, 1.f / 6.f);
    s = __builtin_fmaf(s, x, 0.5f);
    return x * x * s;
}

// On which side of 1 a token's ratio is cut, by the sign of its advantage: above `high` to `ratio`, below `low`.
struct Side {
    float high, low, ratio;
};
__device__ __forceinline__ Side side_of(const PolicyIn &in, float A) {
    if (A > 0.f) return {(float)in.high, -INFINITY, in.ratio_high};
    if (A < 0.f) return {(float)in.far, (float)in.low, in.ratio_far};
    return {INFINITY, -INFINITY, 1.f};
}

template <typename T>
struct Tokens {                      // four tokens as they are in memory
    Raw4<T> logprob, old, ref, entropy;
    Raw4<Single> advantage;
    uint32_t mask;
};

// The six sums of every thread in v[0..5], over the workgroup: all[0..5] of the slots, valid behind the last barrier.
__device__ __forceinline__ void workgroup_sums(double *v, double (*slots)[8], double *all) {
    v[6] = v[7] = 0;
    const double s = wave_sum8(v);
    if (threadIdx.x % 8 == 0) slots[threadIdx.x / kWave][threadIdx.x % kWave / 8] = s;
    __syncthreads();
    if (threadIdx.x < kSums) {
        double t = 0;
        for (int w = 0; w < (int)blockDim.x / kWave; w++) t += slots[w][threadIdx.x];
        all[threadIdx.x] = t;
    }
    __syncthreads();
}

// COL: one advantage for each token, not one for a row.  kWhole: the workgroup's lanes work on one unit; kGroups: groups of
// in.lanes lanes of a wave do; kTiny: the same for rows of up to three tokens.
enum Form { kWhole, kGroups, kTiny };
template <typename T, Form FORM, bool COL>
__global__ __launch_bounds__(kLossThreads) void policy_loss_kernel(PolicyIn in, uint32_t units, float *__restrict__ saved,
                                                                   float *__restrict__ weights, double *__restrict__ sums) {
    typedef typename Elem<T>::Bits Bits;
    // Long fp32 rows are read past the caches, which leaves them to what the backward pass reads: 8.4 M tokens with reference
    // and entropy 40.6 / 43.4 us past / through the caches, both launches; bf16 without entropy 27.6 / 26.4.
    constexpr bool WHOLE = FORM == kWhole, PAST = WHOLE && sizeof(Bits) == 4;
    const int lanes = WHOLE ? kLossThreads : in.lanes, groups = kLossThreads / lanes;
    const int lane = threadIdx.x % lanes, group = WHOLE ? 0 : threadIdx.x / lanes, step = lanes * 4;
    const bool split = in.chunks > 1;
    __shared__ double slots[kLossThreads / kWave][8], all[8];
    double total[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (uint32_t first = blockIdx.x * groups; first < units; first += gridDim.x * groups) {
        const uint32_t unit = first + group;
        const bool there = unit < units;
        const int64_t row = there ? unit / (uint32_t)in.chunks : 0;
        const int begin = there ? (int)(unit - (uint32_t)row * (uint32_t)in.chunks) * in.unit : 0;
        const int end = there ? (in.time - begin < in.unit ? in.time : begin + in.unit) : 0;
        const Bits *lp = (const Bits *)in.logprob + row * in.logprob_row;
        const Bits *op = (const Bits *)in.old + row * in.old_row;
        // without a reference q is 0, or NaN where l is not finite, and not used
        const Bits *fp = in.ref ? (const Bits *)in.ref + row * in.ref_row : lp;
        const Bits *ep = (const Bits *)in.entropy + row * in.entropy_row;
        const uint8_t *mp = in.mask ? in.mask + row * in.mask_row : nullptr;
        const float *ap = in.advantage + row * in.advantage_row;
        const float row_advantage = there && !COL ? ap[0] : 0.f;
        const Side row_side = side_of(in, row_advantage);
        int clipped = 0, tokens = 0;
        double acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        for (int i = begin + lane * 4; i < end; i += step) {
            // The last quad of a row that has fewer than four tokens left starts further in front and leaves out what it
            // shares with its neighbour, so that all loads are whole (a row of one to three tokens has no room for that).
            const int at = FORM == kTiny || i + 4 <= end ? i : end - 4, skip = i - at;
            Tokens<T> now;
            if (FORM == kTiny) {
                now.mask = load_mask4(mp ? mp + at : nullptr, end - at);
                now.logprob.load_some(lp + at, end - at);
                now.old.load_some(op + at, end - at);
                now.ref.load_some(fp + at, end - at);
                if (in.entropy) now.entropy.load_some(ep + at, end - at);
                if (COL) now.advantage.load_some((const uint32_t *)ap + at, end - at);
            } else {
                now.mask = mp ? *(const u32_any1 *)(mp + at) : 0x01010101u;
                now.logprob.template load<PAST>(lp + at);
                now.old.template load<PAST>(op + at);
                now.ref.template load<PAST>(fp + at);
                if (in.entropy) now.entropy.template load<PAST>(ep + at);
                if (COL) now.advantage.load((const uint32_t *)ap + at);
                now.mask &= 0xFFFFFFFFu << (8 * skip);
            }
            float sum[4] = {0, 0, 0, 0};                  // of these four tokens: policy, kl, entropy, old_kl
            float g[4], d[4], q[4], A[4], most = 0.f;
            bool on[4], tie = false;
            Side side[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                // what is masked counts as d = q = A = 0, which adds nothing anywhere
                const float l = now.logprob.get(k);
                on[k] = mask_set(now.mask, k);
                d[k] = on[k] ? l - now.old.get(k) : 0.f;
                q[k] = on[k] ? now.ref.get(k) - l : 0.f;
                A[k] = on[k] ? COL ? now.advantage.get(k) : row_advantage : 0.f;
                side[k] = COL ? side_of(in, A[k]) : row_side;
                most = fmaxf(most, fmaxf(fabsf(d[k]), fabsf(q[k])));
                // rounding keeps the order, so the rounded d against a rounded border is the answer unless they are equal
                tie |= d[k] == side[k].high || d[k] == side[k].low;
            }
            const bool careful = __any(!(most < 1.f) || tie);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float old_kl = exp_tail_series(d[k]), rm1 = d[k] + old_kl;       // e^d - 1 - d, e^d - 1
                float kl = exp_tail_series(q[k]), qm1 = q[k] + kl;
                bool over = d[k] > side[k].high, under = d[k] < side[k].low;
                if (careful) {
                    const double wide = on[k] ? (double)now.logprob.get(k) - (double)now.old.get(k) : 0.0;
                    over = A[k] > 0.f ? wide > in.high : A[k] < 0.f && wide > in.far;
                    under = A[k] < 0.f && wide < in.low;
                    if (!(fabsf(d[k]) < 1.f)) {
                        rm1 = expf(d[k]) - 1.f, old_kl = rm1 - d[k];
                        if (A[k] == 0.f && rm1 == INFINITY) rm1 = 0.f;      // e^d beyond fp32 times 0 is 0, not NaN
                    }
                    if (!(fabsf(q[k]) < 1.f)) qm1 = expf(q[k]) - 1.f, kl = qm1 - q[k];
                }
                const float r = over ? side[k].ratio : under ? in.ratio_low : 1.f + rm1;
                const float policy = -r * A[k];
                g[k] = (over || under ? 0.f : policy) - (in.kl_coef != 0.f ? in.kl_coef * qm1 : 0.f);
                sum[0] += policy;
                sum[1] += kl;
                if (in.entropy) sum[2] += on[k] ? now.entropy.get(k) : 0.f;
                sum[3] += old_kl;
                clipped += over || under ? 1 : 0;
                tokens += on[k] ? 1 : 0;
            }
            acc[0] += (double)sum[0];
            if (in.ref) acc[1] += (double)sum[1];
            if (in.entropy) acc[2] += (double)sum[2];
            acc[4] += (double)sum[3];
            if (saved) {
                uint32_t *to = (uint32_t *)saved + row * in.time + at;
                if (FORM == kTiny) {
                    store4<Single>(to, end - at, g);
                } else if (skip == 0) {
                    store4<Single>(to, 4, g);
                } else {
#pragma unroll
                    for (int k = 1; k < 4; k++)
                        if (k >= skip) to[k] = Elem<Single>::put(g[k]);
                }
            }
        }
        acc[3] = clipped, acc[5] = tokens;
        if (!split && in.reduction == kSequence) {        // the row is this group's: its own mean
            if (WHOLE) {
                workgroup_sums(acc, slots, all);
#pragma unroll
                for (int k = 0; k < kSums; k++) acc[k] = all[k];
            } else {
#pragma unroll
                for (int k = 0; k < kSums; k++) acc[k] = lanes_sum(acc[k], lanes);
            }
            const double weight = acc[5] > 0 ? 1.0 / acc[5] : 0.0;
            if (lane == 0 && there) {
                weights[1 + row] = (float)weight;
#pragma unroll
                for (int k = 0; k < 5; k++) total[k] += acc[k] * weight;
                total[5] += acc[5] > 0 ? 1.0 : 0.0;
            }
        } else {
#pragma unroll
            for (int k = 0; k < kSums; k++) total[k] += acc[k];
        }
    }
    __syncthreads();
    workgroup_sums(total, slots, all);
    if (threadIdx.x < kSums) sums[(int64_t)blockIdx.x * kSums + threadIdx.x] = all[threadIdx.x];
}

// Adds the sums of all workgroups.  by_row: `parts` = rows x chunks, and every row's mean is formed first.
// stats: R(policy), R(kl), R(entropy), R(clipped), R(old_kl).  weights[0]: 1 / (tokens or sequences counted), behind it
// the rows' own weights (sequence mean only).
__global__ __launch_bounds__(kFinishThreads) void policy_finish_kernel(const double *__restrict__ sums, int64_t parts,
                                                                       int32_t chunks, int32_t reduction, float kl_coef,
                                                                       float entropy_coef, float *__restrict__ weights,
                                                                       float *__restrict__ loss, float *__restrict__ stats) {
    const bool by_row = reduction == kSequence && chunks > 1;
    double acc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
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
    __shared__ double slots[kFinishThreads / kWave][8], all[8];
    workgroup_sums(acc, slots, all);
    if (threadIdx.x == 0) {
        const double share = reduction == kSum ? 1.0 : all[5] > 0 ? 1.0 / all[5] : 0.0;     // nothing counts: loss 0
        for (int k = 0; k < 5; k++) all[k] *= share;
        // a term without weight is only measured: no 0 * inf
        loss[0] = (float)(all[0] + (kl_coef != 0.f ? (double)kl_coef * all[1] : 0.0) -
                          (entropy_coef != 0.f ? (double)entropy_coef * all[2] : 0.0));
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
        const uint32_t m = load_mask4(mask ? mask + row * mask_row + i : nullptr, count);
        float g[4];
#pragma unroll
        for (int k = 0; k < 4; k++) g[k] = mask_set(m, k) && entropy_coef != 0.f ? -entropy_coef * scale : 0.f;
        store4<T>(grad_entropy + at, count, g);
    }
}

struct Shape {
    int lanes;
    int32_t unit, chunks;
    int64_t units, grid;
};
// A row of up to 256 tokens is that of 8 to 64 lanes, four tokens each; up to 1,024 it is a workgroup's while there are few
// rows, where it is the latency that counts, and a wave's when there are many.  Longer rows are split into parts of a
// workgroup each, the shortest from 1,024 to 16,384 tokens that give at most 1,024 parts: a workgroup's start and its
// sums cost as much as some 2,000 tokens (8.4 M tokens fp32 with reference and entropy: 40.6 us in parts of 8,192 tokens,
// 42.3 of 4,096, 46.4 of 2,048, 63 of 1,024; both launches).
static Shape shape_of(int64_t rows, int64_t time) {
    Shape s;
    s.unit = 1024;
    while (s.unit < 16384 && rows * ((time + s.unit - 1) / s.unit) > 1024) s.unit *= 2;
    s.chunks = (int32_t)((time + s.unit - 1) / s.unit);
    s.lanes = 8;
    while (s.lanes < 64 && s.lanes * 4 < time) s.lanes *= 2;
    if (time > 1024 || (time > 256 && rows < 4096)) s.lanes = kLossThreads;
    s.units = rows * s.chunks;
    const int64_t groups = kLossThreads / s.lanes;
    s.grid = (s.units + groups - 1) / groups;
    if (s.chunks == 1 && s.grid > kMaxWorkgroups) s.grid = kMaxWorkgroups;
    return s;
}

template <typename T, bool COL>
static void loss_launch(const PolicyIn &in, const Shape &s, float *saved, float *weights, double *sums, hipStream_t stream) {
    const dim3 grid((unsigned)s.grid), threads(kLossThreads);
    if (s.lanes == kLossThreads)
        hipLaunchKernelGGL((policy_loss_kernel<T, kWhole, COL>), grid, threads, 0, stream, in, (uint32_t)s.units, saved, weights, sums);
    else if (in.time >= 4)
        hipLaunchKernelGGL((policy_loss_kernel<T, kGroups, COL>), grid, threads, 0, stream, in, (uint32_t)s.units, saved, weights, sums);
    else
        hipLaunchKernelGGL((policy_loss_kernel<T, kTiny, COL>), grid, threads, 0, stream, in, (uint32_t)s.units, saved, weights, sums);
}
template <typename T>
static void loss_pick(const PolicyIn &in, const Shape &s, float *saved, float *weights, double *sums, hipStream_t stream) {
    if (in.advantage_col) loss_launch<T, true>(in, s, saved, weights, sums, stream);
    else loss_launch<T, false>(in, s, saved, weights, sums, stream);
}

static bool fits(int64_t rows, int64_t time) {
    if (rows > 0x7FFFFFFF || time > 0x3FFFFFFF || !launch_fits(rows * ((time + 3) / 4) / kLossThreads + 1, kLossThreads))
        return false;
    const Shape s = shape_of(rows, time);
    return s.units < 0x7FFFFFFF && launch_fits(s.grid, kLossThreads);
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
    Shape shape = {64, 1024, 1, 0, 0};
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
        in.rows = (int32_t)rows, in.time = (int32_t)time, in.reduction = reduction;
        in.chunks = shape.chunks, in.unit = shape.unit, in.lanes = shape.lanes;
        in.high = log1p(clip_high), in.low = log1p(-clip_low);          // clip_low = 1: log 0 = -inf, never below it
        in.far = dual_clip != 0 ? log(dual_clip) : (double)INFINITY;
        in.ratio_high = (float)(1 + clip_high), in.ratio_low = (float)(1 - clip_low), in.ratio_far = (float)dual_clip;
        in.kl_coef = ref_logprob ? kl_coef : 0.f;                       // no KL, no gradient of it
        if (type == kFp32) loss_pick<Single>(in, shape, (float *)saved, (float *)weights, (double *)workspace, s);
        else if (type == kFp16) loss_pick<Half>(in, shape, (float *)saved, (float *)weights, (double *)workspace, s);
        else loss_pick<BFloat16>(in, shape, (float *)saved, (float *)weights, (double *)workspace, s);
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
