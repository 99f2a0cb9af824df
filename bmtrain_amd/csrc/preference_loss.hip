// Loss of paired answers (chosen against rejected) on sums of token log-ratios, and its gradient, for gfx950.
//
// Rows 0 .. P-1 hold the chosen answers' token log-probabilities l, rows P .. 2P-1 the rejected ones', f the reference
// model's.  With the mask's token count n_i (an empty row has sum 0):
//     s_i = sum_t m (l - f)            (divided by n_i for length-normalised sums)
//     h   = s_chosen - s_rejected
//     logistic : -(1 - e) log sigmoid(b h) - e log sigmoid(-b h)
//     squared  : (h - 1 / (2 b))^2
//     hinge    : max(0, 1 - b h)
//     loss     = mean over the pairs that have a token in either row;      rewards b s_i
// Back: dl[i, t] = +-m (dloss/dh) / pairs (/ n_i), the sign that of the row.
// h is a small difference of large sums, so the sums and everything per pair are held in 64 bits.
//
// A unit is a row's part of up to 1,024 tokens (4,096 in large batches; 8, 64 or 256 lanes); one workgroup turns the units'
// sums into pairs.
// Bound by HBM for large batches (fp32: 9 B read per token forward, 1 read and 4 written back), by launches for small.
#include "bmt_vec.h"
#include "../../include/bmt_hip.h"

namespace bmt {
namespace {

constexpr int kThreads = 256;
constexpr int kPairThreads = 1024;

enum : int32_t { kLogistic = 0, kSquared = 1, kHinge = 2 };

struct RowSum {
    double sum;
    int64_t tokens;
};

template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void preference_sum_kernel(
    int64_t units, int32_t chunks, int32_t part, int32_t time, const typename Elem<T>::Bits *__restrict__ logprob, int64_t logprob_row,
    const typename Elem<T>::Bits *__restrict__ ref, int64_t ref_row, const uint8_t *__restrict__ mask, int64_t mask_row,
    RowSum *__restrict__ sums) {
    typedef typename Elem<T>::Bits Bits;
    constexpr int GROUPS = kThreads / LANES;
    const int lane = threadIdx.x % LANES;
    const int64_t unit = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LANES;
    double sum = 0;
    int tokens = 0;
    if (unit < units) {
        const int64_t row = unit / chunks;
        const int begin = (int)(unit - row * chunks) * part;
        const int end = time - begin < part ? time : begin + part;
        const Bits *lp = logprob + row * logprob_row;
        const Bits *fp = ref ? ref + row * ref_row : nullptr;
        const uint8_t *mp = mask ? mask + row * mask_row : nullptr;
        for (int i = begin + lane * 4; i < end; i += LANES * 4) {
            // the last quad of a row starts further in front and leaves out what it shares with its neighbour, so that
            // all loads are whole; a row of one to three tokens has no room for that
            const int at = time < 4 || i + 4 <= end ? i : end - 4;
            uint32_t m;
            Raw4<T> l, f;
            if (time >= 4) {
                m = mp ? *(const u32_any1 *)(mp + at) : 0x01010101u;
                l.load(lp + at);
                if (fp) f.load(fp + at);
                m &= 0xFFFFFFFFu << (8 * (i - at));
            } else {
                m = load_mask4(mp ? mp + at : nullptr, end - at);
                l.load_some(lp + at, end - at);
                if (fp) f.load_some(fp + at, end - at);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (mask_set(m, k)) sum += (double)l.get(k) - (fp ? (double)f.get(k) : 0.0);
            tokens += mask_count(m);
        }
    }
    sum = lanes_sum(sum, LANES < kWave ? LANES : kWave);
    tokens = lanes_sum(tokens, LANES < kWave ? LANES : kWave);
    if (LANES > kWave) {
        __shared__ RowSum slots[kThreads / kWave];
        if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave] = RowSum{sum, tokens};
        __syncthreads();
        if (threadIdx.x != 0) return;
        RowSum all = slots[0];
        for (int w = 1; w < kThreads / kWave; w++) all.sum += slots[w].sum, all.tokens += slots[w].tokens;
        sums[unit] = all;
    } else if (lane == 0 && unit < units) {
        sums[unit] = RowSum{sum, tokens};
    }
}

__device__ __forceinline__ double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }
__device__ __forceinline__ double sigmoid(double x) { return 1.0 / (1.0 + exp(-x)); }

// slope[0]: 1 / pairs counted, behind it dloss/ds of every row before the mean over pairs.
__global__ __launch_bounds__(kPairThreads) void preference_pair_kernel(int64_t pairs, int32_t chunks, const RowSum *__restrict__ sums,
                                                                       int32_t kind, int32_t average, double beta,
                                                                       double smoothing, float *__restrict__ loss_out,
                                                                       float *__restrict__ chosen, float *__restrict__ rejected,
                                                                       float *__restrict__ slope) {
    double loss = 0, counted = 0;
    for (int64_t p = threadIdx.x; p < pairs; p += kPairThreads) {
        double s[2], per[2];
        int64_t tokens = 0;
        for (int side = 0; side < 2; side++) {
            const RowSum *part = sums + (p + side * pairs) * chunks;
            double sum = 0;
            int64_t n = 0;
            for (int32_t c = 0; c < chunks; c++) sum += part[c].sum, n += part[c].tokens;
            per[side] = average && n > 0 ? 1.0 / (double)n : 1.0;
            s[side] = sum * per[side];
            tokens += n;
        }
        chosen[p] = (float)(beta * s[0]);
        rejected[p] = (float)(beta * s[1]);
        const double h = s[0] - s[1], x = beta * h;
        double one = 0, d = 0;
        if (kind == kLogistic) {
            // a side without weight adds nothing, not 0 * inf: a rejected answer of probability 0 has the margin +inf, the loss 0
            one = (smoothing < 1.0 ? (1.0 - smoothing) * softplus(-x) : 0.0) + (smoothing > 0.0 ? smoothing * softplus(x) : 0.0);
            d = beta * (smoothing * sigmoid(x) - (1.0 - smoothing) * sigmoid(-x));
        } else if (kind == kSquared) {
            const double off = h - 0.5 / beta;
            one = off * off;
            d = 2.0 * off;
        } else {
            one = x >= 1.0 ? 0.0 : 1.0 - x;              // a NaN margin gives a NaN loss
            d = x >= 1.0 ? 0.0 : -beta;
        }
        if (tokens > 0) loss += one, counted += 1.0;
        slope[1 + p] = (float)(d * per[0]);
        slope[1 + p + pairs] = (float)(-d * per[1]);
    }
    __shared__ double slots[kPairThreads / kWave][2];
    loss = lanes_sum(loss, kWave);
    counted = lanes_sum(counted, kWave);
    if (threadIdx.x % kWave == 0) slots[threadIdx.x / kWave][0] = loss, slots[threadIdx.x / kWave][1] = counted;
    __syncthreads();
    if (threadIdx.x == 0) {
        double l = 0, c = 0;
        for (int w = 0; w < kPairThreads / kWave; w++) l += slots[w][0], c += slots[w][1];
        const double share = c > 0 ? 1.0 / c : 0.0;       // no pair counts: loss 0
        loss_out[0] = (float)(l * share);
        slope[0] = (float)share;
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void preference_backward_kernel(int32_t time, int64_t quads_per_row, int64_t quads,
                                                                       const float *__restrict__ slope,
                                                                       const float *__restrict__ upstream,
                                                                       const uint8_t *__restrict__ mask, int64_t mask_row,
                                                                       typename Elem<T>::Bits *__restrict__ grad) {
    const int64_t q = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (q >= quads) return;
    const int64_t row = q / quads_per_row;
    const int i = (int)(q - row * quads_per_row) * 4, count = time - i;
    const uint32_t m = load_mask4(mask ? mask + row * mask_row + i : nullptr, count);
    const float v = slope[1 + row] * (upstream[0] * slope[0]);
    float g[4];
#pragma unroll
    for (int k = 0; k < 4; k++) g[k] = mask_set(m, k) ? v : 0.f;
    store4<T>(grad + row * (int64_t)time + i, count, g);
}

// Tokens of a unit: one step of a workgroup's lanes up to 4,096 units, four beyond.
int64_t part_of(int64_t pairs, int64_t time) { return 2 * pairs * ((time + 1023) / 1024) <= 4096 ? 1024 : 4096; }
int64_t chunks_of(int64_t pairs, int64_t time) { return time <= 0 ? 1 : (time + part_of(pairs, time) - 1) / part_of(pairs, time); }

// Lanes to a row of up to 1,024 tokens, or to a part of a longer one: eight lanes for up to 32 tokens (four each), a wave
// for up to 256; up to 1,024 a workgroup while there are few rows, where it is the latency that counts, and a wave when
// there are many; a workgroup for a part.
int lanes_of(int64_t rows, int64_t time) { return time <= 32 ? 8 : time <= 256 || (time <= 1024 && rows >= 4096) ? 64 : kThreads; }

bool fits(int64_t pairs, int64_t time) {
    return pairs <= 0x3FFFFFFF && time <= 0x3FFFFFFF && launch_fits(2 * pairs * ((time + 3) / 4) / kThreads + 1, kThreads) &&
           launch_fits(2 * pairs * chunks_of(pairs, time) + kThreads, lanes_of(2 * pairs, time));
}

template <typename T, int LANES>
void sum_launch(int64_t rows, int64_t time, const void *logprob, int64_t logprob_row, const void *ref, int64_t ref_row,
                const void *mask, int64_t mask_row, RowSum *sums, hipStream_t s) {
    const int64_t chunks = chunks_of(rows / 2, time), units = rows * chunks, groups = kThreads / LANES;
    typedef typename Elem<T>::Bits Bits;
    hipLaunchKernelGGL((preference_sum_kernel<T, LANES>), dim3((unsigned)((units + groups - 1) / groups)), dim3(kThreads), 0, s,
                       units, (int32_t)chunks, (int32_t)part_of(rows / 2, time), (int32_t)time, (const Bits *)logprob, logprob_row,
                       (const Bits *)ref, ref_row, (const uint8_t *)mask, mask_row, sums);
}
template <typename T>
void sum_pick(int64_t rows, int64_t time, const void *logprob, int64_t logprob_row, const void *ref, int64_t ref_row,
              const void *mask, int64_t mask_row, RowSum *sums, hipStream_t s) {
    const int lanes = lanes_of(rows, time);
    if (lanes == 8) sum_launch<T, 8>(rows, time, logprob, logprob_row, ref, ref_row, mask, mask_row, sums, s);
    else if (lanes == 64) sum_launch<T, 64>(rows, time, logprob, logprob_row, ref, ref_row, mask, mask_row, sums, s);
    else sum_launch<T, 256>(rows, time, logprob, logprob_row, ref, ref_row, mask, mask_row, sums, s);
}

}  // namespace
}  // namespace bmt

extern "C" int64_t preference_loss_workspace_doubles(int64_t pairs, int64_t time) {
    if (pairs <= 0 || !bmt::fits(pairs, time)) return 1;
    return 2 * pairs * bmt::chunks_of(pairs, time) * 2;
}

extern "C" int preference_loss_forward_launcher(int64_t pairs, int64_t time, int32_t type, const void *logprob, int64_t logprob_row,
                                                const void *ref_logprob, int64_t ref_row, const void *mask, int64_t mask_row,
                                                int32_t kind, int32_t average, double beta, double label_smoothing,
                                                void *workspace, void *loss, void *chosen, void *rejected, void *slope,
                                                void *stream) {
    using namespace bmt;
    const char *who = "preference_loss_forward_launcher";
    if (pairs < 0 || time < 0) return refuse(who, "negative size");
    if (kind < kLogistic || kind > kHinge) return refuse(who, "unknown kind of loss");
    if (type != kFp32 && type != kFp16 && type != kBf16) return refuse(who, "unknown type code");
    if (!(beta > 0) || !(beta <= 1e30)) return refuse(who, "beta must be positive and finite");
    if (!(label_smoothing >= 0 && label_smoothing <= 1)) return refuse(who, "label_smoothing must be in [0, 1]");
    if (!fits(pairs, time)) return refuse(who, "too many tokens for one launch");
    if (!loss || !workspace || !slope || (pairs > 0 && (!chosen || !rejected || (time > 0 && !logprob))))
        return refuse(who, "null pointer");
    if ((uintptr_t)workspace % 8 || ((uintptr_t)loss | (uintptr_t)chosen | (uintptr_t)rejected | (uintptr_t)slope) % 4)
        return refuse(who, "misaligned output");
    if (((uintptr_t)logprob | (uintptr_t)ref_logprob) % (type == kFp32 ? 4 : 2)) return refuse(who, "misaligned input");
    hipStream_t s = (hipStream_t)stream;
    RowSum *sums = (RowSum *)workspace;
    if (pairs > 0) {           // rows without a column give units without tokens
        if (type == kFp32) sum_pick<Single>(2 * pairs, time, logprob, logprob_row, ref_logprob, ref_row, mask, mask_row, sums, s);
        else if (type == kFp16) sum_pick<Half>(2 * pairs, time, logprob, logprob_row, ref_logprob, ref_row, mask, mask_row, sums, s);
        else sum_pick<BFloat16>(2 * pairs, time, logprob, logprob_row, ref_logprob, ref_row, mask, mask_row, sums, s);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return fail((int)e, who, e);
    }
    hipLaunchKernelGGL(preference_pair_kernel, dim3(1), dim3(kPairThreads), 0, s, pairs, (int32_t)chunks_of(pairs, time), sums,
                       kind, average, beta, label_smoothing, (float *)loss, (float *)chosen, (float *)rejected, (float *)slope);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}

extern "C" int preference_loss_backward_launcher(int64_t pairs, int64_t time, int32_t type, const void *slope,
                                                 const void *upstream, const void *mask, int64_t mask_row, void *grad_logprob,
                                                 void *stream) {
    using namespace bmt;
    const char *who = "preference_loss_backward_launcher";
    if (pairs <= 0 || time <= 0) return 0;
    if (!fits(pairs, time)) return refuse(who, "too many tokens for one launch");
    if (type != kFp32 && type != kFp16 && type != kBf16) return refuse(who, "unknown type code");
    if (!slope || !upstream || !grad_logprob) return refuse(who, "null pointer");
    if ((uintptr_t)grad_logprob % (type == kFp32 ? 4 : 2) || ((uintptr_t)slope | (uintptr_t)upstream) % 4)
        return refuse(who, "misaligned pointer");
    const int64_t per_row = (time + 3) / 4, quads = 2 * pairs * per_row;
    const dim3 grid((unsigned)((quads + kThreads - 1) / kThreads));
    hipStream_t s = (hipStream_t)stream;
#define BMT_LAUNCH(T)                                                                                                       \
    hipLaunchKernelGGL((preference_backward_kernel<T>), grid, dim3(kThreads), 0, s, (int32_t)time, per_row, quads,          \
                       (const float *)slope, (const float *)upstream, (const uint8_t *)mask, mask_row,                       \
                       (Elem<T>::Bits *)grad_logprob)
    if (type == kFp32) BMT_LAUNCH(Single);
    else if (type == kFp16) BMT_LAUNCH(Half);
    else BMT_LAUNCH(BFloat16);
#undef BMT_LAUNCH
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : fail((int)e, who, e);
}
