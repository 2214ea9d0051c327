// balance.cu: the balance loss of a mixture-of-experts router, with the per-expert counts and the
// gradient of the router's logits.
//
// With f_e the share of the choices that fell on expert e and p = softmax(z) of a row:
//     loss = w E (1/n) sum_i sum_e f_e p_ie,     dloss / dz_ie = w E / n p_ie (f_e - sum_e' f_e' p_ie')
// so a row needs f and itself alone: its share of the loss is the same dot product that its gradient
// subtracts. f needs every choice of every row first: one launch counts, the next does the rows.

#include "loss_common.cuh"

namespace b200amp
{

constexpr int BALANCE_THREADS = 256;

struct BalanceArgs
{
    const void *logits;
    void *dlogits;
    long long ld, dld, rows;
    int experts;
    const int *chosen;
    int k;
    const int *targets;
    double weight;
    int accumulate, add_to_state;
    b200amp_step_state *st;
    int *counts;
    float *loss;
    LossWorkspace *ws;
};

// Integer sums, so the order of the atomics does not show in the result.
__global__ void __launch_bounds__(BALANCE_THREADS) balance_count_kernel(BalanceArgs a)
{
    __shared__ unsigned int bins[B200AMP_MAX_EXPERTS];
    for (int e = threadIdx.x; e < a.experts; e += BALANCE_THREADS)
    {
        bins[e] = 0u;
    }
    __syncthreads();
    const long long stride = static_cast<long long>(gridDim.x) * BALANCE_THREADS;
    const long long first = static_cast<long long>(blockIdx.x) * BALANCE_THREADS + threadIdx.x;
    bool beyond = false;
    for (long long i = first; i < a.rows * a.k; i += stride)
    {
        if (a.targets == nullptr || a.targets[i / a.k] >= 0)
        {
            const int e = a.chosen[i];
            beyond = beyond || e >= a.experts;
            if (e >= 0 && e < a.experts)
            {
                atomicAdd(&bins[e], 1u);
            }
        }
    }
    unsigned int mine = 0u;
    for (long long i = first; i < a.rows; i += stride)
    {
        mine += a.targets == nullptr || a.targets[i] >= 0 ? 1u : 0u;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0 && mine != 0u)
    {
        atomicAdd(&a.ws->rows_counted, mine);
    }
    if (__syncthreads_or(beyond) && threadIdx.x == 0)
    {
        atomicOr(&a.ws->beyond, 1u);
    }
    for (int e = threadIdx.x; e < a.experts; e += BALANCE_THREADS)
    {
        if (bins[e] != 0u)
        {
            atomicAdd(&a.ws->counts[e], bins[e]);
        }
    }
}

// A warp a row.
template <typename T>
__global__ void __launch_bounds__(BALANCE_THREADS) balance_rows_kernel(BalanceArgs a)
{
    __shared__ float share[B200AMP_MAX_EXPERTS];
    __shared__ double scratch[BALANCE_THREADS / 32];
    __shared__ int last_block;
    const int lane = threadIdx.x & 31;
    const unsigned int n = a.ws->rows_counted;
    const bool beyond = a.ws->beyond != 0u;
    const double n_or_1 = n > 0u ? n : 1u;
    for (int e = threadIdx.x; e < a.experts; e += BALANCE_THREADS)
    {
        share[e] = beyond ? NAN : static_cast<float>(a.ws->counts[e] / (n_or_1 * a.k));
    }
    __syncthreads();
    const double factor = a.weight * a.experts / n_or_1;
    const float grad_factor = static_cast<float>(factor * a.st->loss_scale);
    const float log2e = 1.4426950408889634f;
    double mine = 0.0;
    const long long warps = static_cast<long long>(gridDim.x) * (BALANCE_THREADS / 32);
    for (long long row = static_cast<long long>(blockIdx.x) * (BALANCE_THREADS / 32) + (threadIdx.x >> 5);
         row < a.rows; row += warps)
    {
        const T *z = static_cast<const T *>(a.logits) + row * a.ld;
        T *dz = a.dlogits != nullptr ? static_cast<T *>(a.dlogits) + row * a.dld : nullptr;
        if (a.targets != nullptr && a.targets[row] < 0)
        {
            for (int e = lane; dz != nullptr && a.accumulate == 0 && e < a.experts; e += 32)
            {
                dz[e] = from_float<T>(0.0f);
            }
            continue;
        }
        float m = -INFINITY;
        for (int e = lane; e < a.experts; e += 32)
        {
            m = max_nan(m, to_float(z[e]));
        }
        m = warp_max_nan(m);
        float sum = 0.0f, dot = 0.0f;
        for (int e = lane; e < a.experts; e += 32)
        {
            const float p = exp2_fast((to_float(z[e]) - m) * log2e);
            sum += p;
            dot = fmaf(p, share[e], dot);
        }
        sum = warp_sum_f32(sum);
        dot = warp_sum_f32(dot) / sum;
        mine += lane == 0 ? static_cast<double>(dot) : 0.0;
        const float f = grad_factor / sum;
        for (int e = lane; dz != nullptr && e < a.experts; e += 32)
        {
            const float p = exp2_fast((to_float(z[e]) - m) * log2e);
            const float g = f * p * (share[e] - dot);
            dz[e] = from_float<T>(a.accumulate != 0 ? to_float(dz[e]) + g : g);
        }
    }
    mine = block_sum_f64<BALANCE_THREADS>(mine, scratch);
    if (threadIdx.x == 0)
    {
        a.ws->partial[blockIdx.x] = mine;
    }
    if (!take_last_ticket(&a.ws->balance_ticket, gridDim.x, &last_block))
    {
        return;
    }
    double total = 0.0;
    for (unsigned int b = threadIdx.x; b < gridDim.x; b += BALANCE_THREADS)
    {
        total += __ldcg(&a.ws->partial[b]);
    }
    total = block_sum_f64<BALANCE_THREADS>(total, scratch);
    for (int e = threadIdx.x; e < a.experts; e += BALANCE_THREADS)
    {
        a.counts[e] = static_cast<int>(a.ws->counts[e]);
        a.ws->counts[e] = 0u;
    }
    if (threadIdx.x == 0)
    {
        const float loss = beyond ? NAN : static_cast<float>(factor * total);
        a.loss[0] = loss;
        if (a.add_to_state != 0)
        {
            a.st->loss += loss;
        }
        a.ws->rows_counted = 0u;
        a.ws->beyond = 0u;
    }
}

template <typename T>
static int launch_balance(const BalanceArgs &a, int sms, cudaStream_t stream)
{
    const long long work = a.rows * a.k;
    const long long count_blocks = (work + 4 * BALANCE_THREADS - 1) / (4 * BALANCE_THREADS);
    const int count_grid = static_cast<int>(count_blocks < 1 ? 1 : count_blocks < sms ? count_blocks : sms);
    balance_count_kernel<<<count_grid, BALANCE_THREADS, 0, stream>>>(a);
    B200AMP_LAUNCHED();
    const long long blocks = (a.rows + BALANCE_THREADS / 32 - 1) / (BALANCE_THREADS / 32);
    const long long most = 8ll * sms < 2368 ? 8ll * sms : 2368;
    const int grid = static_cast<int>(blocks < 1 ? 1 : blocks < most ? blocks : most);
    balance_rows_kernel<T><<<grid, BALANCE_THREADS, 0, stream>>>(a);
    B200AMP_LAUNCHED();
    return B200AMP_OK;
}

} // namespace b200amp

using namespace b200amp;

extern "C" B200AMP_API int b200amp_balance_loss(const void *logits, long long ld, void *dlogits, long long dld, int dtype,
                                                long long rows, int experts, const int *chosen, int k,
                                                const int *targets, double weight, int accumulate, int add_to_state,
                                                b200amp_step_state *st, int *counts, float *loss, void *workspace,
                                                b200amp_stream s)
{
    B200AMP_REQUIRE(dtype_known(dtype), "balance_loss: dtype %d is none of F16, BF16, F32", dtype);
    B200AMP_REQUIRE(experts >= 1 && experts <= B200AMP_MAX_EXPERTS && experts <= ld,
                    "balance_loss: %d experts, ld %lld: need 1..%d, at most ld", experts, ld, B200AMP_MAX_EXPERTS);
    B200AMP_REQUIRE(k >= 1 && k <= 1024, "balance_loss: k = %d, must be 1..1024", k);
    B200AMP_REQUIRE(rows >= 0 && rows <= INT_MAX / k, "balance_loss: %lld rows of %d choices: need rows * k < 2^31", rows,
                    k);
    B200AMP_REQUIRE(std::isfinite(weight), "balance_loss: weight %g", weight);
    const size_t size = static_cast<size_t>(dtype_size(dtype));
    B200AMP_REQUIRE((logits != nullptr && chosen != nullptr) || rows == 0, "balance_loss: logits or chosen is null");
    B200AMP_REQUIRE(aligned(logits, size) && aligned(dlogits, size) && aligned(chosen, 4) && aligned(targets, 4),
                    "balance_loss: an array is not aligned to its element type");
    if (dlogits != nullptr)
    {
        B200AMP_REQUIRE(experts <= dld, "balance_loss: dld %lld is less than %d experts", dld, experts);
        B200AMP_REQUIRE(dlogits != logits || (dld == ld && accumulate == 0),
                        "balance_loss: in place needs dld == ld (%lld, %lld) and accumulate 0", dld, ld);
    }
    B200AMP_REQUIRE(st != nullptr && counts != nullptr && loss != nullptr && workspace != nullptr,
                    "balance_loss: state, counts, loss or workspace is null");
    B200AMP_REQUIRE(aligned(st, 4) && aligned(counts, 4) && aligned(loss, 4) && aligned(workspace, 16),
                    "balance_loss: state, counts, loss or workspace is misaligned");
    const int sms = sm_count();
    if (sms <= 0)
    {
        return B200AMP_ERR_CUDA;
    }
    const BalanceArgs a = {logits, dlogits, ld, dld, rows, experts, chosen, k, targets, weight, accumulate,
                           add_to_state, st, counts, loss, static_cast<LossWorkspace *>(workspace)};
    switch (dtype)
    {
    case B200AMP_F16:
        return launch_balance<__half>(a, sms, as_stream(s));
    case B200AMP_BF16:
        return launch_balance<__nv_bfloat16>(a, sms, as_stream(s));
    default:
        return launch_balance<float>(a, sms, as_stream(s));
    }
}
