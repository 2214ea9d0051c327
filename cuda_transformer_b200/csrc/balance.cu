// balance.cu: the balance loss of a mixture-of-experts router, with the per-expert counts and the
// gradient of the router's logits.
//
// With f_e the share of the choices that fell on expert e and p = softmax(z) of a row:
//     loss = w E (1/n) sum_i sum_e f_e p_ie,     dloss / dz_ie = w E / n p_ie (f_e - sum_e' f_e' p_ie')
// so a row needs f and itself alone: its share of the loss is the same dot product that its gradient
// subtracts. f needs every choice of every row first: one launch counts, the next does the rows (its blocks start
// while the first still counts, and have their first rows in registers by then). Few choices are counted by every block
// of the rows' launch for itself, which saves the other.

#include "row_tile.cuh"

namespace b200amp
{

constexpr int BALANCE_THREADS = 256;
constexpr int COUNT_HERE = 4096;        // choices up to which every block counts for itself: 16 a thread

struct BalanceArgs
{
    const void *logits;
    void *dlogits;
    long long ld, dld;
    int rows, experts;
    const int *chosen;
    int k;
    const int *targets;
    double weight;
    int accumulate, add_to_state;
    b200amp_step_state *st;
    int *counts;
    float *loss;
    LossWorkspace *ws;
    int count_here;
};

// This block's share (of `blocks`) of the choices into bins and of the rows that count into *rows; true where this
// thread met an expert beyond the last. Integer sums, so the order of the atomics does not show.
__device__ __forceinline__ bool count_choices(const BalanceArgs &a, unsigned int block, unsigned int blocks, unsigned int *bins,
                                              unsigned int *rows)
{
    const unsigned int first = block * BALANCE_THREADS + threadIdx.x, stride = blocks * BALANCE_THREADS;
    const unsigned int choices = static_cast<unsigned int>(a.rows) * static_cast<unsigned int>(a.k);
    bool beyond = false;
    constexpr int AT_ONCE = 8;                  // choices of a thread on their way together
    for (unsigned int i = first; i < choices; i += AT_ONCE * stride)
    {
        int e[AT_ONCE], y[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
        {
            const unsigned int at = i + u * stride;     // below 2^31 + 2^20: no wrap
            e[u] = at < choices ? __ldg(&a.chosen[at]) : -1;
            y[u] = at < choices && a.targets != nullptr ? __ldg(&a.targets[at / static_cast<unsigned int>(a.k)]) : 0;
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
        {
            if (e[u] >= 0 && y[u] >= 0)
            {
                beyond = beyond || e[u] >= a.experts;
                if (e[u] < a.experts)
                {
                    atomicAdd(&bins[e[u]], 1u);
                }
            }
        }
    }
    unsigned int mine = 0u;
    for (unsigned int i = first; i < static_cast<unsigned int>(a.rows); i += stride)
    {
        mine += a.targets == nullptr || __ldg(&a.targets[i]) >= 0 ? 1u : 0u;
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if ((threadIdx.x & 31) == 0 && mine != 0u)
    {
        atomicAdd(rows, mine);
    }
    return beyond;
}

__global__ void __launch_bounds__(BALANCE_THREADS) balance_count_kernel(const BalanceArgs a)
{
    __shared__ unsigned int bins[B200AMP_MAX_EXPERTS];
    asm volatile("griddepcontrol.launch_dependents;" : : : "memory");
    for (int e = threadIdx.x; e < a.experts; e += BALANCE_THREADS)
    {
        bins[e] = 0u;
    }
    __syncthreads();
    const bool beyond = count_choices(a, blockIdx.x, gridDim.x, bins, &a.ws->rows_counted);
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

// max.NaN of three, in one instruction
__device__ __forceinline__ float max3_nan(float a, float b, float c)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// ITEMS accesses of VEC elements (a 16-byte vector, or one) a lane, held in registers as pairs for the instructions
// that take two. Access i of lane l starts at element (l + LANES i) VEC.
template <typename T, int VEC, int ITEMS, int LANES>
struct BalanceRow
{
    static constexpr int PAIRS = ITEMS * VEC / 2;
    float2 v[PAIRS];

    static __device__ __forceinline__ int element(int lane, int pair)   // of a pair's first value
    {
        return VEC == 1 ? lane + LANES * 2 * pair : (lane + LANES * (2 * pair / VEC)) * VEC + 2 * pair % VEC;
    }
    static constexpr int STEP = VEC == 1 ? LANES : 1;                   // to its second
    __device__ __forceinline__ void load(const T *z, int lane, int experts, float fill)
    {
        if constexpr (VEC == 1)
        {
#pragma unroll
            for (int i = 0; i < PAIRS; i++)
            {
                const int e = element(lane, i);
                v[i].x = e < experts ? to_float(z[e]) : fill;
                v[i].y = e + STEP < experts ? to_float(z[e + STEP]) : fill;
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < ITEMS; i++)
            {
                const int e = (lane + LANES * i) * VEC;
                float2 f[VEC / 2];
#pragma unroll
                for (int q = 0; q < VEC / 2; q++)
                {
                    f[q] = make_float2(fill, fill);
                }
                if (e < experts)
                {
                    Vec16<T> w;
                    w.w = *reinterpret_cast<const uint4 *>(z + e);
                    unpack(w, f);
                }
#pragma unroll
                for (int q = 0; q < VEC / 2; q++)
                {
                    v[i * (VEC / 2) + q] = f[q];
                }
            }
        }
    }
    __device__ __forceinline__ void store(T *z, int lane, int experts) const
    {
        if constexpr (VEC == 1)
        {
#pragma unroll
            for (int i = 0; i < PAIRS; i++)
            {
                const int e = element(lane, i);
                if (e < experts)
                {
                    z[e] = from_float<T>(v[i].x);
                }
                if (e + STEP < experts)
                {
                    z[e + STEP] = from_float<T>(v[i].y);
                }
            }
        }
        else
        {
#pragma unroll
            for (int i = 0; i < ITEMS; i++)
            {
                const int e = (lane + LANES * i) * VEC;
                if (e < experts)
                {
                    float2 f[VEC / 2];
#pragma unroll
                    for (int q = 0; q < VEC / 2; q++)
                    {
                        f[q] = v[i * (VEC / 2) + q];
                    }
                    Vec16<T> w;
                    pack(w, f);
                    *reinterpret_cast<uint4 *>(z + e) = w.w;
                }
            }
        }
    }
};

// LANES threads a row; a row is read once and stays in registers, with the next one on its way. 65536 rows of 256 fp32
// experts, k 8: 37 us with the counting, 137 MB (the bytes alone 21 us); the counting's latency, about 10 us, is what
// the rows cannot hide.
template <typename T, int VEC, int ITEMS, int LANES>
__global__ void __launch_bounds__(BALANCE_THREADS, ITEMS * VEC <= 16 ? 3 : 1) balance_rows_kernel(const BalanceArgs a)
{
    using Row = BalanceRow<T, VEC, ITEMS, LANES>;
    constexpr int PAIRS = Row::PAIRS;
    __shared__ unsigned int bins[B200AMP_MAX_EXPERTS];
    __shared__ double scratch[BALANCE_THREADS / 32];
    __shared__ unsigned int rows_here;
    __shared__ int last_block;
    constexpr int GROUPS = BALANCE_THREADS / LANES;
    const int lane = threadIdx.x & (LANES - 1);
    const long long stride = static_cast<long long>(gridDim.x) * GROUPS;
    const long long row = static_cast<long long>(blockIdx.x) * GROUPS + threadIdx.x / LANES;
    const T *const logits = static_cast<const T *>(a.logits);

    Row next = {};
    int next_y = -1;
    auto fetch = [&](long long r) {
        next_y = r >= a.rows ? -1 : a.targets != nullptr ? __ldg(&a.targets[r]) : 0;
        if (r < a.rows)
        {
            next.load(logits + r * a.ld, lane, a.experts, -INFINITY);
        }
    };
    fetch(row);

    bool beyond;
    unsigned int n;
    if (a.count_here != 0)
    {
        for (int e = threadIdx.x; e < a.experts; e += BALANCE_THREADS)
        {
            bins[e] = 0u;
        }
        if (threadIdx.x == 0)
        {
            rows_here = 0u;
        }
        __syncthreads();
        beyond = __syncthreads_or(count_choices(a, 0u, 1u, bins, &rows_here)) != 0;
        n = rows_here;
    }
    else
    {
        asm volatile("griddepcontrol.wait;" : : : "memory");    // the counting launch is done and its sums are visible
        for (int e = threadIdx.x; e < a.experts; e += BALANCE_THREADS)
        {
            bins[e] = __ldcg(&a.ws->counts[e]);
        }
        beyond = __ldcg(&a.ws->beyond) != 0u;
        n = __ldcg(&a.ws->rows_counted);
        __syncthreads();
    }
    const double n_or_1 = n > 0u ? n : 1u, per_choice = 1.0 / (n_or_1 * a.k);
    float2 share[PAIRS];
#pragma unroll
    for (int i = 0; i < PAIRS; i++)
    {
        const int e = Row::element(lane, i);
        share[i].x = beyond ? NAN : e < a.experts ? static_cast<float>(bins[e] * per_choice) : 0.0f;
        share[i].y = beyond ? NAN : e + Row::STEP < a.experts ? static_cast<float>(bins[e + Row::STEP] * per_choice) : 0.0f;
    }
    const double factor = a.weight * a.experts / n_or_1;
    const float grad_factor = static_cast<float>(factor * a.st->loss_scale);
    const float log2e = 1.4426950408889634f;
    double loss = 0.0;
    // every thread of a warp stays for the shuffles, those past the last row too
    for (long long at = row; at - static_cast<int>(threadIdx.x & 31) / LANES < a.rows; at += stride)
    {
        Row z = next;
        const int y = next_y;
        fetch(at + stride);
        float m = max_nan(z.v[0].x, z.v[0].y);
#pragma unroll
        for (int i = 1; i < PAIRS; i++)
        {
            m = max3_nan(m, z.v[i].x, z.v[i].y);
        }
#pragma unroll
        for (int offset = LANES / 2; offset > 0; offset >>= 1)
        {
            m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, offset));
        }
        float2 sum = make_float2(0.0f, 0.0f), dots = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < PAIRS; i++)
        {
            const float2 x = mul2(add2(z.v[i], make_float2(-m, -m)), make_float2(log2e, log2e));
            z.v[i] = make_float2(exp2_fast(x.x), exp2_fast(x.y));
            sum = add2(sum, z.v[i]);
            dots = fma2(z.v[i], share[i], dots);
        }
        sum.x += sum.y;
        sum.y = dots.x + dots.y;
#pragma unroll
        for (int offset = LANES / 2; offset > 0; offset >>= 1)
        {
            const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, sum.x, offset), __shfl_xor_sync(0xffffffffu, sum.y, offset));
            sum = add2(sum, other);
        }
        const float inv = __fdividef(1.0f, sum.x), dot = sum.y * inv;
        if (at >= a.rows)
        {
            continue;
        }
        loss += lane == 0 && y >= 0 ? static_cast<double>(dot) : 0.0;
        if (a.dlogits == nullptr || (y < 0 && a.accumulate != 0))
        {
            continue;
        }
        T *const dz = static_cast<T *>(a.dlogits) + at * a.dld;
        const float f = grad_factor * inv;
#pragma unroll
        for (int i = 0; i < PAIRS; i++)
        {
            z.v[i] = mul2(mul2(z.v[i], make_float2(f, f)), add2(share[i], make_float2(-dot, -dot)));
        }
        if (y < 0)
        {
#pragma unroll
            for (int i = 0; i < PAIRS; i++)
            {
                z.v[i] = make_float2(0.0f, 0.0f);       // whatever the row held
            }
        }
        if (a.accumulate != 0)
        {
            Row old;
            old.load(dz, lane, a.experts, 0.0f);
#pragma unroll
            for (int i = 0; i < PAIRS; i++)
            {
                z.v[i] = add2(z.v[i], old.v[i]);
            }
        }
        z.store(dz, lane, a.experts);
    }
    loss = block_sum_f64<BALANCE_THREADS>(loss, scratch);
    if (threadIdx.x == 0)
    {
        a.ws->partial[blockIdx.x] = loss;
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
        a.counts[e] = static_cast<int>(bins[e]);
        a.ws->counts[e] = 0u;
    }
    if (threadIdx.x == 0)
    {
        const float value = beyond ? NAN : static_cast<float>(factor * total);
        a.loss[0] = value;
        if (a.add_to_state != 0)
        {
            a.st->loss += value;
        }
        a.ws->rows_counted = 0u;
        a.ws->beyond = 0u;
    }
}

template <typename T, int VEC, int ITEMS, int LANES>
static int launch_balance(const BalanceArgs &a, int sms, cudaStream_t stream)
{
    if (a.count_here == 0)
    {
        const long long choices = static_cast<long long>(a.rows) * a.k;
        const long long blocks = (choices + 4 * BALANCE_THREADS - 1) / (4 * BALANCE_THREADS);
        balance_count_kernel<<<static_cast<int>(blocks < 2 * sms ? blocks : 2 * sms), BALANCE_THREADS, 0, stream>>>(a);
        B200AMP_LAUNCHED();
    }
    constexpr int GROUPS = BALANCE_THREADS / LANES;
    const long long blocks = (static_cast<long long>(a.rows) + GROUPS - 1) / GROUPS;
    const long long most = 3ll * sms < 2368 ? 3ll * sms : 2368;     // as many as are resident: each has several rows
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(blocks < 1 ? 1 : blocks < most ? blocks : most));
    config.blockDim = dim3(BALANCE_THREADS);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = a.count_here == 0 ? 1 : 0;        // only behind the counting launch, which lets it start early
    B200AMP_CUDA(cudaLaunchKernelEx(&config, balance_rows_kernel<T, VEC, ITEMS, LANES>, a));
    B200AMP_LAUNCHED();
    return B200AMP_OK;
}

template <typename T>
static int launch_balance(BalanceArgs a, cudaStream_t stream)
{
    const int sms = sm_count();
    if (sms <= 0)
    {
        return B200AMP_ERR_CUDA;
    }
    a.count_here = static_cast<long long>(a.rows) * a.k <= COUNT_HERE ? 1 : 0;
    constexpr int N = Vec16<T>::N;
    // 16-byte accesses where every row allows them, else one element at a time
    const bool wide = a.experts % N == 0 && a.ld % N == 0 && aligned(a.logits, 16) &&
                      (a.dlogits == nullptr || (a.dld % N == 0 && aligned(a.dlogits, 16)));
    if (wide)
    {
        // 16 values a lane: with fewer, the shuffles between the lanes and the addresses are most of the instructions
        // (65536 rows of 256 fp32 experts: 4 values 48 us, 8 values 42 us, 16 values 40 us)
        constexpr int ITEMS = 16 / N;
        const int lanes = (a.experts + 15) / 16;
        return lanes <= 1    ? launch_balance<T, N, ITEMS, 1>(a, sms, stream)
               : lanes <= 2  ? launch_balance<T, N, ITEMS, 2>(a, sms, stream)
               : lanes <= 4  ? launch_balance<T, N, ITEMS, 4>(a, sms, stream)
               : lanes <= 8  ? launch_balance<T, N, ITEMS, 8>(a, sms, stream)
               : lanes <= 16 ? launch_balance<T, N, ITEMS, 16>(a, sms, stream)
               : lanes <= 32 ? launch_balance<T, N, ITEMS, 32>(a, sms, stream)
                             : launch_balance<T, N, 2 * ITEMS, 32>(a, sms, stream);
    }
    return a.experts <= 32    ? launch_balance<T, 1, 4, 8>(a, sms, stream)
           : a.experts <= 256 ? launch_balance<T, 1, 8, 32>(a, sms, stream)
                              : launch_balance<T, 1, 32, 32>(a, sms, stream);
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
    const BalanceArgs a = {logits, dlogits, ld, dld, static_cast<int>(rows), experts, chosen, k, targets, weight, accumulate,
                           add_to_state, st, counts, loss, static_cast<LossWorkspace *>(workspace), 0};
    switch (dtype)
    {
    case B200AMP_F16:
        return launch_balance<__half>(a, as_stream(s));
    case B200AMP_BF16:
        return launch_balance<__nv_bfloat16>(a, as_stream(s));
    default:
        return launch_balance<float>(a, as_stream(s));
    }
}
