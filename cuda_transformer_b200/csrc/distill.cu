// distill.cu: distillation from a teacher's top logits mixed with the cross-entropy of a label,
// forward and backward, with the gradient multiplied by the step's loss scale.
//
// With x_v = z_v / T - max, S_o the sum of e^x over the columns not listed, S = S_o + the listed
// terms, p_j the teacher's masses, M = sum p + rest:
//     KL  = sum_j p_j (log p_j - x_j) + rest (log rest - log S_o) + M log S
//     dKL / dz_v = 1/T (M e^x / S - p_v)              listed
//                = 1/T e^x (M / S - rest / S_o)       not listed
// The few listed columns (and the label's) are taken out of the row before the fp32 sum and
// added in fp64: an error d of S_o then enters the loss as d (S_o / S - rest) and not as d, which
// matters where student and teacher agree and the loss is a small difference of large terms. The
// sum is taken relative to the maximum of the columns that are left, so that it does not vanish
// where the listed ones stand far above them: S_o divides the rest term.

#include "loss_common.cuh"

namespace b200amp
{

constexpr int DISTILL_THREADS = 512;

struct DistillArgs
{
    const void *logits;
    void *dlogits;
    long long ld, dld, rows;
    int vocab, cols;
    const int *targets;
    const void *values;
    const int *indices;
    const float *lse;
    int value_dtype, k;
    double temperature, soft, hard;
    b200amp_step_state *st;
    float *row_loss;
    LossWorkspace *ws;
};

// Rows that count: every block counts for itself, as the gradient needs the number from its first row on.
template <int THREADS>
__device__ __forceinline__ long long count_rows(const int *targets, long long rows, double *scratch)
{
    if (targets == nullptr)
    {
        return rows;
    }
    int mine = 0;
    for (long long i = threadIdx.x; i < rows; i += THREADS)
    {
        mine += targets[i] >= 0 ? 1 : 0;
    }
    return static_cast<long long>(block_sum_f64<THREADS>(mine, scratch));
}

// One block a row, three sweeps over it in global memory (maximum, sums, gradient). A bit a column in
// shared memory marks what is listed.
template <typename T>
__global__ void __launch_bounds__(DISTILL_THREADS) distill_rows_kernel(DistillArgs a)
{
    extern __shared__ unsigned int marked[];
    __shared__ double scratch[DISTILL_THREADS / 32];
    __shared__ int last_block;
    const int tid = threadIdx.x;
    const long long n_valid = count_rows<DISTILL_THREADS>(a.targets, a.rows, scratch);
    const double grad_scale = static_cast<double>(a.st->loss_scale) / static_cast<double>(n_valid > 0 ? n_valid : 1);
    const double inv_t = 1.0 / a.temperature;
    const double log2e = 1.4426950408889634;
    const float c_t = static_cast<float>(log2e * inv_t), c_1 = static_cast<float>(log2e);
    const int words = (a.vocab + 31) / 32;
    const float inf = INFINITY;

    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x)
    {
        const T *z = static_cast<const T *>(a.logits) + row * a.ld;
        T *dz = a.dlogits != nullptr ? static_cast<T *>(a.dlogits) + row * a.dld : nullptr;
        const int y = a.targets != nullptr ? a.targets[row] : 0;
        if (y < 0)
        {
            for (int v = tid; dz != nullptr && v < a.cols; v += DISTILL_THREADS)
            {
                dz[v] = from_float<T>(0.0f);
            }
            if (tid == 0)
            {
                a.row_loss[row] = 0.0f;
            }
            continue;
        }
        const int *index = a.indices + row * a.k;
        const bool hard = a.hard != 0.0;

        // what the teacher lists
        for (int w = tid; w < words; w += DISTILL_THREADS)
        {
            marked[w] = 0u;
        }
        __syncthreads();
        bool bad = hard && y >= a.vocab, twice = false;
        float t_max = -inf;
        for (int j = tid; j < a.k; j += DISTILL_THREADS)
        {
            const int v = index[j];
            bad = bad || v >= a.vocab;
            if (v >= 0 && v < a.vocab)
            {
                t_max = max_nan(t_max, load_typed(a.values, a.value_dtype, row * a.k + j));
                twice = twice || (atomicOr(&marked[v >> 5], 1u << (v & 31)) >> (v & 31) & 1u) != 0;
            }
        }
        const bool any_bad = __syncthreads_or(bad) != 0;
        const bool any_twice = __syncthreads_or(twice) != 0;
        t_max = block_max_nan<DISTILL_THREADS>(t_max, scratch);
        const bool label_in = hard && y < a.vocab;
        const bool label_listed = label_in && (marked[y >> 5] >> (y & 31) & 1u) != 0;
        __syncthreads();
        if (tid == 0 && label_in)
        {
            marked[y >> 5] |= 1u << (y & 31);
        }
        __syncthreads();

        // the teacher's normaliser: its lse, or the sum over what it lists
        double log_norm;
        const double shift = a.lse != nullptr ? 0.0 : (t_max > -inf || t_max != t_max ? t_max * inv_t : 0.0);
        if (a.lse != nullptr)
        {
            log_norm = a.lse[row];
        }
        else
        {
            double mine = 0.0;
            for (int j = tid; j < a.k; j += DISTILL_THREADS)
            {
                if (index[j] >= 0)
                {
                    mine += exp(load_typed(a.values, a.value_dtype, row * a.k + j) * inv_t - shift);
                }
            }
            mine = block_sum_f64<DISTILL_THREADS>(mine, scratch);
            log_norm = mine == 0.0 ? 0.0 : log(mine);
        }

        // maximum of the columns that are not marked, and the sums relative to it
        float m_u = -inf;
        for (int v = tid; v < a.vocab; v += DISTILL_THREADS)
        {
            if ((marked[v >> 5] >> (v & 31) & 1u) == 0)
            {
                m_u = max_nan(m_u, to_float(z[v]));
            }
        }
        m_u = block_max_nan<DISTILL_THREADS>(m_u, scratch);
        const float m_sub = m_u == -inf ? 0.0f : m_u;       // nothing but -inf: every term is 0
        float sum_t = 0.0f, sum_1 = 0.0f;
        for (int v = tid; v < a.vocab; v += DISTILL_THREADS)
        {
            if ((marked[v >> 5] >> (v & 31) & 1u) == 0)
            {
                const float d = to_float(z[v]) - m_sub;
                sum_t += exp2_fast(d * c_t);
                sum_1 += hard ? exp2_fast(d * c_1) : 0.0f;
            }
        }

        // maximum of the row
        const float z_y = label_in ? to_float(z[y]) : -inf;
        const float m_o = label_listed ? m_u : max_nan(m_u, z_y);           // of the columns not listed
        float m_l = -inf;
        for (int j = tid; j < a.k; j += DISTILL_THREADS)
        {
            if (index[j] >= 0 && index[j] < a.vocab)
            {
                m_l = max_nan(m_l, to_float(z[index[j]]));
            }
        }
        const float m = max_nan(block_max_nan<DISTILL_THREADS>(m_l, scratch), m_o);

        // the listed columns: a column listed more than once counts at its first place, with all its mass
        auto first_place = [&](int j) {
            for (int i = 0; any_twice && i < j; i++)
            {
                if (index[i] == index[j])
                {
                    return false;
                }
            }
            return true;
        };
        auto log_mass = [&](int j) {
            double lp = load_typed(a.values, a.value_dtype, row * a.k + j) * inv_t - shift - log_norm;
            if (any_twice)
            {
                double p = 0.0;
                for (int i = j; i < a.k; i++)
                {
                    if (index[i] == index[j])
                    {
                        p += exp(load_typed(a.values, a.value_dtype, row * a.k + i) * inv_t - shift - log_norm);
                    }
                }
                lp = log(p);
            }
            return lp;
        };
        double mass = 0.0, part = 0.0, listed_t = 0.0, listed_1 = 0.0;
        for (int j = tid; j < a.k; j += DISTILL_THREADS)
        {
            const int v = index[j];
            if (v < 0 || v >= a.vocab || !first_place(j))
            {
                continue;
            }
            const double lp = log_mass(j), p = exp(lp);
            const double d = static_cast<double>(to_float(z[v])) - static_cast<double>(m);
            mass += p;
            part += p != 0.0 ? p * (lp - d * inv_t) : 0.0;
            listed_t += exp(d * inv_t);
            listed_1 += hard ? exp(d) : 0.0;
        }
        mass = block_sum_f64<DISTILL_THREADS>(mass, scratch);
        part = block_sum_f64<DISTILL_THREADS>(part, scratch);
        listed_t = block_sum_f64<DISTILL_THREADS>(listed_t, scratch);
        listed_1 = block_sum_f64<DISTILL_THREADS>(listed_1, scratch);
        const double u_t = block_sum_f64<DISTILL_THREADS>(static_cast<double>(sum_t), scratch);
        const double u_1 = block_sum_f64<DISTILL_THREADS>(static_cast<double>(sum_1), scratch);
        // e^((from - to) * f), 0 from -inf
        auto shifted = [&](float from, float to, double f) {
            return from == -inf ? 0.0 : exp((static_cast<double>(from) - static_cast<double>(to)) * f);
        };
        // not listed, relative to their own maximum, then all relative to the row's
        const double u_in_o = shifted(m_u, m_o, inv_t);
        const double others = u_t * u_in_o + (label_listed ? 0.0 : shifted(z_y, m_o, inv_t));
        const double o_in_all = shifted(m_o, m, inv_t);
        const double total = others * o_in_all + listed_t;
        const double u_in_all_1 = shifted(m_u, m, 1.0);
        const double total_1 = u_1 * u_in_all_1 + listed_1 + (label_listed ? 0.0 : shifted(z_y, m, 1.0));
        const double rest = a.lse != nullptr && a.k > 0 && others > 0.0 ? fmax(0.0, 1.0 - mass) : 0.0;
        const double whole = mass + rest;
        const double log_o = rest > 0.0 ? log(others) + (static_cast<double>(m_o) - static_cast<double>(m)) * inv_t : 0.0;
        const double d_y = static_cast<double>(z_y) - static_cast<double>(m);

        // loss
        double loss = 0.0;
        if (a.k > 0)
        {
            loss = part + whole * log(total) + (rest > 0.0 ? rest * (log(rest) - log_o) : 0.0);
            loss *= a.soft;
        }
        if (hard)
        {
            loss += a.hard * (log(total_1) - d_y);
        }
        const double poison = any_bad || !isfinite(m) ? nan("") : 0.0;
        if (tid == 0)
        {
            a.row_loss[row] = static_cast<float>(loss + poison);
        }
        if (dz == nullptr)
        {
            __syncthreads();                    // marked is cleared for the next row
            continue;
        }

        // gradient
        const double soft_scale = a.k > 0 ? grad_scale * a.soft * inv_t : 0.0;
        const double hard_scale = hard ? grad_scale * a.hard : 0.0;
        const double per_o = whole * o_in_all / total - (rest > 0.0 ? rest / others : 0.0);     // of e^(x - m_o)
        const float f_t = static_cast<float>(soft_scale * per_o * u_in_o + poison);
        const float f_1 = hard ? static_cast<float>(hard_scale * u_in_all_1 / total_1) : 0.0f;
        for (int v = tid; v < a.cols; v += DISTILL_THREADS)
        {
            if (v >= a.vocab)
            {
                dz[v] = from_float<T>(0.0f);
            }
            else if ((marked[v >> 5] >> (v & 31) & 1u) == 0)
            {
                const float d = to_float(z[v]) - m_sub;
                float g = exp2_fast(d * c_t) * f_t;
                if (hard)
                {
                    g += exp2_fast(d * c_1) * f_1;
                }
                dz[v] = from_float<T>(g);
            }
        }
        for (int j = tid; j < a.k; j += DISTILL_THREADS)
        {
            const int v = index[j];
            if (v < 0 || v >= a.vocab || !first_place(j))
            {
                continue;
            }
            const double d = static_cast<double>(to_float(z[v])) - static_cast<double>(m);
            double g = soft_scale * (whole * exp(d * inv_t) / total - exp(log_mass(j)));
            if (hard)
            {
                g += hard_scale * (exp(d) - (v == y ? total_1 : 0.0)) / total_1;
            }
            dz[v] = from_float<T>(static_cast<float>(g + poison));
        }
        if (tid == 0 && label_in && !label_listed)
        {
            const double g = hard_scale * (exp(d_y) - total_1) / total_1 + soft_scale * per_o * shifted(z_y, m_o, inv_t);
            dz[y] = from_float<T>(static_cast<float>(g + poison));
        }
        __syncthreads();                        // marked is cleared for the next row
    }

    if (!take_last_ticket(&a.ws->distill_ticket, gridDim.x, &last_block))
    {
        return;
    }
    double mine = 0.0;
    for (long long i = tid; i < a.rows; i += DISTILL_THREADS)
    {
        mine += static_cast<double>(__ldcg(&a.row_loss[i]));
    }
    mine = block_sum_f64<DISTILL_THREADS>(mine, scratch);
    if (tid == 0)
    {
        a.st->loss = static_cast<float>(mine / static_cast<double>(n_valid > 0 ? n_valid : 1));
        a.st->n_valid = static_cast<int>(n_valid);
    }
}

template <typename T>
static int launch_distill(const DistillArgs &a, int sms, cudaStream_t stream)
{
    const int smem = (a.vocab + 31) / 32 * 4;
    B200AMP_CUDA(cudaFuncSetAttribute(distill_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const long long most = 4ll * sms;
    const int grid = static_cast<int>(a.rows < 1 ? 1 : a.rows < most ? a.rows : most);
    distill_rows_kernel<T><<<grid, DISTILL_THREADS, smem, stream>>>(a);
    B200AMP_LAUNCHED();
    return B200AMP_OK;
}

} // namespace b200amp

using namespace b200amp;

extern "C" B200AMP_API int b200amp_loss_workspace_init(void *workspace, b200amp_stream s)
{
    B200AMP_REQUIRE(workspace != nullptr && aligned(workspace, 16), "loss_workspace_init: null or misaligned pointer");
    B200AMP_CUDA(cudaMemsetAsync(workspace, 0, B200AMP_LOSS_WORKSPACE_BYTES, as_stream(s)));
    return B200AMP_OK;
}

extern "C" B200AMP_API int b200amp_distill_loss(const void *logits, long long ld, void *dlogits, long long dld, int dtype,
                                                long long rows, int vocab, int cols, const int *targets,
                                                const void *values, int value_dtype, const int *indices,
                                                const float *lse, int k, double temperature, double soft_weight,
                                                double hard_weight, b200amp_step_state *st, float *row_loss,
                                                void *workspace, b200amp_stream s)
{
    B200AMP_REQUIRE(dtype_known(dtype), "distill_loss: dtype %d is none of F16, BF16, F32", dtype);
    B200AMP_REQUIRE(rows >= 0 && rows <= INT_MAX, "distill_loss: %lld rows, must be 0..%d", rows, INT_MAX);
    B200AMP_REQUIRE(vocab >= 1 && vocab <= cols && cols <= ld, "distill_loss: vocab %d, cols %d, ld %lld: need "
                                                               "1 <= vocab <= cols <= ld", vocab, cols, ld);
    B200AMP_REQUIRE(k >= 0 && k <= B200AMP_MAX_LISTED, "distill_loss: k = %d, must be 0..%d", k, B200AMP_MAX_LISTED);
    B200AMP_REQUIRE(std::isfinite(temperature) && temperature > 0.0 && std::isfinite(static_cast<float>(1.4426950408889634 / temperature)) &&
                        static_cast<float>(1.4426950408889634 / temperature) > 0.0f,
                    "distill_loss: temperature %g", temperature);
    B200AMP_REQUIRE(std::isfinite(soft_weight) && std::isfinite(hard_weight), "distill_loss: weights %g and %g",
                    soft_weight, hard_weight);
    const size_t size = static_cast<size_t>(dtype_size(dtype));
    B200AMP_REQUIRE(logits != nullptr || rows == 0, "distill_loss: logits is null");
    B200AMP_REQUIRE(aligned(logits, size) && aligned(dlogits, size), "distill_loss: logits or dlogits is not aligned "
                                                                     "to its element type");
    if (dlogits != nullptr)
    {
        B200AMP_REQUIRE(cols <= dld, "distill_loss: dld %lld is less than cols %d", dld, cols);
        B200AMP_REQUIRE(dlogits != logits || dld == ld, "distill_loss: in place needs dld == ld (%lld, %lld)", dld, ld);
    }
    B200AMP_REQUIRE(targets != nullptr || hard_weight == 0.0 || rows == 0, "distill_loss: a hard weight needs targets");
    B200AMP_REQUIRE(aligned(targets, 4), "distill_loss: targets is not 4-byte aligned");
    if (soft_weight == 0.0)
    {
        k = 0;
    }
    if (k > 0 && rows > 0)
    {
        B200AMP_REQUIRE(values != nullptr && indices != nullptr, "distill_loss: k = %d needs values and indices", k);
        B200AMP_REQUIRE(dtype_known(value_dtype), "distill_loss: value dtype %d", value_dtype);
        B200AMP_REQUIRE(aligned(values, dtype_size(value_dtype)) && aligned(indices, 4) && aligned(lse, 4),
                        "distill_loss: values, indices or lse is misaligned");
    }
    B200AMP_REQUIRE(st != nullptr && (row_loss != nullptr || rows == 0) && workspace != nullptr,
                    "distill_loss: state, row_loss or workspace is null");
    B200AMP_REQUIRE(aligned(st, 4) && aligned(row_loss, 4) && aligned(workspace, 16),
                    "distill_loss: state, row_loss or workspace is misaligned");
    if (vocab > 1 << 20)
    {
        set_error("distill_loss: a vocabulary of %d is beyond the maximum of %d", vocab, 1 << 20);
        return B200AMP_ERR_LIMIT;
    }
    const int sms = sm_count();
    if (sms <= 0)
    {
        return B200AMP_ERR_CUDA;
    }
    DistillArgs a = {logits, dlogits, ld, dld, rows, vocab, cols, targets, values, indices, lse, value_dtype, k,
                     temperature, soft_weight, hard_weight, st, row_loss, static_cast<LossWorkspace *>(workspace)};
    switch (dtype)
    {
    case B200AMP_F16:
        return launch_distill<__half>(a, sms, as_stream(s));
    case B200AMP_BF16:
        return launch_distill<__nv_bfloat16>(a, sms, as_stream(s));
    default:
        return launch_distill<float>(a, sms, as_stream(s));
    }
}
