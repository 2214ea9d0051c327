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

#include "row_tile.cuh"

namespace b200amp
{

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

// What a block knows of its segment of a row; with several blocks a row each sends its own to all.
struct alignas(16) SegmentSums
{
    float m_u;              // maximum of the columns that are neither listed nor the label
    float m_l;              // maximum of the listed ones
    float z_y;              // the label's logit, -inf where it is in another segment
    int label_listed;
    double s_t, s_1;        // sums over the first kind, relative to m_u, at the temperature and at 1
    double l_t, l_1;        // sums over the listed, relative to m_l
    double part, own;       // sum p (log p - (z - m_l) / T), sum p
};

// What the gradient needs of a whole row.
struct RowFactors
{
    float m_u, f_t, f_1;    // a column that is not listed: e^((z - m_u) / T) f_t + e^(z - m_u) f_1
    float m;
    double l_t, l_1;        // a listed one: e^((z - m) / T) l_t + e^(z - m) l_1 - p soft_scale
    double y;               // what the label's column has besides
    double label;           // the label's column where it is not listed
};

// e^((from - to) f), 0 from -inf
__device__ __forceinline__ double shifted(float from, float to, double f)
{
    return from == -INFINITY ? 0.0 : from == to ? 1.0 : exp((static_cast<double>(from) - static_cast<double>(to)) * f);
}

// A cluster a row, the row in its shared memory between the sweeps. Barriers of a block and row: the row has
// arrived; listed columns are taken out; maximum; sums; factors; the gradient is out.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) distill_rows_kernel(const DistillArgs a, const RowPlan plan)
{
    namespace cg = cooperative_groups;
    using Tile = RowTile<T, THREADS>;
    constexpr int N = Tile::N, PAIRS = N / 2, WARPS = THREADS / 32;
    extern __shared__ __align__(16) char dynamic[];
    __shared__ SegmentSums slots[2][MAX_CLUSTER];
    __shared__ RowFactors factors;
    __shared__ double scratch[WARPS];
    __shared__ double warp_sums[WARPS][8];
    __shared__ float2 warp_max[WARPS];
    __shared__ float label_logit;
    __shared__ int label_listed, last_block;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const cg::cluster_group cluster = cg::this_cluster();
    const int blocks = plan.cluster, rank = blocks > 1 ? static_cast<int>(cluster.block_rank()) : 0;
    const float inf = INFINITY;

    const size_t tile_bytes = (static_cast<size_t>(plan.segment) * sizeof(T) + 31) & ~static_cast<size_t>(15);
    Tile tile;
    tile.buf = dynamic;
    double *rec_lp = reinterpret_cast<double *>(dynamic + tile_bytes);      // log p, p, logit and column of what is listed
    double *rec_p = rec_lp + a.k;
    float *rec_z = reinterpret_cast<float *>(rec_p + a.k);
    int *rec_col = reinterpret_cast<int *>(rec_z + a.k);
    unsigned int *marked = reinterpret_cast<unsigned int *>(rec_col + a.k); // a bit a column of the segment
    for (int w = tid; w < plan.segment / 32; w += THREADS)
    {
        marked[w] = 0u;
    }

    const bool hard = a.hard != 0.0;
    const double inv_t = a.k > 0 ? 1.0 / a.temperature : 1.0;      // the label's softmax alone is at 1
    const bool two = hard && a.k > 0 && a.temperature != 1.0;   // two softmaxes of a row
    const double log2e = 1.4426950408889634;
    const float c_t = static_cast<float>(log2e * inv_t), c_1 = static_cast<float>(log2e);
    const int segment_first = rank * plan.segment;
    const long long clusters = gridDim.x / blocks;
    auto row_of = [&](long long row) { return static_cast<const T *>(a.logits) + row * a.ld; };
    auto label_of = [&](long long row) { return a.targets != nullptr ? __ldg(&a.targets[row]) : 0; };

    long long row = blockIdx.x / blocks;
    bool started = false;
    if (row < a.rows && label_of(row) >= 0)
    {
        tile.start(row_of(row), segment_first, plan.segment, a.vocab, a.cols);
        started = true;
    }
    const long long n_valid = count_rows<THREADS>(a.targets, a.rows, scratch);
    const double grad_scale = static_cast<double>(a.st->loss_scale) / static_cast<double>(n_valid > 0 ? n_valid : 1);
    const double soft_scale = a.k > 0 ? grad_scale * a.soft * inv_t : 0.0;
    const double hard_scale = hard ? grad_scale * a.hard : 0.0;
    __syncthreads();
    if (blocks > 1)
    {
        cluster.sync();                         // every block of the cluster runs before one writes to another
    }

    for (int parity = 0; row < a.rows; row += clusters)
    {
        T *out = a.dlogits != nullptr ? static_cast<T *>(a.dlogits) + row * a.dld : nullptr;
        const int y = label_of(row);
        if (y < 0)
        {
            const int held = max(0, min(plan.segment, a.cols - segment_first));
            for (int i = tid; out != nullptr && i < held; i += THREADS)
            {
                out[segment_first + i] = from_float<T>(0.0f);
            }
            if (rank == 0 && tid == 0)
            {
                a.row_loss[row] = 0.0f;
            }
            started = false;
            continue;
        }
        if (!started)
        {
            tile.start(row_of(row), segment_first, plan.segment, a.vocab, a.cols);
        }
        const bool label_in = hard && y < a.vocab;

        // the record, while the row is on its way
        bool twice = false;
        double norm_max = 0.0, log_norm = 0.0;
        if (a.lse == nullptr && a.k > 0)
        {
            float t_max = -inf;
            for (int j = tid; j < a.k; j += THREADS)
            {
                if (a.indices[row * a.k + j] >= 0)
                {
                    t_max = max_nan(t_max, load_typed(a.values, a.value_dtype, row * a.k + j));
                }
            }
            t_max = block_max_nan<THREADS>(t_max, scratch);
            norm_max = t_max == -inf ? 0.0 : t_max * inv_t;
            double sum = 0.0;
            for (int j = tid; j < a.k; j += THREADS)
            {
                if (a.indices[row * a.k + j] >= 0)
                {
                    sum += exp(load_typed(a.values, a.value_dtype, row * a.k + j) * inv_t - norm_max);
                }
            }
            sum = block_sum_f64<THREADS>(sum, scratch);
            log_norm = sum == 0.0 ? 0.0 : log(sum);
        }
        else if (a.lse != nullptr)
        {
            log_norm = a.lse[row];
        }
        double mass = 0.0;
        for (int j = tid; j < a.k; j += THREADS)
        {
            const int v = a.indices[row * a.k + j];
            const bool fits = v >= 0 && v < a.vocab;
            const double lp = load_typed(a.values, a.value_dtype, row * a.k + j) * inv_t - norm_max - log_norm;
            const double p = fits ? exp(lp) : v < 0 ? 0.0 : nan("");    // beyond the vocabulary: the row is NaN
            mass += p;
            rec_lp[j] = lp;
            rec_p[j] = p;
            rec_col[j] = fits ? v : -1;
            if (fits && tile.holds(v))
            {
                const int at = v - segment_first;
                twice = twice || (atomicOr(&marked[at >> 5], 1u << (at & 31)) >> (at & 31) & 1u) != 0;
            }
        }
        if (tid == 0)
        {
            label_logit = -inf;
            label_listed = 0;
        }
        copy_async_wait();
        if (__syncthreads_or(twice) != 0)
        {
            // a column listed more than once keeps its first place, with all its mass
            for (int j = tid; j < a.k; j += THREADS)
            {
                const int v = rec_col[j];
                bool first = true;
                double p = 0.0;
                for (int i = 0; v >= 0 && i < a.k; i++)
                {
                    first = first && !(i < j && rec_col[i] == v);
                    p += rec_col[i] == v ? rec_p[i] : 0.0;
                }
                rec_z[j] = first ? 1.0f : 0.0f;
                rec_lp[j] = log(p);
            }
            __syncthreads();
            for (int j = tid; j < a.k; j += THREADS)
            {
                if (rec_col[j] >= 0)
                {
                    rec_p[j] = exp(rec_lp[j]);
                    rec_col[j] = rec_z[j] != 0.0f ? rec_col[j] : -1;
                }
            }
        }

        // take the listed columns and the label out of the row
        float m_l = -inf;
        for (int j = tid; j < a.k; j += THREADS)
        {
            const int v = rec_col[j];
            if (tile.holds(v))
            {
                const float z = to_float(*tile.at(v));
                *tile.at(v) = minus_infinity<T>();
                rec_z[j] = z;
                m_l = max_nan(m_l, z);
                if (label_in && v == y)
                {
                    label_logit = z;
                    label_listed = 1;
                }
            }
        }
        if (tid == 0 && label_in && tile.holds(y))
        {
            const int at = y - segment_first;
            if ((marked[at >> 5] >> (at & 31) & 1u) == 0)
            {
                label_logit = to_float(*tile.at(y));
                *tile.at(y) = minus_infinity<T>();
            }
        }
        __syncthreads();
        for (int j = tid; j < a.k; j += THREADS)
        {
            if (tile.holds(rec_col[j]))
            {
                marked[(rec_col[j] - segment_first) >> 5] = 0u;
            }
        }

        // maxima
        Vec16<T> best;
        {
            const T low = minus_infinity<T>();
            T *e = reinterpret_cast<T *>(&best);
#pragma unroll
            for (int i = 0; i < N; i++)
            {
                e[i] = low;
            }
        }
        for (int i = tid; i < tile.vecs; i += THREADS)
        {
            max_into(best, tile.vec(i));
        }
        const float m_warp = warp_max_nan(max_of(best));
        m_l = warp_max_nan(m_l);
        if (lane == 0)
        {
            warp_max[warp] = make_float2(m_warp, m_l);
        }
        __syncthreads();
        float m_u = -inf;
        m_l = -inf;
#pragma unroll
        for (int w = 0; w < WARPS; w++)
        {
            m_u = max_nan(m_u, warp_max[w].x);
            m_l = max_nan(m_l, warp_max[w].y);
        }

        // sums, relative to them
        {
            const float ref = m_u == -inf ? 0.0f : m_u;         // nothing but -inf: every term is 0
            const float2 minus_ref = make_float2(-ref, -ref), c_t2 = make_float2(c_t, c_t), c_12 = make_float2(c_1, c_1);
            float2 sum_t = make_float2(0.0f, 0.0f), sum_1 = make_float2(0.0f, 0.0f);
            for (int i = tid; i < tile.vecs; i += THREADS)
            {
                float2 f[PAIRS];
                unpack(tile.vec(i), f);
#pragma unroll
                for (int q = 0; q < PAIRS; q++)
                {
                    const float2 d = add2(f[q], minus_ref);
                    const float2 x = mul2(d, c_t2);
                    sum_t = add2(sum_t, make_float2(exp2_fast(x.x), exp2_fast(x.y)));
                    if (two)
                    {
                        const float2 x1 = mul2(d, c_12);
                        sum_1 = add2(sum_1, make_float2(exp2_fast(x1.x), exp2_fast(x1.y)));
                    }
                }
            }
            double l_t = 0.0, l_1 = 0.0, part = 0.0, own = 0.0;
            const double ref_l = m_l == -inf ? 0.0 : m_l;
            for (int j = tid; j < a.k; j += THREADS)
            {
                if (tile.holds(rec_col[j]))
                {
                    const double d = rec_z[j] - ref_l, p = rec_p[j];
                    l_t += exp(d * inv_t);
                    l_1 += two ? exp(d) : 0.0;
                    part += p != 0.0 ? p * (rec_lp[j] - d * inv_t) : 0.0;
                    own += p;
                }
            }
            const float s_t = warp_sum_f32(sum_t.x + sum_t.y), s_1 = warp_sum_f32(sum_1.x + sum_1.y);
            if (warp * 32 < a.k)                // the others have no listed columns
            {
                l_t = warp_sum_f64(l_t);
                l_1 = warp_sum_f64(l_1);
                part = warp_sum_f64(part);
                own = warp_sum_f64(own);
                mass = warp_sum_f64(mass);
            }
            if (lane == 0)
            {
                double *w = warp_sums[warp];
                w[0] = s_t;
                w[1] = s_1;
                w[2] = l_t;
                w[3] = l_1;
                w[4] = part;
                w[5] = own;
                w[6] = mass;
            }
        }
        __syncthreads();

        // the blocks of the cluster exchange theirs; the first warp of each works out the row's factors
        double others = 0.0, o_in_all = 0.0, total = 0.0, total_1 = 0.0, part = 0.0, rest = 0.0, whole = 0.0, d_y = 0.0;
        float m = 0.0f, m_o = 0.0f;
        if (warp == 0)
        {
            double sum = 0.0;
            if (lane < 7)
            {
                for (int w = 0; w < WARPS; w++)
                {
                    sum += warp_sums[w][lane];
                }
            }
            SegmentSums mine;
            mine.m_u = m_u;
            mine.m_l = m_l;
            mine.z_y = label_logit;
            mine.label_listed = label_listed;
            mine.s_t = __shfl_sync(0xffffffffu, sum, 0);
            mine.s_1 = __shfl_sync(0xffffffffu, sum, 1);
            mine.l_t = __shfl_sync(0xffffffffu, sum, 2);
            mine.l_1 = __shfl_sync(0xffffffffu, sum, 3);
            mine.part = __shfl_sync(0xffffffffu, sum, 4);
            mine.own = __shfl_sync(0xffffffffu, sum, 5);
            mass = __shfl_sync(0xffffffffu, sum, 6);
            if (blocks == 1)
            {
                slots[parity][0] = mine;        // every lane writes the same
            }
            else if (lane < blocks)
            {
                *cluster.map_shared_rank(&slots[parity][rank], lane) = mine;
            }
        }
        if (blocks > 1)
        {
            cluster.sync();
        }
        if (warp == 0)
        {
            __syncwarp();
            SegmentSums s = {-inf, -inf, -inf, 0, 0.0, 0.0, 0.0, 0.0, 0.0, 0.0};
            if (lane < blocks)
            {
                s = slots[parity][lane];
            }
            const float all_u = warp_max_nan(s.m_u), all_l = warp_max_nan(s.m_l), z_y = warp_max_nan(s.z_y);
            const bool listed = __any_sync(0xffffffffu, s.label_listed != 0);
            m_o = listed ? all_u : max_nan(all_u, z_y);         // of the columns not listed
            m = max_nan(m_o, all_l);
            const double u_t = warp_sum_f64(s.s_t * shifted(s.m_u, all_u, inv_t));
            const double u_1 = two ? warp_sum_f64(s.s_1 * shifted(s.m_u, all_u, 1.0)) : u_t;
            const double listed_t = warp_sum_f64(s.l_t * shifted(s.m_l, m, inv_t));
            const double listed_1 = two ? warp_sum_f64(s.l_1 * shifted(s.m_l, m, 1.0)) : listed_t;
            const double ref_l = s.m_l == -inf ? 0.0 : s.m_l;
            part = warp_sum_f64(s.part + (s.own != 0.0 ? s.own * (m - ref_l) * inv_t : 0.0));
            const double u_in_o = shifted(all_u, m_o, inv_t), y_in_o = listed ? 0.0 : shifted(z_y, m_o, inv_t);
            others = u_t * u_in_o + y_in_o;
            o_in_all = shifted(m_o, m, inv_t);
            total = others * o_in_all + listed_t;
            const double u_in_all_1 = two ? shifted(all_u, m, 1.0) : u_in_o * o_in_all;
            const double y_in_all_1 = two ? shifted(z_y, m, 1.0) : shifted(z_y, m, inv_t);
            total_1 = u_1 * u_in_all_1 + listed_1 + (listed ? 0.0 : y_in_all_1);
            rest = a.lse != nullptr && others > 0.0 ? fmax(0.0, 1.0 - mass) : 0.0;
            whole = mass + rest;
            d_y = static_cast<double>(z_y) - static_cast<double>(m);
            const double poison = !isfinite(m) || (hard && !label_in) ? nan("") : 0.0;
            part += poison;
            const double per_o = whole * o_in_all / total - (rest > 0.0 ? rest / others : 0.0);     // of e^(x - m_o)
            if (lane == 0)
            {
                const double f_t = soft_scale * per_o * u_in_o + poison;
                const double f_1 = hard ? hard_scale * u_in_all_1 / total_1 : 0.0;
                factors.m_u = all_u == -inf ? 0.0f : all_u;
                factors.f_t = static_cast<float>(two ? f_t : f_t + f_1);
                factors.f_1 = static_cast<float>(f_1);
                factors.m = m;
                factors.l_t = soft_scale * whole / total + poison + (two || !hard ? 0.0 : hard_scale / total_1);
                factors.l_1 = two ? hard_scale / total_1 : 0.0;
                factors.y = hard_scale;
                factors.label = soft_scale * per_o * y_in_o + hard_scale * (y_in_all_1 - total_1) / total_1 + poison;
            }
        }
        parity ^= 1;
        __syncthreads();

        // gradient
        if (out != nullptr && tile.vecs > 0)
        {
            const float ref = factors.m_u, f_t = factors.f_t, f_1 = factors.f_1;
            const float2 minus_ref = make_float2(-ref, -ref), c_t2 = make_float2(c_t, c_t), c_12 = make_float2(c_1, c_1);
            const float2 f_t2 = make_float2(f_t, f_t), f_12 = make_float2(f_1, f_1);
            char *dst = reinterpret_cast<char *>(out + segment_first) - tile.lead * sizeof(T);
            const bool same = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;                 // the row starts as far from a boundary as the logits'
            const int whole_first = tile.lead > 0 ? 1 : 0, whole_end = (tile.lead + tile.held) / N;
            for (int i = tid; i < tile.vecs; i += THREADS)
            {
                float2 f[PAIRS];
                unpack(tile.vec(i), f);
#pragma unroll
                for (int q = 0; q < PAIRS; q++)
                {
                    const float2 d = add2(f[q], minus_ref);
                    const float2 x = mul2(d, c_t2);
                    f[q] = mul2(make_float2(exp2_fast(x.x), exp2_fast(x.y)), f_t2);
                    if (two)
                    {
                        const float2 x1 = mul2(d, c_12);
                        f[q] = fma2(make_float2(exp2_fast(x1.x), exp2_fast(x1.y)), f_12, f[q]);
                    }
                }
                Vec16<T> g;
                pack(g, f);
                if (same && i >= whole_first && i < whole_end)
                {
                    *reinterpret_cast<uint4 *>(dst + 16ll * i) = g.w;
                }
                else if (same)
                {
                    const T *e = reinterpret_cast<const T *>(&g);
#pragma unroll
                    for (int q = 0; q < N; q++)
                    {
                        if (i * N + q >= tile.lead && i * N + q < tile.lead + tile.held)
                        {
                            reinterpret_cast<T *>(dst)[i * N + q] = e[q];
                        }
                    }
                }
                else
                {
                    reinterpret_cast<Vec16<T> *>(tile.buf)[i] = g;
                }
            }
            if (!same)
            {
                __syncthreads();
                for (int i = tid; i < tile.held; i += THREADS)
                {
                    out[segment_first + i] = reinterpret_cast<const T *>(tile.buf)[tile.lead + i];
                }
            }
        }
        __syncthreads();

        // the next row is on its way while the listed columns and the loss are written
        const Tile now = tile;
        started = row + clusters < a.rows && label_of(row + clusters) >= 0;
        if (started)
        {
            tile.start(row_of(row + clusters), segment_first, plan.segment, a.vocab, a.cols);
        }
        for (int j = tid; out != nullptr && j < a.k; j += THREADS)
        {
            const int v = rec_col[j];
            if (now.holds(v))
            {
                const double d = static_cast<double>(rec_z[j]) - static_cast<double>(factors.m);
                double g = exp(d * inv_t) * factors.l_t - soft_scale * rec_p[j];
                if (two)
                {
                    g += exp(d) * factors.l_1;
                }
                out[v] = from_float<T>(static_cast<float>(label_in && v == y ? g - factors.y : g));
            }
        }
        if (out != nullptr && tid == 0 && label_in && now.holds(y) && label_listed == 0)
        {
            out[y] = from_float<T>(static_cast<float>(factors.label));
        }
        if (rank == 0 && tid == 0)
        {
            double loss = part;                 // carries the poison of a row that has gone wrong
            if (a.k > 0)
            {
                const double log_o = rest > 0.0 ? log(others) + (static_cast<double>(m_o) - m) * inv_t : 0.0;
                loss += whole * log(total) + (rest > 0.0 ? rest * (log(rest) - log_o) : 0.0);
                loss *= a.soft;
            }
            if (hard)
            {
                loss += a.hard * (log(total_1) - d_y);
            }
            a.row_loss[row] = static_cast<float>(loss);
        }
        __syncthreads();                        // the record's arrays and the label are written again
    }

    if (!take_last_ticket(&a.ws->distill_ticket, gridDim.x, &last_block))
    {
        return;
    }
    double mine = 0.0;
    for (long long i = tid; i < a.rows; i += THREADS)
    {
        mine += static_cast<double>(__ldcg(&a.row_loss[i]));
    }
    mine = block_sum_f64<THREADS>(mine, scratch);
    if (tid == 0)
    {
        a.st->loss = static_cast<float>(mine / static_cast<double>(n_valid > 0 ? n_valid : 1));
        a.st->n_valid = static_cast<int>(n_valid);
    }
}

template <typename T, int THREADS>
static int launch_distill(const DistillArgs &a, RowPlan plan, cudaStream_t stream)
{
    return launch_rows(distill_rows_kernel<T, THREADS>, a, plan, a.rows, stream);
}

template <typename T>
static int launch_distill(const DistillArgs &a, cudaStream_t stream)
{
    const int record = a.k * (2 * sizeof(double) + sizeof(float) + sizeof(int));
    RowPlan plan;
    const int rc = plan_rows(a.rows, a.cols, sizeof(T), record, &plan);
    if (rc != B200AMP_OK)
    {
        return rc;
    }
    return plan.threads == 128 ? launch_distill<T, 128>(a, plan, stream) : launch_distill<T, 256>(a, plan, stream);
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
    DistillArgs a = {logits, dlogits, ld, dld, rows, vocab, cols, targets, values, indices, lse, value_dtype, k,
                     temperature, soft_weight, hard_weight, st, row_loss, static_cast<LossWorkspace *>(workspace)};
    switch (dtype)
    {
    case B200AMP_F16:
        return launch_distill<__half>(a, as_stream(s));
    case B200AMP_BF16:
        return launch_distill<__nv_bfloat16>(a, as_stream(s));
    default:
        return launch_distill<float>(a, as_stream(s));
    }
}
