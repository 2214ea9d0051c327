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
    long long starved;      // row whose copy a test keeps from completing, -1: none
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

// What the parts of a row tell each other, an array a quantity: n_warps places for the sweeping warps of the cluster,
// `blocks` for its blocks. Every block of a cluster holds all of them.
struct RowSums
{
    double *l_t, *l_1;      // sums over the listed columns, at the temperature and at 1, relative to m_l
    double *part, *own;     // sum w (log w - (z - m_l) / T) and sum w over them; w: the teacher's masses before the norm
    float *m_l, *z_y;       // maximum of the listed ones; the label's logit, -inf where it is in another segment
    float *m_u, *s_t, *s_1; // a warp's maximum and sums of the columns neither listed nor the label

    __device__ __forceinline__ RowSums(char *base, int blocks, int n_warps)
    {
        l_t = reinterpret_cast<double *>(base);
        l_1 = l_t + blocks;
        part = l_1 + blocks;
        own = part + blocks;
        m_l = reinterpret_cast<float *>(own + blocks);
        z_y = m_l + blocks;
        m_u = z_y + blocks;
        s_t = m_u + n_warps;
        s_1 = s_t + n_warps;
    }
};
__host__ __device__ inline int row_sums_bytes(int blocks, int n_warps)
{
    return blocks * static_cast<int>(4 * sizeof(double) + 2 * sizeof(float)) + n_warps * static_cast<int>(3 * sizeof(float));
}

// fp64 functions as calls: inlined a dozen times, code that a single warp runs through once a row is fetched more
// slowly than it is executed.
__device__ __noinline__ double exp64(double x)
{
    return exp(x);
}

// e^((from - to) f), 0 from -inf
__device__ __forceinline__ double shifted(float from, float to, double f)
{
    return from == -INFINITY ? 0.0 : exp64((static_cast<double>(from) - static_cast<double>(to)) * f);
}
__device__ __forceinline__ float shifted_fast(float from, float to, float c)
{
    return from == -INFINITY ? 0.0f : exp2_fast((from - to) * c);
}

// Maximum over the warp with NaN winning, in one instruction.
__device__ __forceinline__ float warp_max_once(float v)
{
    float m;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
    return m;
}

// a / b: to the nearest for fp32 gradients, to 2 ulp for 16-bit ones, whose own rounding is a thousand times that
template <typename T>
__device__ __forceinline__ float quotient(float a, float b)
{
    return sizeof(T) == 4 ? a / b : __fdividef(a, b);
}

// Sum over the first n lanes (a power of two), in every lane.
template <typename V>
__device__ __forceinline__ V sum_lanes(V v, int n)
{
    for (int offset = n >> 1; offset > 0; offset >>= 1)
    {
        v += __shfl_xor_sync(0xffffffffu, v, offset);
    }
    return __shfl_sync(0xffffffffu, v, 0);
}

// The sweeps of the segment. TWO: two softmaxes of a row, at the temperature and at 1. They take several vectors at a
// time: one alone leaves a warp waiting for its own loads, powers and additions.
template <typename T, int THREADS>
__device__ __forceinline__ float sweep_max(const RowTile<T, THREADS> &tile)
{
    constexpr int AT_ONCE = 4;
    Vec16<T> best;
    const T low = minus_infinity<T>();
    T *e = reinterpret_cast<T *>(&best);
#pragma unroll
    for (int i = 0; i < Vec16<T>::N; i++)
    {
        e[i] = low;
    }
    int i = threadIdx.x;
    for (; i + (AT_ONCE - 1) * THREADS < tile.vecs; i += AT_ONCE * THREADS)
    {
        Vec16<T> v[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
        {
            v[u] = tile.vec(i + u * THREADS);
        }
        max_into(v[0], v[1]);
        max_into(v[2], v[3]);
        max_into(best, v[0]);
        max_into(best, v[2]);
    }
    for (; i < tile.vecs; i += THREADS)
    {
        max_into(best, tile.vec(i));
    }
    return warp_max_once(max_of(best));
}

template <bool TWO, typename T, int THREADS>
__device__ __forceinline__ void sweep_sums(const RowTile<T, THREADS> &tile, float ref, float c_t, float c_1, float *s_t, float *s_1)
{
    constexpr int PAIRS = Vec16<T>::N / 2, AT_ONCE = TWO || sizeof(T) == 2 ? 2 : 4;
    const float2 minus_ref = make_float2(-ref, -ref), c_t2 = make_float2(c_t, c_t), c_12 = make_float2(c_1, c_1);
    float2 sum_t[AT_ONCE], sum_1[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; u++)
    {
        sum_t[u] = make_float2(0.0f, 0.0f);
        sum_1[u] = make_float2(0.0f, 0.0f);
    }
    auto add = [&](const float2 (&f)[PAIRS], int u) {
#pragma unroll
        for (int q = 0; q < PAIRS; q++)
        {
            const float2 d = add2(f[q], minus_ref);
            const float2 x = mul2(d, c_t2);
            sum_t[u] = add2(sum_t[u], make_float2(exp2_fast(x.x), exp2_fast(x.y)));
            if (TWO)
            {
                const float2 x1 = mul2(d, c_12);
                sum_1[u] = add2(sum_1[u], make_float2(exp2_fast(x1.x), exp2_fast(x1.y)));
            }
        }
    };
    int i = threadIdx.x;
    for (; i + (AT_ONCE - 1) * THREADS < tile.vecs; i += AT_ONCE * THREADS)
    {
        float2 f[AT_ONCE][PAIRS];
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
        {
            unpack(tile.vec(i + u * THREADS), f[u]);
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; u++)
        {
            add(f[u], u);
        }
    }
    for (; i < tile.vecs; i += THREADS)
    {
        float2 f[PAIRS];
        unpack(tile.vec(i), f);
        add(f, 0);
    }
#pragma unroll
    for (int u = 1; u < AT_ONCE; u++)
    {
        sum_t[0] = add2(sum_t[0], sum_t[u]);
        sum_1[0] = add2(sum_1[0], sum_1[u]);
    }
    *s_t = warp_sum_f32(sum_t[0].x + sum_t[0].y);
    *s_1 = TWO ? warp_sum_f32(sum_1[0].x + sum_1[0].y) : *s_t;
}

template <bool TWO, typename T>
__device__ __forceinline__ Vec16<T> gradient_of(const Vec16<T> &z, float ref, float c_t, float c_1, float f_t, float f_1)
{
    constexpr int PAIRS = Vec16<T>::N / 2;
    const float2 minus_ref = make_float2(-ref, -ref), c_t2 = make_float2(c_t, c_t), c_12 = make_float2(c_1, c_1);
    const float2 f_t2 = make_float2(f_t, f_t), f_12 = make_float2(f_1, f_1);
    float2 f[PAIRS];
    unpack(z, f);
#pragma unroll
    for (int q = 0; q < PAIRS; q++)
    {
        const float2 d = add2(f[q], minus_ref);
        const float2 x = mul2(d, c_t2);
        f[q] = mul2(make_float2(exp2_fast(x.x), exp2_fast(x.y)), f_t2);
        if (TWO)
        {
            const float2 x1 = mul2(d, c_12);
            f[q] = fma2(make_float2(exp2_fast(x1.x), exp2_fast(x1.y)), f_12, f[q]);
        }
    }
    Vec16<T> g;
    pack(g, f);
    return g;
}

// Named barriers: 1 among the sweeping threads, 2 for the block where its two parts come from different code.
template <int THREADS>
__device__ __forceinline__ void sweep_barrier()
{
    asm volatile("bar.sync 1, %0;" : : "n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ void both_barrier()
{
    asm volatile("bar.sync 2, %0;" : : "n"(THREADS) : "memory");
}

// The gradient of the segment's columns; the listed ones and the label's are written over afterwards.
template <bool TWO, typename T, int THREADS>
__device__ __forceinline__ void sweep_gradient(const RowTile<T, THREADS> &tile, T *out, float ref, float c_t, float c_1, float f_t,
                                               float f_1)
{
    constexpr int N = Vec16<T>::N;
    const int tid = threadIdx.x;
    char *dst = reinterpret_cast<char *>(out + tile.first) - tile.lead * sizeof(T);
    if ((reinterpret_cast<uintptr_t>(dst) & 15) == 0)
    {
        // the row starts as far from a 16-byte boundary as the logits' row: whole vectors, then the two ends
        const int whole_first = tile.lead > 0 ? 1 : 0, whole_end = (tile.lead + tile.held) / N;
        int k = whole_first + tid;
        for (; k + THREADS < whole_end; k += 2 * THREADS)
        {
            const Vec16<T> z0 = tile.vec(k), z1 = tile.vec(k + THREADS);
            const Vec16<T> g0 = gradient_of<TWO>(z0, ref, c_t, c_1, f_t, f_1), g1 = gradient_of<TWO>(z1, ref, c_t, c_1, f_t, f_1);
            *reinterpret_cast<uint4 *>(dst + 16ll * k) = g0.w;
            *reinterpret_cast<uint4 *>(dst + 16ll * (k + THREADS)) = g1.w;
        }
        if (k < whole_end)
        {
            *reinterpret_cast<uint4 *>(dst + 16ll * k) = gradient_of<TWO>(tile.vec(k), ref, c_t, c_1, f_t, f_1).w;
        }
        const bool front = tid == 0 && tile.lead > 0;
        const bool back = tid == 1 && whole_end < tile.vecs && whole_end >= whole_first;
        if (front || back)
        {
            const int i = front ? 0 : whole_end;
            const Vec16<T> g = gradient_of<TWO>(tile.vec(i), ref, c_t, c_1, f_t, f_1);
            const T *e = reinterpret_cast<const T *>(&g);
            for (int q = 0; q < N; q++)
            {
                if (i * N + q >= tile.lead && i * N + q < tile.lead + tile.held)
                {
                    reinterpret_cast<T *>(dst)[i * N + q] = e[q];
                }
            }
        }
        return;
    }
    for (int i = tid; i < tile.vecs; i += THREADS)
    {
        reinterpret_cast<Vec16<T> *>(tile.buf)[i] = gradient_of<TWO>(tile.vec(i), ref, c_t, c_1, f_t, f_1);
    }
    before_copies();
    sweep_barrier<THREADS>();
    for (int i = tid; i < tile.held; i += THREADS)
    {
        out[tile.first + i] = reinterpret_cast<const T *>(tile.buf)[tile.lead + i];
    }
}

// Zeros from `from` to `to`, by a warp. A call, for rows that hardly occur.
template <typename T>
__device__ __noinline__ void zero_columns(T *out, int from, int to)
{
    for (int i = from + (threadIdx.x & 31); i < to; i += 32)
    {
        out[i] = from_float<T>(0.0f);
    }
}

// A cluster a row, the row in its shared memory between the sweeps. A block has SWEEP threads that sweep the segment
// and one more warp for what there is one of a row: the listed columns' sums, the factors, the loss. That warp works
// while the others sweep, so its fp64 chains are off the row's path, and they are issued once a block and not once a
// warp (done by every warp they were two thirds of all instructions). The sweeping threads read the record while the
// row is on its way. Barriers of a block and row:
//     arrived   the row is in shared memory, the record has been read
//     marked    the listed columns and the label have been taken out of the row
//     summed    (the cluster's) every warp's sums are with every block
//     factors   the row's factors are known
//     written   the gradient is out; the row's place may be filled again
// 8192 rows of 50257 fp16 columns (k 64, rest and label) take 350 us, 1.6 GB, 4.6 TB/s; the powers alone would take 181 us
// of the special function unit, the bytes 246 us. A block's rows are behind one another, so what bounds it is a row's
// chain: at two blocks an SM about 20,000 cycles, 6,500 for the sums, 5,500 for the gradient, the rest barriers, the
// record and the factors. Registers for two blocks of 256 threads an SM (96 a thread, no spills): with fewer, spills go past
// the little L1 that the rows leave (422 us). Eight blocks of 64 have 80 a thread and spill 28 to 36 bytes.
template <typename T, int SWEEP>
__global__ void __launch_bounds__(SWEEP + 32, 512 / SWEEP) distill_rows_kernel(const DistillArgs a, const RowPlan plan)
{
    namespace cg = cooperative_groups;
    using Tile = RowTile<T, SWEEP>;
    constexpr int THREADS = SWEEP + 32, WARPS = SWEEP / 32;     // WARPS: those that sweep
    // fp32 gradients: the listed columns' and the label's, most of a gradient's magnitude, are worked out in fp64, as their
    // terms cancel where student and teacher agree; a 16-bit one hides the difference (2^-12 against 2^-22).
    constexpr bool WIDE = sizeof(T) == 4;
    extern __shared__ __align__(16) char dynamic[];
    __shared__ double scratch[THREADS / 32];
    __shared__ float shared_ref, shared_f_t, shared_f_1, t_max_of[WARPS];
    __shared__ double shared_scale[2];          // loss scale over rows that count, times the weights (soft: over T too)
    __shared__ double wide[4];                  // l_t and l_1 in fp64, what a mass is multiplied by, the label's gradient
    __shared__ int label_listed[2], beyond_listed[2];
    __shared__ uint64_t row_bar;
    __shared__ int last_block;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool sweeps = warp < WARPS;
    const cg::cluster_group cluster = cg::this_cluster();
    const int blocks = plan.cluster, rank = blocks > 1 ? static_cast<int>(cluster.block_rank()) : 0;
    const int n_warps = blocks * WARPS;
    const float inf = INFINITY;

    // dynamic shared memory: the segment; two rows' sums; two rows' records (mass, its logarithm, logit, column, -1 where
    // that is not of this segment); a bit a column, which finds those listed twice
    const size_t tile_bytes = (static_cast<size_t>(plan.segment) * sizeof(T) + 31) & ~static_cast<size_t>(15);
    const int sums_bytes = (row_sums_bytes(blocks, n_warps) + 7) & ~7;
    Tile tile;
    tile.buf = dynamic;
    tile.uneven = (a.ld * static_cast<long long>(sizeof(T)) & 15) != 0;
    char *const sums = dynamic + tile_bytes;
    double *const rec_w0 = reinterpret_cast<double *>(sums + 2 * sums_bytes);
    double *const rec_lw0 = rec_w0 + 2 * a.k;
    float *const rec_z0 = reinterpret_cast<float *>(rec_lw0 + 2 * a.k);
    int *const rec_col0 = reinterpret_cast<int *>(rec_z0 + 2 * a.k);
    int *const mine = rec_col0 + 2 * a.k;       // places of the listed columns of this segment, in the record's order
    unsigned int *const listed_bits = reinterpret_cast<unsigned int *>(mine + a.k);

    const bool hard = a.hard != 0.0;
    const double inv_t = a.k > 0 ? 1.0 / a.temperature : 1.0;       // the label's softmax alone is at 1
    const bool two = hard && a.k > 0 && a.temperature != 1.0;       // two softmaxes of a row
    const double log2e = 1.4426950408889634;
    const float c_t = static_cast<float>(log2e * inv_t), c_1 = static_cast<float>(log2e);
    const int first = rank * plan.segment;
    const int valid = max(0, min(plan.segment, a.vocab - first)), held = max(0, min(plan.segment, a.cols - first));
    const long long clusters = gridDim.x / blocks;
    auto label_of = [&](long long row) { return row < 0 || row >= a.rows ? -1 : a.targets != nullptr ? __ldg(&a.targets[row]) : 0; };

    // what a sweeping thread fetches of the next row's record while the gradient is swept
    int ahead_v = -1;
    float ahead_t = 0.0f, ahead_lse = 0.0f;
    auto fetch = [&](long long at) {
        if (tid < a.k)
        {
            ahead_v = __ldg(&a.indices[at * a.k + tid]);
            ahead_t = load_typed(a.values, a.value_dtype, at * a.k + tid);
        }
        if (a.lse != nullptr)
        {
            ahead_lse = __ldg(&a.lse[at]);
        }
    };
    // The record of a row into rec[parity], by the sweeping threads. Masses are w = e^(t / T - lse), or, before the norm
    // that the cluster works out, e^((t - max) / T). True where this thread met a column that was listed already.
    auto read_record = [&](long long at, int label, int parity) {
        double *w_of = rec_w0 + parity * a.k, *lw_of = rec_lw0 + parity * a.k;
        int *col_of = rec_col0 + parity * a.k;
        double shift = ahead_lse;
        if (a.lse == nullptr)
        {
            float t_max = tid < a.k && ahead_v >= 0 ? ahead_t : -inf;
            for (int j = tid + SWEEP; j < a.k; j += SWEEP)
            {
                const float t = load_typed(a.values, a.value_dtype, at * a.k + j);
                t_max = max_nan(t_max, __ldg(&a.indices[at * a.k + j]) >= 0 ? t : -inf);
            }
            t_max = warp_max_once(t_max);
            if (lane == 0)
            {
                t_max_of[warp] = t_max;
            }
            sweep_barrier<SWEEP>();
            t_max = warp_max_once(t_max_of[lane & (WARPS - 1)]);
            shift = t_max == -inf ? 0.0 : t_max * inv_t;
        }
        bool twice = false;
        for (int j = tid; j < a.k; j += SWEEP)
        {
            const int v = j < SWEEP ? ahead_v : __ldg(&a.indices[at * a.k + j]);
            const float t = j < SWEEP ? ahead_t : load_typed(a.values, a.value_dtype, at * a.k + j);
            const bool of_segment = v >= first && v < first + valid;
            col_of[j] = of_segment ? v : -1;
            if (v >= a.vocab)
            {
                beyond_listed[parity] = 1;
            }
            if (hard && v == label)
            {
                label_listed[parity] = 1;
            }
            if (of_segment)
            {
                const double lw = t * inv_t - shift;
                lw_of[j] = lw;
                w_of[j] = exp64(lw);
                const unsigned int bit = 1u << ((v - first) & 31);
                twice = twice || (atomicOr(&listed_bits[(v - first) >> 5], bit) & bit) != 0;
            }
        }
        return twice;
    };

    for (int i = tid; i < plan.segment / 32; i += THREADS)
    {
        listed_bits[i] = 0u;
    }
    if (tid < 2)
    {
        label_listed[tid] = 0;
        beyond_listed[tid] = 0;
    }
    if (tid == 0)
    {
        row_barrier_init(&row_bar);
    }
    __syncthreads();
    if (blocks > 1)
    {
        cluster.sync();                         // every block of the cluster runs before one writes to another
    }

    // The first trip has no row yet (row < 0): it starts the first copy and reads the first record. The rows that count
    // take the two places of the sums and of the records in turn: between two uses of a place there is then always one
    // row whose barriers all readers of the first use have reached (a row that does not count has no barrier).
    bool twice = false;
    unsigned int phase = 0u;                    // of row_bar, with what RowTile::wait adds
    float soft_scale = 0.0f, hard_scale = 0.0f;
    long long n_valid = 0;
    int y = -1, parity = 0;
    for (long long row = blockIdx.x / blocks - clusters; row < a.rows; row += clusters)
    {
        T *out = a.dlogits != nullptr && row >= 0 ? static_cast<T *>(a.dlogits) + row * a.dld : nullptr;
        const int next_y = label_of(row + clusters);
        const bool label_in = hard && y >= 0 && y < a.vocab;
        bool listed_y = false;
        int n_listed = 0;
        char *const place = sums + parity * sums_bytes;
        double *const rec_w = rec_w0 + parity * a.k, *const rec_lw = rec_lw0 + parity * a.k;
        float *const rec_z = rec_z0 + parity * a.k;
        int *const rec_col = rec_col0 + parity * a.k;
        float m = 0.0f, per_o = 0.0f, y_in_o = 0.0f, not_y_1 = 0.0f, total_1 = 1.0f, norm = 1.0f, poison = 0.0f;
        float l_t = 0.0f, l_1 = 0.0f;           // the last warp's, for what it writes at the end
        if (y >= 0)
        {
            if (sweeps)
            {
                tile.wait(&row_bar, phase);
            }
            if (__syncthreads_or(twice))        // arrived
            {
                // a column listed more than once keeps its first place, with all its mass
                for (int j = tid; j < a.k; j += THREADS)
                {
                    bool is_first = rec_col[j] >= 0;
                    double w = 0.0;
                    for (int q = 0; rec_col[j] >= 0 && q < a.k; q++)
                    {
                        is_first = is_first && !(q < j && rec_col[q] == rec_col[j]);
                        w += rec_col[q] == rec_col[j] ? rec_w[q] : 0.0;
                    }
                    rec_z[j] = is_first ? 1.0f : 0.0f;
                    rec_lw[j] = log(w);
                }
                __syncthreads();
                for (int j = tid; j < a.k; j += THREADS)
                {
                    rec_w[j] = exp64(rec_lw[j]);
                    rec_col[j] = rec_z[j] != 0.0f ? rec_col[j] : -1;
                }
                __syncthreads();
            }
            listed_y = label_listed[parity] != 0;

            float z_y = -inf;
            if (sweeps)
            {
                for (int j = tid; j < a.k; j += SWEEP)
                {
                    const int v = rec_col[j];
                    if (v >= 0)
                    {
                        rec_z[j] = to_float(*tile.at(v));
                        *tile.at(v) = minus_infinity<T>();
                        before_copies();
                    }
                }
            }
            else
            {
                if (lane == 0 && label_in && !listed_y && y >= first && y < first + valid)
                {
                    // where the tile keeps column y
                    const uintptr_t src = reinterpret_cast<uintptr_t>(static_cast<const T *>(a.logits) + row * a.ld + first);
                    T *const e = reinterpret_cast<T *>(dynamic + (src & 15)) + (y - first);
                    z_y = to_float(*e);
                    *e = minus_infinity<T>();
                    before_copies();
                }
                for (int j0 = 0; j0 < a.k; j0 += 32)
                {
                    const bool has = j0 + lane < a.k && rec_col[j0 + lane] >= 0;
                    const unsigned int ballot = __ballot_sync(0xffffffffu, has);
                    if (has)
                    {
                        mine[n_listed + __popc(ballot & ((1u << lane) - 1u))] = j0 + lane;
                    }
                    n_listed += __popc(ballot);
                }
                __syncwarp();
                for (int i = lane; i < n_listed; i += 32)
                {
                    listed_bits[(rec_col[mine[i]] - first) >> 5] = 0u;
                }
            }
            __syncthreads();                    // marked

            if (sweeps)
            {
                // sums of this warp's share, relative to its own maximum
                const float m_u = sweep_max(tile);
                const float ref = m_u == -inf ? 0.0f : m_u;     // nothing but -inf: every term is 0
                float s_t, s_1;
                if (two)
                {
                    sweep_sums<true>(tile, ref, c_t, c_1, &s_t, &s_1);
                }
                else
                {
                    sweep_sums<false>(tile, ref, c_t, c_1, &s_t, &s_1);
                }
                if (lane < blocks)
                {
                    const RowSums to(blocks > 1 ? cluster.map_shared_rank(place, lane) : place, blocks, n_warps);
                    to.m_u[rank * WARPS + warp] = m_u;
                    to.s_t[rank * WARPS + warp] = s_t;
                    to.s_1[rank * WARPS + warp] = s_1;
                }
            }
            else
            {
                float m_l = -inf;
                for (int i = lane; i < n_listed; i += 32)
                {
                    const float z = rec_z[mine[i]];
                    m_l = max_nan(m_l, z);
                    z_y = hard && rec_col[mine[i]] == y ? z : z_y;
                }
                m_l = warp_max_once(m_l);
                z_y = warp_max_once(z_y);
                const double ref_l = m_l == -inf ? 0.0 : m_l;
                double lt = 0.0, l1 = 0.0, part = 0.0, own = 0.0;
                for (int i = lane; i < n_listed; i += 32)
                {
                    const double d = rec_z[mine[i]] - ref_l, w = rec_w[mine[i]];
                    lt += exp64(d * inv_t);
                    l1 += two ? exp64(d) : 0.0;
                    part += w != 0.0 ? w * (rec_lw[mine[i]] - d * inv_t) : 0.0;
                    own += w;
                }
                if (n_listed > 0)
                {
                    lt = warp_sum_f64(lt);
                    l1 = two ? warp_sum_f64(l1) : lt;
                    part = warp_sum_f64(part);
                    own = warp_sum_f64(own);
                }
                if (beyond_listed[parity] != 0)
                {
                    own = nan("");              // a column beyond the vocabulary: the row is NaN
                }
                if (lane < blocks)
                {
                    const RowSums to(blocks > 1 ? cluster.map_shared_rank(place, lane) : place, blocks, n_warps);
                    to.l_t[rank] = lt;
                    to.l_1[rank] = l1;
                    to.part[rank] = part;
                    to.own[rank] = own;
                    to.m_l[rank] = m_l;
                    to.z_y[rank] = z_y;
                }
            }
            if (blocks > 1)
            {
                cluster.sync();                 // summed
            }
            else
            {
                __syncthreads();
            }

            if (sweeps)
            {
                if (next_y >= 0)
                {
                    fetch(row + clusters);
                }
                both_barrier<THREADS>();        // factors
                if (out != nullptr && tile.vecs > 0)
                {
                    if (two)
                    {
                        sweep_gradient<true>(tile, out, shared_ref, c_t, c_1, shared_f_t, shared_f_1);
                    }
                    else
                    {
                        sweep_gradient<false>(tile, out, shared_ref, c_t, c_1, shared_f_t, shared_f_1);
                    }
                }
            }
            else
            {
                // the row's factors; fp32 does for the gradient
                const RowSums all(place, blocks, n_warps);
                const bool is_block = lane < blocks;
                const float block_l = is_block ? all.m_l[lane] : -inf;
                const double block_lt = is_block ? all.l_t[lane] : 0.0, block_l1 = is_block ? all.l_1[lane] : 0.0;
                const double block_own = is_block ? all.own[lane] : 0.0, block_part = is_block ? all.part[lane] : 0.0;
                float all_u = -inf;
                for (int i = lane; i < n_warps; i += 32)
                {
                    all_u = max_nan(all_u, all.m_u[i]);
                }
                all_u = warp_max_once(all_u);
                z_y = warp_max_once(is_block ? all.z_y[lane] : -inf);
                const float m_o = listed_y ? all_u : max_nan(all_u, z_y);       // of the columns not listed
                m = max_nan(m_o, warp_max_once(block_l));
                float u_t = 0.0f, u_1 = 0.0f;
                for (int i = lane; i < n_warps; i += 32)
                {
                    const float in_u = shifted_fast(all.m_u[i], all_u, c_t);
                    u_t = fmaf(all.s_t[i], in_u, u_t);
                    u_1 += two ? all.s_1[i] * shifted_fast(all.m_u[i], all_u, c_1) : 0.0f;
                }
                u_t = warp_sum_f32(u_t);
                u_1 = two ? warp_sum_f32(u_1) : u_t;
                const float listed_t = sum_lanes(static_cast<float>(block_lt) * shifted_fast(block_l, m, c_t), blocks);
                const float listed_1 =
                    two ? sum_lanes(static_cast<float>(block_l1) * shifted_fast(block_l, m, c_1), blocks) : listed_t;
                const double own = sum_lanes(block_own, blocks);
                // mass of the listed columns; what a w is multiplied by
                norm = a.lse != nullptr || own == 0.0 ? 1.0f : __fdividef(1.0f, static_cast<float>(own));
                const double mass = a.lse != nullptr || own == 0.0 || own != own ? own : 1.0;
                const float u_in_o = shifted_fast(all_u, m_o, c_t);
                y_in_o = listed_y ? 0.0f : shifted_fast(z_y, m_o, c_t);
                const float others = fmaf(u_t, u_in_o, y_in_o);
                const float o_in_all = shifted_fast(m_o, m, c_t);
                const float total = fmaf(others, o_in_all, listed_t);
                const double rest = a.lse != nullptr && a.k > 0 && others > 0.0f ? fmax(0.0, 1.0 - mass) : 0.0;
                poison = !isfinite(m) || (hard && !label_in) ? NAN : 0.0f;
                const float whole = static_cast<float>(mass + rest) + poison;
                const float u_in_all_1 = two ? shifted_fast(all_u, m, c_1) : u_in_o * o_in_all;
                not_y_1 = fmaf(u_1, u_in_all_1, listed_1);                      // all but the label, where that is not listed
                total_1 = not_y_1 + (listed_y ? 0.0f : shifted_fast(z_y, m, c_1));
                const float q_per = soft_scale * quotient<T>(whole, total);
                per_o = q_per * o_in_all - (rest > 0.0 ? soft_scale * quotient<T>(static_cast<float>(rest), others) : 0.0f);
                l_1 = hard ? quotient<T>(hard_scale, total_1) : 0.0f;
                l_t = q_per + (two ? 0.0f : l_1);
                const float f_1 = l_1 * u_in_all_1;
                if (lane == 0)
                {
                    beyond_listed[parity] = 0;
                    label_listed[parity] = 0;
                    shared_ref = all_u == -inf ? 0.0f : all_u;
                    shared_f_t = per_o * u_in_o + poison + (two ? 0.0f : f_1);
                    shared_f_1 = f_1;
                }
                both_barrier<THREADS>();        // factors

                // while the gradient is swept: the row in fp64, for the loss (in turn by the cluster's blocks) and for WIDE
                const bool turn = rank == static_cast<int>(row / clusters & (blocks - 1));
                if (WIDE || turn)
                {
                    double u_t64 = 0.0, u_164 = 0.0;
                    for (int i = lane; i < n_warps; i += 32)
                    {
                        u_t64 += all.s_t[i] * shifted(all.m_u[i], all_u, inv_t);
                        u_164 += two ? all.s_1[i] * shifted(all.m_u[i], all_u, 1.0) : 0.0;
                    }
                    u_t64 = warp_sum_f64(u_t64);
                    u_164 = two ? warp_sum_f64(u_164) : u_t64;
                    // the other powers, one a lane: the blocks' listed sums, then what is not listed
                    const float from = is_block ? block_l : lane == 16 || lane == 19 ? all_u : lane == 18 ? m_o : z_y;
                    const float to = lane == 16 || lane == 17 ? m_o : m;
                    const double e = shifted(from, to, lane < 19 ? inv_t : 1.0);
                    const double listed_t64 = sum_lanes(block_lt * e, blocks);
                    const double listed_164 =
                        two ? sum_lanes(is_block ? block_l1 * shifted(block_l, m, 1.0) : 0.0, blocks) : listed_t64;
                    const double ref_l = block_l == -inf ? 0.0 : block_l;
                    const double part =
                        sum_lanes(block_part + (block_own != 0.0 ? block_own * (m - ref_l) * inv_t : 0.0), blocks);
                    const double u_in_o64 = __shfl_sync(0xffffffffu, e, 16), y_in_o64 = __shfl_sync(0xffffffffu, e, 17);
                    const double o_in_all64 = __shfl_sync(0xffffffffu, e, 18), u_in_all64 = __shfl_sync(0xffffffffu, e, 19);
                    const double y_in_all64 = __shfl_sync(0xffffffffu, e, 20);
                    const double o = u_t64 * u_in_o64 + (listed_y ? 0.0 : y_in_o64);
                    const double s = o * o_in_all64 + listed_t64;
                    const double not_y = u_164 * (two ? u_in_all64 : u_in_o64 * o_in_all64) + listed_164;
                    const double s_1 = not_y + (listed_y ? 0.0 : y_in_all64);
                    if (WIDE)
                    {
                        const double soft64 = shared_scale[0], hard64 = shared_scale[1], q = soft64 * (mass + rest) / s;
                        const double by_label = hard64 / s_1;
                        if (lane == 0)
                        {
                            wide[0] = q + (two ? 0.0 : by_label);
                            wide[1] = by_label;
                            wide[2] = a.lse != nullptr || own == 0.0 ? soft64 : soft64 / own;
                            wide[3] = (q * o_in_all64 - (rest > 0.0 ? soft64 * rest / o : 0.0)) * y_in_o64 - by_label * not_y;
                        }
                    }
                    // one logarithm a lane
                    const double of = lane == 0 ? s : lane == 1 ? s_1 : lane == 2 ? o : lane == 3 ? rest : own;
                    const double log_of = of > 0.0 ? log(of) : 0.0;
                    const double log_s = __shfl_sync(0xffffffffu, log_of, 0), log_s1 = __shfl_sync(0xffffffffu, log_of, 1);
                    const double log_o = __shfl_sync(0xffffffffu, log_of, 2), log_rest = __shfl_sync(0xffffffffu, log_of, 3);
                    const double log_own = __shfl_sync(0xffffffffu, log_of, 4);
                    if (lane == 0 && turn)
                    {
                        double loss = 0.0;
                        if (a.k > 0)
                        {
                            loss = a.lse != nullptr ? part : own == 0.0 ? 0.0 : part / own - log_own;
                            loss += (mass + rest) * log_s;
                            loss += rest > 0.0 ? rest * (log_rest - log_o - (static_cast<double>(m_o) - m) * inv_t) : 0.0;
                            loss *= a.soft;
                        }
                        if (hard)
                        {
                            loss += a.hard * (log_s1 - (static_cast<double>(z_y) - m));
                        }
                        a.row_loss[row] = static_cast<float>(loss + poison);
                    }
                }
            }
        }
        else if (row >= 0)
        {
            for (int i = tid; out != nullptr && i < held; i += THREADS)
            {
                out[first + i] = from_float<T>(0.0f);
            }
            if (rank == 0 && tid == 0)
            {
                a.row_loss[row] = 0.0f;
            }
        }

        if (y >= 0)
        {
            both_barrier<THREADS>();            // written
        }
        twice = false;
        if (sweeps && next_y >= 0)
        {
            tile.start(static_cast<const T *>(a.logits) + (row + clusters) * a.ld, first, plan.segment, a.vocab, a.cols,
                       &row_bar, phase, row + clusters == a.starved && rank == blocks - 1);
            if (a.k > 0)
            {
                if (y < 0)
                {
                    fetch(row + clusters);
                }
                twice = read_record(row + clusters, next_y, parity ^ 1);
            }
        }
        if (row < 0)
        {
            n_valid = count_rows<THREADS>(a.targets, a.rows, scratch);
            const double scale = static_cast<double>(a.st->loss_scale) / static_cast<double>(n_valid > 0 ? n_valid : 1);
            soft_scale = a.k > 0 ? static_cast<float>(scale * a.soft * inv_t) : 0.0f;
            hard_scale = hard ? static_cast<float>(scale * a.hard) : 0.0f;
            if (WIDE && tid == SWEEP)           // of the warp that reads it
            {
                shared_scale[0] = a.k > 0 ? scale * a.soft * inv_t : 0.0;
                shared_scale[1] = hard ? scale * a.hard : 0.0;
            }
        }
        if (!sweeps && y >= 0 && out != nullptr)
        {
            // while the next row is on its way: what the sweep left to this warp
            const float p_scale = soft_scale * norm;
            for (int i = lane; i < n_listed; i += 32)
            {
                const int j = mine[i], v = rec_col[j];
                if (WIDE)
                {
                    double g64 = shifted(rec_z[j], m, inv_t) * wide[0] - wide[2] * rec_w[j];
                    g64 += two ? shifted(rec_z[j], m, 1.0) * wide[1] : 0.0;
                    out[v] = from_float<T>(static_cast<float>(hard && v == y ? g64 - shared_scale[1] : g64) + poison);
                    continue;
                }
                float g = fmaf(shifted_fast(rec_z[j], m, c_t), l_t, -p_scale * static_cast<float>(rec_w[j])) + poison;
                if (two)
                {
                    g = fmaf(shifted_fast(rec_z[j], m, c_1), l_1, g);
                }
                out[v] = from_float<T>(hard && v == y ? g - hard_scale : g);
            }
            if (a.cols > a.vocab && !(isfinite(shared_f_t + shared_f_1)))
            {
                // the padding, where 0 times the factor is NaN
                zero_columns(out, max(first, a.vocab), min(first + plan.segment, a.cols));
            }
            if (lane == 0 && label_in && !listed_y && y >= first && y < first + valid)
            {
                out[y] = from_float<T>((WIDE ? static_cast<float>(wide[3])
                                             : per_o * y_in_o - hard_scale * __fdividef(not_y_1, total_1)) + poison);
            }
        }
        y = next_y;
        parity ^= next_y >= 0 ? 1 : 0;
    }
    if (tid == 0)
    {
        row_leave(&row_bar, phase);
    }

    if (!take_last_ticket(&a.ws->distill_ticket, gridDim.x, &last_block))
    {
        return;
    }
    double loss_sum = 0.0;
    for (long long i = tid; i < a.rows; i += THREADS)
    {
        loss_sum += static_cast<double>(__ldcg(&a.row_loss[i]));
    }
    loss_sum = block_sum_f64<THREADS>(loss_sum, scratch);
    if (tid == 0)
    {
        a.st->loss = static_cast<float>(loss_sum / static_cast<double>(n_valid > 0 ? n_valid : 1));
        a.st->n_valid = static_cast<int>(n_valid);
    }
}

template <typename T, int SWEEP>
static int launch_distill(const DistillArgs &a, RowPlan plan, cudaStream_t stream)
{
    return launch_rows(distill_rows_kernel<T, SWEEP>, a, plan, SWEEP + 32, a.rows, stream);
}

template <typename T>
static int launch_distill(const DistillArgs &a, cudaStream_t stream)
{
    const int record = a.k * (2 * (2 * sizeof(double) + sizeof(float) + sizeof(int)) + sizeof(int));
    RowPlan plan;
    const int rc = plan_rows(
        a.rows, a.cols, sizeof(T), 64, 256,
        [&](const RowPlan &p) {
            return record + 2 * ((row_sums_bytes(p.cluster, p.cluster * p.threads / 32) + 7) & ~7) + p.segment / 8;
        },
        &plan);
    if (rc != B200AMP_OK)
    {
        return rc;
    }
    return plan.threads == 64    ? launch_distill<T, 64>(a, plan, stream)
           : plan.threads == 128 ? launch_distill<T, 128>(a, plan, stream)
                                 : launch_distill<T, 256>(a, plan, stream);
}

int distill_timeout_take(int *out)
{
    return take_row_timeout(out);
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
    if (k == 0)
    {
        lse = nullptr;                          // no teacher: not read
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
                     temperature, soft_weight, hard_weight, st, row_loss, static_cast<LossWorkspace *>(workspace),
                     tunables().loss_test_starve - 1ll};
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
