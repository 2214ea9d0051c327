// top_logits.cu: a teacher's record: of every row the k largest logits in descending order
// (ties to the lowest column), their columns, and the log-sum-exp of the whole row.
//
// A row is held in shared memory (row_tile.cuh) and swept twice. The first sweep takes maxima, one for each thread
// and place in a 16-byte vector: a thousand or two groups of columns. A value that k of these maxima reach is reached
// by k columns of the row, and by few more: the second sweep, which also sums the powers for the log-sum-exp, collects
// the columns that reach it, and only they are sorted. Rows where too many do (equal logits, masks) are selected
// by histograms of the keys, digit by digit.

#include "row_tile.cuh"

namespace b200amp
{

constexpr int MOST_BROUGHT = 2048;      // listed columns of a cluster that a block copies before it searches them

struct TopArgs
{
    const void *logits;
    long long ld, rows;
    int vocab, k, room;         // room: columns that a block can collect, a power of two, at least 2 k
    double temperature;
    void *values;
    int *indices;
    float *lse;
    long long starved;          // row whose copy a test keeps from completing, -1: none
};

// A key that orders as the numbers do: -0 as +0, every NaN above +inf.
__device__ __forceinline__ unsigned int order_key(float v)
{
    unsigned int u = __float_as_uint(v);
    if (v != v)
    {
        return 0xFFFFFFFFu;
    }
    if (v == 0.0f)
    {
        u = 0u;
    }
    return (u & 0x80000000u) != 0 ? ~u : u | 0x80000000u;
}
// The number of a key; some NaN for the keys of no number.
__device__ __forceinline__ float key_value(unsigned int key)
{
    return __uint_as_float((key & 0x80000000u) != 0 ? key ^ 0x80000000u : ~key);
}
// Larger first, then the lower column: entries of a row are all different.
__device__ __forceinline__ unsigned long long entry_of(unsigned int key, int column)
{
    return static_cast<unsigned long long>(key) << 32 | static_cast<unsigned int>(~column);
}
__device__ __forceinline__ int column_of(unsigned long long entry)
{
    return static_cast<int>(~static_cast<unsigned int>(entry));
}

// Whether an element may be at least `least` (NaN: yes).
template <typename T>
__device__ __forceinline__ bool reaches(const Vec16<T> &v, float least)
{
    const uint32_t m = max2_nan(max2_nan(v.w.x, v.w.y, T()), max2_nan(v.w.z, v.w.w, T()), T());
    if (sizeof(T) == 4)
    {
        return !(__uint_as_float(m) < least);
    }
    const float2 f = pair_of(m, T());
    return !(f.x < least) || !(f.y < least);
}

// Descending order of list[0 .. n); size: a power of two, n <= size. Every thread.
template <int THREADS>
__device__ __forceinline__ void sort_entries(unsigned long long *list, int n, int size)
{
    for (int i = n + threadIdx.x; i < size; i += THREADS)
    {
        list[i] = 0ull;
    }
    for (int span = 2; span <= size; span <<= 1)
    {
        for (int step = span >> 1; step > 0; step >>= 1)
        {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += THREADS)
            {
                const int lo = 2 * i - (i & (step - 1)), hi = lo + step;
                const unsigned long long x = list[lo], y = list[hi];
                if ((x < y) == ((lo & span) == 0))
                {
                    list[lo] = y;
                    list[hi] = x;
                }
            }
        }
    }
    __syncthreads();
}

// The `kept` largest columns of the segment into list, in no order: their smallest key by four rounds of a histogram
// (8 bits a round, from the top), then one sweep in column order that keeps what is above it and the first of those equal.
template <typename T, int THREADS>
__device__ __noinline__ void select_by_digits(const T *z, int first, int valid, unsigned int kept, unsigned long long *list,
                                              unsigned int *bins)
{
    __shared__ unsigned int warp_above[THREADS / 32], warp_equal[THREADS / 32];
    __shared__ unsigned int prefix_s, need_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned int prefix = 0u, mask = 0u, need = kept;
    for (int shift = 24; shift >= 0; shift -= 8)
    {
        for (int b = tid; b < 256; b += THREADS)
        {
            bins[b] = 0u;
        }
        __syncthreads();
        for (int v = tid; v < valid; v += THREADS)
        {
            const unsigned int key = order_key(to_float(z[v]));
            if ((key & mask) == prefix)
            {
                atomicAdd(&bins[key >> shift & 255u], 1u);
            }
        }
        __syncthreads();
        if (tid == 0)
        {
            unsigned int left = need;
            int b = 255;
            while (b > 0 && bins[b] < left)
            {
                left -= bins[b];
                b--;
            }
            prefix_s = prefix | static_cast<unsigned int>(b) << shift;
            need_s = left;
        }
        __syncthreads();
        prefix = prefix_s;
        need = need_s;                          // of those equal to the prefix
        mask |= 255u << shift;
        __syncthreads();
    }
    const unsigned int above_all = kept - need;
    unsigned int above = 0u, equal = 0u;
    for (int base = 0; base < valid; base += THREADS)
    {
        const int v = base + tid;
        const unsigned int key = v < valid ? order_key(to_float(z[v])) : 0u;
        const bool is_above = v < valid && key > prefix, is_equal = v < valid && key == prefix;
        const unsigned int ba = __ballot_sync(0xffffffffu, is_above), be = __ballot_sync(0xffffffffu, is_equal);
        if (lane == 0)
        {
            warp_above[warp] = __popc(ba);
            warp_equal[warp] = __popc(be);
        }
        __syncthreads();
        unsigned int at_above = above, at_equal = equal;
        for (int w = 0; w < THREADS / 32; w++)
        {
            at_above += w < warp ? warp_above[w] : 0u;
            at_equal += w < warp ? warp_equal[w] : 0u;
            above += warp_above[w];
            equal += warp_equal[w];
        }
        const unsigned int before = (1u << lane) - 1u;
        at_above += __popc(ba & before);
        at_equal += __popc(be & before);
        if (is_above && at_above < kept)        // they are fewer, unless a copy that was given up changes the row meanwhile
        {
            list[at_above] = entry_of(key, first + v);
        }
        if (is_equal && at_equal < need)
        {
            list[above_all + at_equal] = entry_of(key, first + v);
        }
        __syncthreads();
    }
}

// A cluster a row. 8192 rows of 50257 fp16 columns, k 64: 320 us, 0.83 GB, 2.6 TB/s (the bytes alone 126 us, the powers
// 92 us). A row of a block takes about 20,000 cycles: 8,000 the second sweep, 3,000 the threshold, 2,000 each the
// collection and the sorting, 1,500 the first sweep; the next row's copy is under the sorting. 64 registers a thread, for two
// blocks of 512 an SM or eight of 128, with 4 to 24 bytes of spills.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) top_rows_kernel(const TopArgs a, const RowPlan plan)
{
    namespace cg = cooperative_groups;
    using Tile = RowTile<T, THREADS>;
    constexpr int N = Tile::N, PAIRS = N / 2, WARPS = THREADS / 32;
    extern __shared__ __align__(16) char dynamic[];
    __shared__ uint64_t row_bar;
    __shared__ unsigned int bins[256];
    __shared__ unsigned int warp_hi[WARPS], warp_lo[WARPS];
    __shared__ int4 found;                      // a bin, the groups above it, those in it too
    __shared__ float warp_m[WARPS], warp_s[WARPS];
    __shared__ float2 block_ms[2];              // of two rows: this segment's maximum and sum
    __shared__ int collected, met;              // columns that reach, vectors that hold some
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const cg::cluster_group cluster = cg::this_cluster();
    const int blocks = plan.cluster, rank = blocks > 1 ? static_cast<int>(cluster.block_rank()) : 0;
    const int first = rank * plan.segment;
    const long long clusters = gridDim.x / blocks;
    const double inv_t = 1.0 / a.temperature;
    const float c_t = static_cast<float>(1.4426950408889634 * inv_t);

    // dynamic shared memory: the segment; the collected columns and the vectors that hold them; two rows' sorted best of the segment; the cluster's
    const size_t tile_bytes = (static_cast<size_t>(plan.segment) * sizeof(T) + 31) & ~static_cast<size_t>(15);
    Tile tile;
    tile.buf = dynamic;
    tile.uneven = (a.ld * static_cast<long long>(sizeof(T)) & 15) != 0;
    unsigned long long *const list = reinterpret_cast<unsigned long long *>(dynamic + tile_bytes);
    int *const vectors = reinterpret_cast<int *>(list + a.room);
    unsigned long long *const best0 = list + a.room + a.room / 2;
    unsigned long long *const others = best0 + 2 * a.k;     // every segment's, brought over where they are few
    const bool brought = blocks * a.k <= MOST_BROUGHT;
    unsigned int phase = 0u;                    // of row_bar, with what RowTile::wait adds
    auto start = [&](long long row) {
        tile.start(static_cast<const T *>(a.logits) + row * a.ld, first, plan.segment, a.vocab, a.vocab, &row_bar, phase,
                   row == a.starved && rank == blocks - 1);
    };
    if (tid == 0)
    {
        row_barrier_init(&row_bar);
    }
    __syncthreads();
    if (blocks > 1)
    {
        cluster.sync();                         // every block of the cluster runs before one reads of another
    }

    int parity = 0;
    long long row = blockIdx.x / blocks;
    if (row < a.rows)
    {
        start(row);
    }
    for (; row < a.rows; row += clusters, parity ^= 1)
    {
        unsigned long long *const best = best0 + parity * a.k;
        const int valid = tile.valid;
        const int kept = min(a.k, valid);       // of this segment
        if (tid == 0)
        {
            collected = 0;
            met = 0;
        }
        tile.wait(&row_bar, phase);
        __syncthreads();

        // maxima of the groups
        Vec16<T> group;
        {
            const T low = minus_infinity<T>();
            T *e = reinterpret_cast<T *>(&group);
#pragma unroll
            for (int i = 0; i < N; i++)
            {
                e[i] = low;
            }
        }
        {
            int i = tid;
            for (; i + 3 * THREADS < tile.vecs; i += 4 * THREADS)
            {
                Vec16<T> v0 = tile.vec(i), v1 = tile.vec(i + THREADS), v2 = tile.vec(i + 2 * THREADS), v3 = tile.vec(i + 3 * THREADS);
                max_into(v0, v1);
                max_into(v2, v3);
                max_into(group, v0);
                max_into(group, v2);
            }
            for (; i < tile.vecs; i += THREADS)
            {
                max_into(group, tile.vec(i));
            }
        }
        unsigned int key[N];
        float m = -INFINITY;
        {
            float2 f[PAIRS];
            unpack(group, f);
#pragma unroll
            for (int q = 0; q < PAIRS; q++)
            {
                key[2 * q] = order_key(f[q].x);
                key[2 * q + 1] = order_key(f[q].y);
                m = max_nan(m, max_nan(f[q].x, f[q].y));
            }
        }
        // as many groups as are needed: four times k, or all (fewer would let too many columns through)
        int per = N;
#pragma unroll
        for (int half = N / 2; half > 0; half >>= 1)
        {
            if (per == 2 * half && THREADS * half >= 4 * a.k)
            {
                per = half;
#pragma unroll
                for (int i = 0; i < half; i++)
                {
                    key[i] = max(key[i], key[i + half]);
                }
            }
        }
        unsigned int hi = key[0], lo = key[0];
#pragma unroll
        for (int i = 1; i < N; i++)
        {
            if (i < per)
            {
                hi = max(hi, key[i]);
                lo = min(lo, key[i]);
            }
        }
        hi = __reduce_max_sync(0xffffffffu, hi);
        lo = __reduce_min_sync(0xffffffffu, lo);
        m = warp_max_nan(m);
        if (lane == 0)
        {
            warp_hi[warp] = hi;
            warp_lo[warp] = lo;
            warp_m[warp] = m;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WARPS; w++)
        {
            hi = max(hi, warp_hi[w]);
            lo = min(lo, warp_lo[w]);
            m = max_nan(m, warp_m[w]);
        }

        // a key that at least k groups reach, and not many more: their histogram over the range of the keys, and again
        // over the bin of the k-th largest while that holds too many
        unsigned int reach = 0u;                // short segments are collected whole
        if (valid > a.room / 2 && THREADS * N >= a.k)
        {
            int above = 0;                      // groups above the range at hand
            reach = lo;
            unsigned int span = hi - lo;        // the range: reach .. reach + span
            for (;;)
            {
                const int shift = max(0, 24 - __clz(static_cast<int>(span | 1u)));     // 256 bins or fewer
                for (int i = tid; i < 256; i += THREADS)
                {
                    bins[i] = 0u;
                }
                __syncthreads();
#pragma unroll
                for (int i = 0; i < N; i++)
                {
                    if (i < per && key[i] >= reach && key[i] - reach <= span)
                    {
                        atomicAdd(&bins[(key[i] - reach) >> shift], 1u);
                    }
                }
                __syncthreads();
                if (warp == 0)
                {
                    // lane l: bins 255 - 8 l .. 248 - 8 l, from the top
                    int mine = 0;
#pragma unroll
                    for (int i = 0; i < 8; i++)
                    {
                        mine += static_cast<int>(bins[255 - 8 * lane - i]);
                    }
                    int upto = mine;
#pragma unroll
                    for (int offset = 1; offset < 32; offset <<= 1)
                    {
                        const int below = __shfl_up_sync(0xffffffffu, upto, offset);
                        upto += lane >= offset ? below : 0;
                    }
                    const unsigned int enough = __ballot_sync(0xffffffffu, above + upto >= a.k);
                    if (lane == __ffs(static_cast<int>(enough)) - 1)
                    {
                        int count = above + upto - mine;        // above the lane's bins
                        int bin = 255 - 8 * lane, over = count;
                        for (;; bin--)
                        {
                            over = count;
                            count += static_cast<int>(bins[bin]);
                            if (count >= a.k)
                            {
                                break;
                            }
                        }
                        found = make_int4(bin, over, count, 0);
                    }
                }
                __syncthreads();
                const int4 f = found;
                reach += static_cast<unsigned int>(f.x) << shift;
                if (f.z <= a.k + max(16, a.k / 4) || shift == 0)
                {
                    break;
                }
                above = f.y;
                span = (1u << shift) - 1u;
            }
        }

        // the columns that reach it, and the sum
        const float least = key_value(reach), ref = m == -INFINITY ? 0.0f : m;
        const bool sums = a.lse != nullptr;
        float2 sum = make_float2(0.0f, 0.0f);
        auto visit = [&](int i, const Vec16<T> &v) {
            float2 f[PAIRS];
            unpack(v, f);
            if (sums)
            {
#pragma unroll
                for (int q = 0; q < PAIRS; q++)
                {
                    const float2 x = mul2(add2(f[q], make_float2(-ref, -ref)), make_float2(c_t, c_t));
                    sum = add2(sum, make_float2(exp2_fast(x.x), exp2_fast(x.y)));
                }
            }
            if (reaches(v, least))
            {
                const int to = atomicAdd(&met, 1);
                if (to < a.room)
                {
                    vectors[to] = i;            // looked at once the sweep is over, by as many threads as it has elements
                }
            }
        };
        {
            int i = tid;
            for (; i + THREADS < tile.vecs; i += 2 * THREADS)
            {
                const Vec16<T> v0 = tile.vec(i), v1 = tile.vec(i + THREADS);
                visit(i, v0);
                visit(i + THREADS, v1);
            }
            if (i < tile.vecs)
            {
                visit(i, tile.vec(i));
            }
        }
        const float s = warp_sum_f32(sum.x + sum.y);
        if (lane == 0)
        {
            warp_s[warp] = s;
        }
        __syncthreads();
        int n = met;
        if (n <= a.room)
        {
            for (int x = tid; x < n * N; x += THREADS)
            {
                const int at = vectors[x / N] * N + x % N, column = at - tile.lead;
                const unsigned int at_key = order_key(to_float(reinterpret_cast<const T *>(tile.buf)[at]));
                if (at_key >= reach && column >= 0 && column < valid)
                {
                    const int to = atomicAdd(&collected, 1);
                    if (to < a.room)
                    {
                        list[to] = entry_of(at_key, first + column);
                    }
                }
            }
            __syncthreads();
            n = collected;
        }
        if (n > a.room)
        {
            select_by_digits<T, THREADS>(reinterpret_cast<const T *>(tile.buf) + tile.lead, first, valid, kept, list, bins);
            n = kept;
        }
        if (row + clusters < a.rows)
        {
            start(row + clusters);              // on its way while this row's few columns are sorted
        }
        if (tid == 0)
        {
            double total = 0.0;
            for (int w = 0; w < WARPS; w++)
            {
                total += warp_s[w];
            }
            block_ms[parity] = make_float2(m, static_cast<float>(total));
        }

        // the best of the segment in order
        if (n <= 2 * THREADS)
        {
            // an entry's place is the number of larger ones, counted by `lanes` neighbours
            int lanes = 1;
            while (lanes < 8 && 2 * lanes * n <= THREADS)
            {
                lanes *= 2;
            }
            for (int x0 = 0; x0 < n * lanes; x0 += THREADS)
            {
                const int x = x0 + tid, i = x / lanes;
                const unsigned long long mine = i < n ? list[i] : ~0ull;
                int place = 0;
                if (x0 + warp * 32 < n * lanes)
                {
#pragma unroll 4
                    for (int j = x % lanes; j < n; j += lanes)
                    {
                        place += list[j] > mine ? 1 : 0;
                    }
                }
                for (int offset = lanes >> 1; offset > 0; offset >>= 1)
                {
                    place += __shfl_xor_sync(0xffffffffu, place, offset);
                }
                if (i < n && x % lanes == 0 && place < kept)
                {
                    best[place] = mine;
                }
            }
            __syncthreads();
        }
        else
        {
            int size = 2;
            while (size < n)
            {
                size <<= 1;
            }
            sort_entries<THREADS>(list, n, size);
            for (int i = tid; i < kept; i += THREADS)
            {
                best[i] = list[i];
            }
            __syncthreads();
        }

        // the best of the row: an entry's place is the number of larger ones in every segment
        if (blocks > 1)
        {
            cluster.sync();
            for (int i = tid; brought && i < blocks * a.k; i += THREADS)
            {
                const int b = i / a.k, j = i - b * a.k;
                const int there_kept = min(a.k, max(0, min(plan.segment, a.vocab - b * plan.segment)));
                others[i] = j < there_kept ? cluster.map_shared_rank(best, b)[j] : 0ull;
            }
            __syncthreads();
        }
        for (int j = tid; j < kept; j += THREADS)
        {
            const unsigned long long entry = best[j];
            int place = j;
            for (int b = 0; b < blocks && place < a.k; b++)
            {
                if (b != rank)
                {
                    const unsigned long long *other = brought ? others + b * a.k : cluster.map_shared_rank(best, b);
                    int from = 0, to = min(a.k, max(0, min(plan.segment, a.vocab - b * plan.segment)));
                    while (from < to)
                    {
                        const int mid = (from + to) / 2;
                        if (other[mid] > entry)
                        {
                            from = mid + 1;
                        }
                        else
                        {
                            to = mid;
                        }
                    }
                    place += from;
                }
            }
            if (place < a.k)
            {
                a.indices[row * a.k + place] = column_of(entry);
                static_cast<T *>(a.values)[row * a.k + place] = from_float<T>(key_value(static_cast<unsigned int>(entry >> 32)));
            }
        }
        if (rank == 0)
        {
            for (int j = a.vocab + tid; j < a.k; j += THREADS)
            {
                a.indices[row * a.k + j] = -1;  // fewer columns than asked for
                static_cast<T *>(a.values)[row * a.k + j] = minus_infinity<T>();
            }
            if (sums && tid == 0)
            {
                float all = -INFINITY;
                for (int b = 0; b < blocks; b++)
                {
                    all = max_nan(all, (blocks > 1 ? cluster.map_shared_rank(block_ms, b) : block_ms)[parity].x);
                }
                double total = 0.0;
                for (int b = 0; b < blocks; b++)
                {
                    const float2 ms = (blocks > 1 ? cluster.map_shared_rank(block_ms, b) : block_ms)[parity];
                    total += ms.x == -INFINITY ? 0.0 : ms.y * exp((static_cast<double>(ms.x) - all) * inv_t);
                }
                // a row of nothing but -inf has the log of 0; +inf has itself
                a.lse[row] = isinf(all) ? all : static_cast<float>(all * inv_t + log(total));
            }
        }
    }
    if (tid == 0)
    {
        row_leave(&row_bar, phase);
    }
    if (blocks > 1)
    {
        cluster.sync();                         // no block leaves while another reads its last row
    }
}

template <typename T>
static int launch_top(TopArgs a, cudaStream_t stream)
{
    a.room = 256;
    while (a.room < 2 * a.k)
    {
        a.room *= 2;
    }
    RowPlan plan;
    const int rc = plan_rows(
        a.rows, a.vocab, sizeof(T), 128, 512, [&](const RowPlan &p) {
            return (a.room + a.room / 2 + 2 * a.k + (p.cluster > 1 && p.cluster * a.k <= MOST_BROUGHT ? p.cluster * a.k : 0)) *
                   static_cast<int>(sizeof(unsigned long long));
        },
        &plan);
    if (rc != B200AMP_OK)
    {
        return rc;
    }
    return plan.threads == 128   ? launch_rows(top_rows_kernel<T, 128>, a, plan, 128, a.rows, stream)
           : plan.threads == 256 ? launch_rows(top_rows_kernel<T, 256>, a, plan, 256, a.rows, stream)
                                 : launch_rows(top_rows_kernel<T, 512>, a, plan, 512, a.rows, stream);
}

int top_timeout_take(int *out)
{
    return take_row_timeout(out);
}

} // namespace b200amp

using namespace b200amp;

extern "C" B200AMP_API int b200amp_top_logits(const void *logits, int dtype, long long rows, int vocab, long long ld,
                                              int k, double temperature, void *values, int *indices, float *lse,
                                              b200amp_stream s)
{
    B200AMP_REQUIRE(dtype_known(dtype), "top_logits: dtype %d is none of F16, BF16, F32", dtype);
    B200AMP_REQUIRE(rows >= 0 && rows <= INT_MAX, "top_logits: %lld rows, must be 0..%d", rows, INT_MAX);
    B200AMP_REQUIRE(vocab >= 1 && vocab <= ld, "top_logits: vocab %d, ld %lld: need 1 <= vocab <= ld", vocab, ld);
    B200AMP_REQUIRE(k >= 1 && k <= B200AMP_MAX_LISTED, "top_logits: k = %d, must be 1..%d", k, B200AMP_MAX_LISTED);
    B200AMP_REQUIRE(std::isfinite(temperature) && temperature > 0.0 && std::isfinite(static_cast<float>(1.4426950408889634 / temperature)) &&
                        static_cast<float>(1.4426950408889634 / temperature) > 0.0f,
                    "top_logits: temperature %g", temperature);
    const size_t size = static_cast<size_t>(dtype_size(dtype));
    B200AMP_REQUIRE((logits != nullptr && values != nullptr && indices != nullptr) || rows == 0,
                    "top_logits: logits, values or indices is null");
    B200AMP_REQUIRE(aligned(logits, size) && aligned(values, size) && aligned(indices, 4) && aligned(lse, 4),
                    "top_logits: an array is not aligned to its element type");
    if (rows == 0)
    {
        return B200AMP_OK;
    }
    const TopArgs a = {logits, ld, rows, vocab, k, 0, temperature, values, indices, lse, tunables().loss_test_starve - 1ll};
    switch (dtype)
    {
    case B200AMP_F16:
        return launch_top<__half>(a, as_stream(s));
    case B200AMP_BF16:
        return launch_top<__nv_bfloat16>(a, as_stream(s));
    default:
        return launch_top<float>(a, as_stream(s));
    }
}
