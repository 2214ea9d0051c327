// row_tile.cuh: one row of a matrix held in the shared memory of a thread-block cluster.
//
// A vocabulary row is swept several times (maximum, sums, gradient) but should cross HBM once each way. The C
// blocks of a cluster take a segment of the row each (C = 1: the whole row) and keep it in shared memory between
// the sweeps; what the segments have to tell each other goes through distributed shared memory. A segment sits at the
// same offset from a 16-byte boundary as in global memory, so that all but its two ends moves in 16-byte accesses
// whatever the row's alignment.
#pragma once

#include <cooperative_groups.h>

#include <mutex>

#include "loss_common.cuh"

namespace b200amp
{

constexpr int MAX_CLUSTER = 16;
constexpr int MAX_ROW_SMEM = 220 * 1024;        // dynamic shared memory of a block at most

// How a matrix is spread: decided on the host, the same for every row.
struct RowPlan
{
    int cluster;            // blocks a row
    int segment;            // columns a block, a multiple of 64
    int threads;            // that sweep; the kernel may have a warp more
    int smem;               // dynamic shared memory of a block
};

// Cluster and block size (least .. most threads) for rows of `cols` elements of `size` bytes, with more(plan) bytes of shared memory
// besides the segment. B200AMP_ERR_LIMIT where a row does not fit the largest cluster.
template <typename More>
int plan_rows(long long rows, int cols, int size, int least, int most, More more, RowPlan *plan)
{
    auto fill = [&](int cluster, int threads) {
        plan->cluster = cluster;
        plan->threads = threads;
        plan->segment = static_cast<int>(((static_cast<long long>(cols) + cluster - 1) / cluster + 63) / 64 * 64);
        plan->smem = ((plan->segment * size + 31) & ~15) + more(*plan);
    };
    if (static_cast<long long>(cols) * size > MAX_CLUSTER * static_cast<long long>(MAX_ROW_SMEM))
    {
        set_error("rows of %d columns are beyond the maximum of %lld", cols,
                  MAX_CLUSTER * static_cast<long long>(MAX_ROW_SMEM) / size);
        return B200AMP_ERR_LIMIT;
    }
    // The fewest blocks that hold the row: what there is one of a segment (its barriers, its listed columns, its exchange
    // with the others) costs about as much as sweeping 10,000 columns, so fewer and longer segments win for 16-bit rows, even
    // where one block fills an SM (510 rows of 128,001 bf16 columns, top_logits: 2 blocks a row 160 us, 4 blocks 186 us; 8192
    // rows of 50,304 fp16 columns, distill_loss: 1 block 351 us, 2 blocks 452 us). For long fp32 rows it is about even (2048
    // rows of 131,072, distill_loss: 4 blocks 593 us, 8 blocks 582 us).
    int cluster = 1;
    for (fill(1, 256); cluster < MAX_CLUSTER && plan->smem > MAX_ROW_SMEM; fill(cluster, 256))
    {
        cluster *= 2;
    }
    if (plan->smem > MAX_ROW_SMEM)
    {
        set_error("rows of %d columns with what they list need %d bytes of shared memory in each of %d blocks, at most %d", cols,
                  plan->smem, MAX_CLUSTER, MAX_ROW_SMEM);
        return B200AMP_ERR_LIMIT;
    }
    const int sms = sm_count();
    if (sms <= 0)
    {
        return B200AMP_ERR_CUDA;
    }
    // A handful of rows: long ones are worth spreading over SMs that would stand idle.
    while (cluster < 4 && rows * cluster < sms && plan->segment > 16384)
    {
        cluster *= 2;
        fill(cluster, 256);
    }
    // A row costs a block some thousand cycles of barriers and short chains whatever its length, so short segments want
    // more and smaller blocks side by side (distill_loss, 8192 rows: of 700 fp16 columns 64 threads 59 us, 128 threads
    // 86 us, 256 threads 158 us; of 12,000 bf16 columns 117, 126 and 170 us), unless there are hardly rows for them; and
    // a block that has an SM to itself wants its threads (top_logits, 510 rows of 128,001 bf16 columns: 256 threads
    // 160 us, 512 threads 121 us), but not two that share one (8192 rows of 50,257 fp16 columns: 300 and 303 us).
    if (rows * cluster > 2ll * sms)
    {
        const int bytes = plan->segment * size;
        fill(cluster, bytes <= 32 * 1024 ? least : bytes <= 56 * 1024 ? 128 : 256);
    }
    if (plan->smem > 112 * 1024)
    {
        fill(cluster, most);
    }
    return B200AMP_OK;
}

#ifdef __CUDACC__

template <typename T>
struct Vec16                // 16 bytes of a row
{
    static constexpr int N = 16 / sizeof(T);
    uint4 w;
};

__device__ __forceinline__ float2 pair_of(uint32_t w, __half)
{
    return half2_bits_to_float2(w);
}
__device__ __forceinline__ float2 pair_of(uint32_t w, __nv_bfloat16)
{
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
__device__ __forceinline__ float2 pair_of(uint32_t w, float)
{
    return make_float2(__uint_as_float(w), __uint_as_float(w));
}

// the elements as pairs of floats
__device__ __forceinline__ void unpack(const Vec16<__half> &v, float2 (&f)[4])
{
    const uint32_t words[4] = {v.w.x, v.w.y, v.w.z, v.w.w};
#pragma unroll
    for (int i = 0; i < 4; i++)
    {
        f[i] = half2_bits_to_float2(words[i]);
    }
}
__device__ __forceinline__ void unpack(const Vec16<__nv_bfloat16> &v, float2 (&f)[4])
{
    const uint32_t words[4] = {v.w.x, v.w.y, v.w.z, v.w.w};
#pragma unroll
    for (int i = 0; i < 4; i++)
    {
        f[i] = make_float2(__uint_as_float(words[i] << 16), __uint_as_float(words[i] & 0xFFFF0000u));
    }
}
__device__ __forceinline__ void unpack(const Vec16<float> &v, float2 (&f)[2])
{
    f[0] = make_float2(__uint_as_float(v.w.x), __uint_as_float(v.w.y));
    f[1] = make_float2(__uint_as_float(v.w.z), __uint_as_float(v.w.w));
}

__device__ __forceinline__ void pack(Vec16<__half> &v, const float2 (&f)[4])
{
    v.w = make_uint4(float2_to_half2_bits(f[0].x, f[0].y), float2_to_half2_bits(f[1].x, f[1].y),
                     float2_to_half2_bits(f[2].x, f[2].y), float2_to_half2_bits(f[3].x, f[3].y));
}
__device__ __forceinline__ uint32_t bf16_pair(float2 f)
{
    __nv_bfloat162 b = __floats2bfloat162_rn(f.x, f.y);
    return *reinterpret_cast<uint32_t *>(&b);
}
__device__ __forceinline__ void pack(Vec16<__nv_bfloat16> &v, const float2 (&f)[4])
{
    v.w = make_uint4(bf16_pair(f[0]), bf16_pair(f[1]), bf16_pair(f[2]), bf16_pair(f[3]));
}
__device__ __forceinline__ void pack(Vec16<float> &v, const float2 (&f)[2])
{
    v.w = make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
}

// maximum with NaN winning, pair by pair in the element type
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, __half)
{
    __half2 r = __hmax2_nan(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
    return *reinterpret_cast<uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, __nv_bfloat16)
{
    __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162 *>(&a), *reinterpret_cast<__nv_bfloat162 *>(&b));
    return *reinterpret_cast<uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b, float)
{
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
}
template <typename T>
__device__ __forceinline__ void max_into(Vec16<T> &m, const Vec16<T> &v)
{
    m.w.x = max2_nan(m.w.x, v.w.x, T());
    m.w.y = max2_nan(m.w.y, v.w.y, T());
    m.w.z = max2_nan(m.w.z, v.w.z, T());
    m.w.w = max2_nan(m.w.w, v.w.w, T());
}
template <typename T>
__device__ __forceinline__ float max_of(const Vec16<T> &v)
{
    float2 f[Vec16<T>::N / 2];
    unpack(v, f);
    float m = max_nan(f[0].x, f[0].y);
#pragma unroll
    for (int i = 1; i < Vec16<T>::N / 2; i++)
    {
        m = max_nan(m, max_nan(f[i].x, f[i].y));
    }
    return m;
}

template <typename T>
__device__ __forceinline__ T minus_infinity()
{
    return from_float<T>(-INFINITY);
}

// two fp32 operations in one instruction
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return r;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(r))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
          "l"(reinterpret_cast<unsigned long long &>(c)));
    return r;
}

// Set when a wait for a row's copy ran out; each source file that includes this has its own.
static __device__ int g_row_timeout = 0;

// Bulk copies: one thread hands a whole segment to the copy engine, which completes its bytes on a barrier in shared
// memory. (Copied by cp.async, 16 bytes a thread, the threads themselves wait for the memory system to take the
// requests: a fifth of a row's time.)
__device__ __forceinline__ uint32_t shared_address(const void *p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void row_barrier_init(uint64_t *bar)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" : : "r"(shared_address(bar)) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" : : : "memory");
}
// never: bytes that are announced and do not come (a test's, else 0).
__device__ __forceinline__ void row_copy(void *dst, const void *src, unsigned bytes, unsigned never, uint64_t *bar)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                 :
                 : "r"(shared_address(bar)), "r"(bytes + never)
                 : "memory");
    if (bytes > 0)
    {
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     :
                     : "r"(shared_address(dst)), "l"(src), "r"(bytes), "r"(shared_address(bar))
                     : "memory");
    }
}
// Bounded: false when the limit ran out, which only a copy that never completes can bring about. A poll of an open phase
// takes 2 us (distill_loss) to 4 us (top_logits), as the hardware suspends the thread: half a second to one second in all.
__device__ __forceinline__ bool row_wait(uint64_t *bar, unsigned parity)
{
    for (unsigned tries = 0; tries < 1u << 18; tries++)
    {
        unsigned ok;
        asm volatile("{\n\t.reg .pred p;\n\t"
                     "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                     "selp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(ok)
                     : "r"(shared_address(bar)), "r"(parity)
                     : "memory");
        if (ok != 0)
        {
            return true;
        }
    }
    return false;
}
// What this thread wrote to shared memory comes before copies that are started after a barrier.
__device__ __forceinline__ void before_copies()
{
    asm volatile("fence.proxy.async.shared::cta;" : : : "memory");
}

// NaN in the place of a row that did not come. A call, so that it costs the rows that come nothing.
static __device__ __noinline__ void lose_row(char *buf, int vecs, int threads)
{
    g_row_timeout = 1;
    for (int i = threadIdx.x; i < vecs; i += threads)
    {
        reinterpret_cast<uint4 *>(buf)[i] = make_uint4(~0u, ~0u, ~0u, ~0u);
    }
}

// This block's segment of the current row.
template <typename T, int THREADS>
struct RowTile
{
    static constexpr int N = Vec16<T>::N;
    char *buf;              // 16-byte aligned: segment * sizeof(T) + 16 bytes
    int first;              // first column of the segment
    int lead;               // elements between buf and the first column's place (0 .. N - 1)
    int valid, held;        // columns of the segment that hold logits, and with the padding behind them
    int vecs;               // 16-byte vectors to sweep; what is in none of the columns holds -inf
    bool uneven;            // rows start at different places between 16-byte boundaries, so a copy covers other rows' ends
    int edge_at;            // this thread's element outside the whole vectors, -1: none
    T edge;

    __device__ __forceinline__ T *at(int column)            // of this segment, in shared memory
    {
        return reinterpret_cast<T *>(buf) + lead + (column - first);
    }
    __device__ __forceinline__ Vec16<T> vec(int i) const
    {
        return reinterpret_cast<const Vec16<T> *>(buf)[i];
    }

    // Starts the copy of columns [first, first + valid) of the row at z; padding and ends are set to -inf. Every
    // thread, after a barrier behind the last use of the segment; the row is there after row_wait and a barrier.
    // phase: the one that wait() keeps. starved: a test's, this copy never completes.
    __device__ __forceinline__ void start(const T *z, int first_column, int segment, int vocab, int cols, uint64_t *bar, unsigned phase,
                                          bool starved)
    {
        first = first_column;
        valid = max(0, min(segment, vocab - first));
        held = max(0, min(segment, cols - first));
        const char *src = reinterpret_cast<const char *>(z + first);
        const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15);
        lead = skew / static_cast<int>(sizeof(T));
        vecs = held > 0 ? (lead + held + N - 1) / N : 0;
        const int whole_first = lead > 0 ? 1 : 0, whole_end = (lead + valid) / N;      // vectors inside the columns
        src -= skew;
        if (threadIdx.x == 0 && phase < 2u)
        {
            row_copy(buf + 16 * whole_first, src + 16 * whole_first, 16u * max(0, whole_end - whole_first), starved ? 16u : 0u, bar);
        }
        // the elements of the other vectors: at most N - 1 at the front, then the end and the padding. Those that hold
        // logits (2 N - 2 at most, one a thread) are fetched here and put in place by finish.
        T *e = reinterpret_cast<T *>(buf);
        const T *g = reinterpret_cast<const T *>(src);
        const int front = whole_first * N, back = max(front, whole_end * N);
        edge_at = -1;
        bool wrote = false;
        for (int i = threadIdx.x; i < front + (vecs * N - back); i += THREADS)
        {
            const int k = i < front ? i : back + i - front;
            if (k >= lead && k < lead + valid)
            {
                edge = g[k];
                edge_at = k;
            }
            else
            {
                e[k] = minus_infinity<T>();
                wrote = true;
            }
        }
        if (wrote && uneven)
        {
            before_copies();
        }
    }
    // Waits for the row and puts the elements in place that the copy engine does not move; a barrier follows. phase: the
    // barrier's, 0 at first. Where the wait gives up, 2 is added to it and stays: the phase is still open, so this block
    // waits for and (thread 0) starts no copy any more, and from this row on it has NaN in place of the logits.
    __device__ __forceinline__ void wait(uint64_t *bar, unsigned &phase)
    {
        if (phase < 2u && row_wait(bar, phase))
        {
            phase ^= 1u;
        }
        else
        {
            phase |= 2u;
            lose_row(buf, vecs, THREADS);
        }
        if (edge_at >= 0)
        {
            reinterpret_cast<T *>(buf)[edge_at] = edge;
            if (uneven)
            {
                before_copies();
            }
        }
    }
};

// Before a block leaves, thread 0: another bounded wait for a copy that was given up, so that shared memory is not handed
// back with it on its way.
__device__ __forceinline__ void row_leave(uint64_t *bar, unsigned phase)
{
    if (phase >= 2u)
    {
        row_wait(bar, phase & 1u);
    }
}

// *out |= 1 if a wait for a row's copy gave up in this source file's kernels since the last call (clears it).
static int take_row_timeout(int *out)
{
    int flag = 0;
    B200AMP_CUDA(cudaMemcpyFromSymbol(&flag, g_row_timeout, sizeof(int)));
    if (flag != 0)
    {
        const int zero = 0;
        B200AMP_CUDA(cudaMemcpyToSymbol(g_row_timeout, &zero, sizeof(int)));
        *out |= 1;
    }
    return B200AMP_OK;
}

// Blocks of a kernel that fit the device at once, as whole clusters (asked once for each shape).
template <typename Kernel>
int resident_clusters(Kernel kernel, const RowPlan &plan, int threads, int *clusters)
{
    struct Known
    {
        const void *kernel;
        int device, cluster, smem, clusters;
    };
    static std::mutex lock;
    static Known known[64];
    static int count = 0;
    int device = 0;
    B200AMP_CUDA(cudaGetDevice(&device));
    std::lock_guard<std::mutex> hold(lock);
    for (int i = 0; i < count && i < 64; i++)
    {
        if (known[i].kernel == reinterpret_cast<const void *>(kernel) && known[i].device == device && known[i].cluster == plan.cluster && known[i].smem == plan.smem)
        {
            *clusters = known[i].clusters;
            return B200AMP_OK;
        }
    }
    B200AMP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_ROW_SMEM));
    B200AMP_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(plan.cluster);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = plan.smem;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim = {static_cast<unsigned>(plan.cluster), 1u, 1u};
    config.attrs = attribute;
    config.numAttrs = 1;
    int n = 0;
    B200AMP_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &config));
    if (n < 1)
    {
        set_error("no cluster of %d blocks with %d bytes of shared memory fits the device", plan.cluster, plan.smem);
        return B200AMP_ERR_CUDA;
    }
    known[count % 64] = {reinterpret_cast<const void *>(kernel), device, plan.cluster, plan.smem, n};
    count++;
    *clusters = n;
    return B200AMP_OK;
}

template <typename Kernel, typename Args>
int launch_rows(Kernel kernel, const Args &args, RowPlan plan, int threads, long long rows, cudaStream_t stream)
{
    int clusters = 0;
    const int rc = resident_clusters(kernel, plan, threads, &clusters);
    if (rc != B200AMP_OK)
    {
        return rc;
    }
    clusters = static_cast<int>(rows < 1 ? 1 : rows < clusters ? rows : clusters);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(clusters * plan.cluster);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = plan.smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim = {static_cast<unsigned>(plan.cluster), 1u, 1u};
    config.attrs = attribute;
    config.numAttrs = 1;
    B200AMP_CUDA(cudaLaunchKernelEx(&config, kernel, args, plan));
    B200AMP_LAUNCHED();
    return B200AMP_OK;
}

#endif // __CUDACC__

} // namespace b200amp
