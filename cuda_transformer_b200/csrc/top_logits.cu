// top_logits.cu: a teacher's record: of every row the k largest logits in descending order
// (ties to the lowest column), their columns, and the log-sum-exp of the whole row.

#include "loss_common.cuh"

namespace b200amp
{

constexpr int TOP_THREADS = 512;

struct TopArgs
{
    const void *logits;
    long long ld, rows;
    int vocab, k;
    double temperature;
    void *values;
    int *indices;
    float *lse;
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

// One block a row: the k-th largest key by four rounds of a 256-bin histogram (8 bits a round, from
// the top), then one sweep in column order that keeps what is above it and the first of those equal to it.
template <typename T>
__global__ void __launch_bounds__(TOP_THREADS) top_rows_kernel(TopArgs a)
{
    __shared__ unsigned long long list[B200AMP_MAX_LISTED];
    __shared__ unsigned int bins[256];
    __shared__ double scratch[TOP_THREADS / 32];
    __shared__ unsigned int warp_above[TOP_THREADS / 32], warp_equal[TOP_THREADS / 32];
    __shared__ unsigned int prefix_s, need_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kept = a.k < a.vocab ? a.k : a.vocab;
    const double inv_t = 1.0 / a.temperature;
    const float c_t = static_cast<float>(1.4426950408889634 * inv_t);

    for (long long row = blockIdx.x; row < a.rows; row += gridDim.x)
    {
        const T *z = static_cast<const T *>(a.logits) + row * a.ld;
        if (a.lse != nullptr)
        {
            float m = -INFINITY;
            for (int v = tid; v < a.vocab; v += TOP_THREADS)
            {
                m = max_nan(m, to_float(z[v]));
            }
            m = block_max_nan<TOP_THREADS>(m, scratch);
            float sum = 0.0f;
            for (int v = tid; v < a.vocab; v += TOP_THREADS)
            {
                sum += exp2_fast((to_float(z[v]) - m) * c_t);
            }
            const double total = block_sum_f64<TOP_THREADS>(static_cast<double>(sum), scratch);
            if (tid == 0)
            {
                // a row of nothing but -inf has the log of 0; +inf has itself
                a.lse[row] = isinf(m) ? m : static_cast<float>(m * inv_t + log(total));
            }
        }

        unsigned int prefix = 0u, mask = 0u, need = kept;
        for (int shift = 24; shift >= 0; shift -= 8)
        {
            for (int b = tid; b < 256; b += TOP_THREADS)
            {
                bins[b] = 0u;
            }
            __syncthreads();
            for (int v = tid; v < a.vocab; v += TOP_THREADS)
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
            need = need_s;                      // of those equal to the prefix
            mask |= 255u << shift;
            __syncthreads();
        }

        // prefix is the key of the k-th largest: all above it, and the first `need` equal to it
        const unsigned int above_all = kept - need;
        unsigned int above = 0u, equal = 0u;
        for (int base = 0; base < a.vocab; base += TOP_THREADS)
        {
            const int v = base + tid;
            const unsigned int key = v < a.vocab ? order_key(to_float(z[v])) : 0u;
            const bool is_above = v < a.vocab && key > prefix, is_equal = v < a.vocab && key == prefix;
            const unsigned int ba = __ballot_sync(0xffffffffu, is_above), be = __ballot_sync(0xffffffffu, is_equal);
            if (lane == 0)
            {
                warp_above[warp] = __popc(ba);
                warp_equal[warp] = __popc(be);
            }
            __syncthreads();
            unsigned int at_above = above, at_equal = equal;
            for (int w = 0; w < TOP_THREADS / 32; w++)
            {
                at_above += w < warp ? warp_above[w] : 0u;
                at_equal += w < warp ? warp_equal[w] : 0u;
                above += warp_above[w];
                equal += warp_equal[w];
            }
            const unsigned int before = (1u << lane) - 1u;
            at_above += __popc(ba & before);
            at_equal += __popc(be & before);
            const unsigned long long entry = static_cast<unsigned long long>(key) << 32 | static_cast<unsigned int>(~v);
            if (is_above)
            {
                list[at_above] = entry;
            }
            if (is_equal && at_equal < need)
            {
                list[above_all + at_equal] = entry;
            }
            __syncthreads();
        }

        // descending order of (key, -column)
        int size = 1;
        while (size < kept)
        {
            size <<= 1;
        }
        for (int i = kept + tid; i < size; i += TOP_THREADS)
        {
            list[i] = 0ull;
        }
        for (int span = 2; span <= size; span <<= 1)
        {
            for (int step = span >> 1; step > 0; step >>= 1)
            {
                __syncthreads();
                for (int i = tid; i < size; i += TOP_THREADS)
                {
                    const int j = i ^ step;
                    if (j > i && ((list[i] < list[j]) == ((i & span) == 0)))
                    {
                        const unsigned long long t = list[i];
                        list[i] = list[j];
                        list[j] = t;
                    }
                }
            }
        }
        __syncthreads();
        for (int j = tid; j < a.k; j += TOP_THREADS)
        {
            const int v = j < kept ? static_cast<int>(~static_cast<unsigned int>(list[j])) : -1;
            a.indices[row * a.k + j] = v;
            static_cast<T *>(a.values)[row * a.k + j] = v >= 0 ? z[v] : from_float<T>(-INFINITY);
        }
        __syncthreads();
    }
}

template <typename T>
static int launch_top(const TopArgs &a, int sms, cudaStream_t stream)
{
    const long long most = 4ll * sms;
    const int grid = static_cast<int>(a.rows < most ? a.rows : most);
    top_rows_kernel<T><<<grid, TOP_THREADS, 0, stream>>>(a);
    B200AMP_LAUNCHED();
    return B200AMP_OK;
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
    if (vocab > 1 << 20)
    {
        set_error("top_logits: a vocabulary of %d is beyond the maximum of %d", vocab, 1 << 20);
        return B200AMP_ERR_LIMIT;
    }
    const int sms = sm_count();
    if (sms <= 0)
    {
        return B200AMP_ERR_CUDA;
    }
    if (rows == 0)
    {
        return B200AMP_OK;
    }
    const TopArgs a = {logits, ld, rows, vocab, k, temperature, values, indices, lse};
    switch (dtype)
    {
    case B200AMP_F16:
        return launch_top<__half>(a, sms, as_stream(s));
    case B200AMP_BF16:
        return launch_top<__nv_bfloat16>(a, sms, as_stream(s));
    default:
        return launch_top<float>(a, sms, as_stream(s));
    }
}
