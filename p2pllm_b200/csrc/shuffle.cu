// Routed experts, the tokens' way there and back, without a word to the host (p2p_moe_route reads its counts back):
//
//   p2p_moe_sort     the (token, slot) pairs with an expert sorted by expert, pairs of one expert in their own order
//   p2p_moe_spread   out[where[t K + j]] = x[t]: the tokens' rows in that order (and the gradient's way back from sums)
//   p2p_moe_sum      out[t] = sum_j w[t, j] y[where[t K + j]], fp32 in slot order (w = 1: the gradient of the spread)
//   p2p_moe_sum_back dy[where[t K + j]] = w[t, j] dout[t] and dw[t, j] = <dout[t], y[where[t K + j]]>
//
// The row kernels are bound by the memory: 8192 tokens x 8 rows of 4 KB: spread 302 MB in 49 us (6.1 TB/s), sum the same in
// 55 us (5.5 TB/s), its gradient 604 MB in 94 us (6.4 TB/s). The sort of those 65536 pairs is bound by latency: 17 us.
//
// Rows of an order are `pairs` long whatever the routing: behind the last routed pair order is -1 and rows are zero.
// p2p/compact.py:241-256 leaves all of this to SGLang's fused MoE.
#include "sm100.cuh"

namespace p2p {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortExperts = 1024;
constexpr int kClusterCtas = 8;
constexpr int kKept = 8;
constexpr int64_t kOneCtaPairs = 8192;

struct SortParams {
    const void* ids;
    int n, experts;
    int32_t *order, *where, *offsets;
    int32_t *items, *n_items;
    int max_items, item_tokens;
};

// A stable counting sort by one CTA, or by a cluster of 8 above 8192 pairs (each then counts and places an eighth).
// Every warp owns a run of consecutive pairs: it counts them into a histogram of its own, 32 at a step (lanes with the
// same expert find each other by one ballot a bit of the expert -- match.any takes a turn for every expert among them --
// so no atomics and no order to lose), the histograms turn into first places
// by sums over warps, CTAs (through distributed shared memory) and experts, and the warp walks its run again and places
// the pairs.
template <typename I>
__global__ void __launch_bounds__(kSortThreads) sort_kernel(const SortParams p) {
    extern __shared__ int sm[];
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, E = p.experts;
    int* hist = sm;                                  // [warps][E]
    int* mine = hist + warps * E;                    // [E]: this CTA's pairs of each expert, which the others read
    int* base = mine + E;                            // [E]: the place of this CTA's first pair of each expert
    __shared__ int s_sum[2][32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int cta = blockIdx.x, ctas = gridDim.x;    // the grid is one cluster
    for (int i = threadIdx.x; i < warps * E; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int runs = warps * ctas, per = ((p.n + runs - 1) / runs + 31) / 32 * 32;
    const int begin = min(p.n, (cta * warps + warp) * per), end = min(p.n, begin + per);
    const I* ids = reinterpret_cast<const I*>(p.ids);
    const unsigned below = (1u << lane) - 1u;
    int* h = hist + warp * E;
    auto expert_at = [&](int i) -> int {             // -1: routed nowhere
        const int64_t e = i < end ? (int64_t)__ldcg(ids + i) : -1;
        return e >= 0 && e < E ? (int)e : -1;
    };
    // Up to kKept steps of 32 pairs are kept in registers between the two walks, and loaded all at once.
    int kept[kKept];
    unsigned peers[kKept];
#pragma unroll
    for (int s = 0; s < kKept; ++s) kept[s] = expert_at(begin + s * 32 + lane);
    const int bits = 32 - __clz(E);                  // of 0..E, E standing for nowhere
    auto same_expert = [&](int e) -> unsigned {
        const unsigned key = e >= 0 ? (unsigned)e : (unsigned)E;
        unsigned same = 0xffffffffu;
        for (int b = 0; b < bits; ++b) {
            const bool one = (key >> b) & 1u;
            const unsigned ones = __ballot_sync(0xffffffffu, one);
            same &= one ? ones : ~ones;
        }
        return same;
    };
    auto count = [&](int e, unsigned same) {
        if (e >= 0 && (same & below) == 0) h[e] += __popc(same);
        __syncwarp();
    };
#pragma unroll
    for (int s = 0; s < kKept; ++s) {
        if (begin + s * 32 < end) {
            peers[s] = same_expert(kept[s]);
            count(kept[s], peers[s]);
        }
    }
    for (int i0 = begin + kKept * 32; i0 < end; i0 += 32) {
        const int e = expert_at(i0 + lane);
        count(e, same_expert(e));
    }
    __syncthreads();
    if (threadIdx.x < E) {                                           // first places within this CTA; E <= blockDim
        int run = 0;
        for (int w0 = 0; w0 < warps; w0 += 8) {
            int c[8];
#pragma unroll
            for (int w = 0; w < 8; ++w) c[w] = w0 + w < warps ? hist[(w0 + w) * E + threadIdx.x] : 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                if (w0 + w < warps) hist[(w0 + w) * E + threadIdx.x] = run;
                run += c[w];
            }
        }
        mine[threadIdx.x] = run;
    }
    if (ctas > 1) sm100::cluster_sync_all(); else __syncthreads();
    // totals over the CTAs, and exclusive sums over the experts: of the pairs and of the items
    int all = 0, before = 0;
    if (threadIdx.x < E) {
        if (ctas > 1) {
            const uint32_t at = sm100::smem_u32(mine + threadIdx.x);
            int v[kClusterCtas];
#pragma unroll
            for (int c = 0; c < kClusterCtas; ++c)
                asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v[c]) : "r"(sm100::cluster_addr(at, c)) : "memory");
#pragma unroll
            for (int c = 0; c < kClusterCtas; ++c) {
                if (c < cta) before += v[c];
                all += v[c];
            }
        } else {
            all = mine[threadIdx.x];
        }
    }
    const int n_it = (all + p.item_tokens - 1) / p.item_tokens;
    int pairs = all, items = n_it;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, pairs, o), b = __shfl_up_sync(0xffffffffu, items, o);
        if (lane >= o) { pairs += a; items += b; }
    }
    if (lane == 31) { s_sum[0][warp] = pairs; s_sum[1][warp] = items; }
    __syncthreads();
    int pair_base = 0, item_base = 0, pair_total = 0, item_total = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) { pair_base += s_sum[0][w]; item_base += s_sum[1][w]; }
        pair_total += s_sum[0][w];
        item_total += s_sum[1][w];
    }
    const int start = pair_base + pairs - all, first_item = item_base + items - n_it;
    if (threadIdx.x < E) {
        base[threadIdx.x] = start + before;
        if (cta == 0) {
            p.offsets[threadIdx.x] = start;
            for (int k = 0; k < n_it && first_item + k < p.max_items; ++k)
                reinterpret_cast<int4*>(p.items)[first_item + k] =
                    make_int4(threadIdx.x, start + k * p.item_tokens, min(p.item_tokens, all - k * p.item_tokens), 0);
        }
    }
    if (cta == 0 && threadIdx.x == 0) {
        p.offsets[E] = pair_total;
        *p.n_items = min(item_total, p.max_items);
    }
    __syncthreads();
    auto place = [&](int i, int e, unsigned same) {
        const int at = e >= 0 ? h[e] : 0;
        __syncwarp();
        if (e >= 0 && (same & below) == 0) h[e] = at + __popc(same);
        __syncwarp();
        if (i < end) {
            const int to = e >= 0 ? base[e] + at + __popc(same & below) : -1;
            p.where[i] = to;
            if (e >= 0) p.order[to] = i;
        }
    };
#pragma unroll
    for (int s = 0; s < kKept; ++s)
        if (begin + s * 32 < end) place(begin + s * 32 + lane, kept[s], peers[s]);
    for (int i0 = begin + kKept * 32; i0 < end; i0 += 32) {
        const int e = expert_at(i0 + lane);
        place(i0 + lane, e, same_expert(e));
    }
    for (int i = pair_total + cta * blockDim.x + threadIdx.x; i < p.n; i += ctas * blockDim.x) p.order[i] = -1;
    if (ctas > 1) sm100::cluster_sync_all();         // nobody leaves while its counts may still be read
}

// --- rows there and back: vectors of N elements of T, 16 bytes where every row allows it, else one element -------------

// 16-bit values stay in pairs: kept one by one they took the sum's kernel past its registers.
template <typename T, int N> struct alignas(sizeof(T) * N) Vec {
    using Word = std::conditional_t<N == 1, T, uint32_t>;
    static constexpr int kPer = sizeof(Word) / sizeof(T);
    Word v[N / kPer];
    __device__ __forceinline__ void to(float (&f)[N]) const {
        if constexpr (kPer == 2) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const float2 u = unpack2<T>(v[i]);
                f[2 * i] = u.x;
                f[2 * i + 1] = u.y;
            }
        } else if constexpr (N == 1) {
            f[0] = to_f32(v[0]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = __uint_as_float(v[i]);
        }
    }
    __device__ __forceinline__ void from(const float (&f)[N]) {
        if constexpr (kPer == 2) {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) {
                const T pair[2] = {from_f32<T>(f[2 * i]), from_f32<T>(f[2 * i + 1])};
                uint16_t bits[2];
                memcpy(bits, pair, 4);
                v[i] = (uint32_t)bits[0] | (uint32_t)bits[1] << 16;
            }
        } else if constexpr (N == 1) {
            v[0] = from_f32<T>(f[0]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = __float_as_uint(f[i]);
        }
    }
};

struct RowParams {
    const void *x, *y;                               // [tokens, hidden] (x, or dout) and [pairs, hidden]
    void* out;
    int64_t ldx, ldy, ldo;
    const int32_t *where, *last;                     // last: the number of routed pairs
    const void* w;                                   // null: 1
    void* dw;
    int w_dtype, tokens, k, vecs;                    // vectors a row
};

__device__ __forceinline__ float load_weight(const void* w, int dtype, int64_t i) {
    if (dtype == P2P_F32) return reinterpret_cast<const float*>(w)[i];
    if (dtype == P2P_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
    return __half2float(reinterpret_cast<const __half*>(w)[i]);
}
__device__ __forceinline__ void store_weight(void* w, int dtype, int64_t i, float v) {
    if (dtype == P2P_F32) reinterpret_cast<float*>(w)[i] = v;
    else if (dtype == P2P_BF16) reinterpret_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(w)[i] = __float2half_rn(v);
}

template <typename T, int N> __device__ __forceinline__ Vec<T, N> load_vec(const void* p, int64_t at) {
    return *reinterpret_cast<const Vec<T, N>*>(reinterpret_cast<const T*>(p) + at);
}
template <typename T, int N> __device__ __forceinline__ void store_vec(void* p, int64_t at, const Vec<T, N>& v) {
    *reinterpret_cast<Vec<T, N>*>(reinterpret_cast<T*>(p) + at) = v;
}

// Zeroes the rows of p.out behind the last routed pair; the whole grid takes part.
template <typename T, int N> __device__ __forceinline__ void zero_behind(const RowParams& p) {
    const int threads = blockDim.x * blockDim.y, last = *p.last;
    const int64_t pairs = (int64_t)p.tokens * p.k, n = (pairs - last) * p.vecs;
    const float none[N] = {};
    Vec<T, N> zero;
    zero.from(none);
    for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * threads + threadIdx.y * blockDim.x + threadIdx.x;
         i < n; i += (int64_t)gridDim.x * gridDim.y * threads)
        store_vec<T, N>(p.out, (last + i / p.vecs) * p.ldo + i % p.vecs * N, zero);
}

constexpr int kBatch = 4;                            // slots whose rows a thread holds at a time: eight cost half the blocks
                                                     // an SM (8192 x 8 rows of 4 KB: gradient 128 us, four 98)
constexpr int kRowThreads = 256;

// A token's places (-1: nowhere) and weights, a slot a lane: one load a warp for 32 slots, dealt out by shuffles. (A load a
// batch puts more trips to memory in a row. With it and the pairs of Vec, 8192 x 8 rows of 4 KB: weighted sum 68 us to
// 55, gradient 98 to 94.)
template <int N> struct Slots { int at[N]; float w[N]; };
struct LaneSlots {
    int at;
    float w;
    // of slots j0 / 32 * 32.. of token t, when j0 is the first of 32
    __device__ __forceinline__ void load(const RowParams& p, int64_t t, int j0, bool live) {
        if (j0 % 32) return;
        const int j = j0 + (threadIdx.x & 31);
        const bool in = live && j < p.k;
        const int64_t i = t * p.k + j;
        at = in ? __ldcg(p.where + i) : -1;
        w = in && p.w ? load_weight(p.w, p.w_dtype, i) : 1.f;
    }
    template <int N> __device__ __forceinline__ Slots<N> batch(int j0) const {
        Slots<N> s;
#pragma unroll
        for (int b = 0; b < N; ++b) {
            s.at[b] = __shfl_sync(0xffffffffu, at, (j0 + b) & 31);
            s.w[b] = __shfl_sync(0xffffffffu, w, (j0 + b) & 31);
        }
        return s;
    }
};

template <typename T, int N> __global__ void __launch_bounds__(kRowThreads) spread_kernel(const RowParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    LaneSlots mine;
    for (int j0 = 0; j0 < p.k && t < p.tokens; j0 += kBatch) {       // a warp's rows are one token's
        mine.load(p, t, j0, true);
        const Slots<kBatch> s = mine.batch<kBatch>(j0);
        for (int v = blockIdx.y * blockDim.x + threadIdx.x; v < p.vecs; v += gridDim.y * blockDim.x) {
            const Vec<T, N> val = load_vec<T, N>(p.x, t * p.ldx + (int64_t)v * N);
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (s.at[b] >= 0) store_vec<T, N>(p.out, s.at[b] * p.ldo + (int64_t)v * N, val);
        }
    }
    zero_behind<T, N>(p);
}

// A thread's loads of a batch go out together: a slot routed nowhere reads the batch's row 0 and drops it.
template <typename T, int N> __global__ void __launch_bounds__(kRowThreads, 4) sum_kernel(const RowParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= p.tokens) return;
    const int lane = threadIdx.x & 31;
    LaneSlots mine;
    mine.load(p, t, 0, true);
    // whole warps go round, so that all lanes of one are there when it loads its slots
    for (int v0 = blockIdx.y * blockDim.x + threadIdx.x - lane; v0 < p.vecs; v0 += gridDim.y * blockDim.x) {
        const bool on = v0 + lane < p.vecs;
        const int64_t col = (int64_t)(on ? v0 + lane : 0) * N;
        float acc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
        for (int j0 = 0; j0 < p.k; j0 += kBatch) {
            if (p.k > 32) mine.load(p, t, j0, true);
            const Slots<kBatch> s = mine.batch<kBatch>(j0);
            Vec<T, N> rows[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (j0 + b < p.k) rows[b] = load_vec<T, N>(p.y, max(s.at[b], 0) * p.ldy + col);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (s.at[b] < 0) continue;
                float row[N];
                rows[b].to(row);
#pragma unroll
                for (int i = 0; i < N; ++i) acc[i] = fmaf(s.w[b], row[i], acc[i]);
            }
        }
        if (!on) continue;
        Vec<T, N> o;
        o.from(acc);
        store_vec<T, N>(p.out, t * p.ldo + col, o);
    }
}

// blockDim.x is whole warps: a token's dots are summed by shuffles, then over its warps in warp order.
template <typename T, int N> __global__ void __launch_bounds__(kRowThreads, 4) sum_back_kernel(const RowParams p) {
    __shared__ float s_dot[kRowThreads / 32][kBatch];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int lane = threadIdx.x & 31, row_warps = blockDim.x >> 5, row_warp = threadIdx.x >> 5;
    const bool live = t < p.tokens;
    LaneSlots mine;
    for (int j0 = 0; j0 < p.k; j0 += kBatch) {
        mine.load(p, t, j0, live);
        const Slots<kBatch> s = mine.batch<kBatch>(j0);
        float dot[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) dot[b] = 0.f;
        for (int v = threadIdx.x; live && v < p.vecs; v += blockDim.x) {
            float grad[N];
            load_vec<T, N>(p.x, t * p.ldx + (int64_t)v * N).to(grad);
            Vec<T, N> rows[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b)
                if (j0 + b < p.k) rows[b] = load_vec<T, N>(p.y, max(s.at[b], 0) * p.ldy + (int64_t)v * N);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (s.at[b] < 0) continue;
                float row[N], scaled[N];
                rows[b].to(row);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    dot[b] = fmaf(grad[i], row[i], dot[b]);
                    scaled[i] = s.w[b] * grad[i];
                }
                Vec<T, N> o;
                o.from(scaled);
                store_vec<T, N>(p.out, s.at[b] * p.ldo + (int64_t)v * N, o);
            }
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
#pragma unroll
            for (int o = 16; o; o >>= 1) dot[b] += __shfl_xor_sync(0xffffffffu, dot[b], o);
            if (lane == 0) s_dot[threadIdx.y * row_warps + row_warp][b] = dot[b];
        }
        __syncthreads();
        const int b = threadIdx.x;
        if (live && b < kBatch && j0 + b < p.k) {
            float sum = 0.f;
            for (int r = 0; r < row_warps; ++r) sum += s_dot[threadIdx.y * row_warps + r][b];
            store_weight(p.dw, p.w_dtype, t * p.k + j0 + b, sum);
        }
        __syncthreads();
    }
    zero_behind<T, N>(p);
}

enum RowOp { kSpread, kSum, kSumBack };

template <typename T, int N> int launch_rows(RowOp op, RowParams& p, int64_t hidden, cudaStream_t st, const char* what) {
    p.vecs = (int)(hidden / N);
    int bx = 32;
    while (bx < kRowThreads && bx < p.vecs) bx *= 2;
    const int by = kRowThreads / bx;
    const int64_t gx = ((int64_t)p.tokens + by - 1) / by;
    // few tokens: a row's vectors are dealt over blocks too (the backward sum reduces over a row in one block)
    int64_t gy = 1;
    if (op != kSumBack && gx < sm_count()) gy = (p.vecs + bx - 1) / bx;
    if (gy > 65535) gy = 65535;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)gx, (unsigned)gy);
    cfg.blockDim = dim3((unsigned)bx, (unsigned)by);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, op == kSpread ? spread_kernel<T, N> : op == kSum ? sum_kernel<T, N> : sum_back_kernel<T, N>,
                       (const RowParams)p);
    return launch_status(what);
}

int run_rows(RowOp op, RowParams& p, int dtype, int64_t hidden, cudaStream_t st, const char* what) {
    const int size = dtype_size(dtype), n = 16 / size;
    // strides that no access uses (of null pointers) are 0
    const bool vec = hidden % n == 0 && p.ldx % n == 0 && p.ldy % n == 0 && p.ldo % n == 0 && aligned16(p.x) &&
                     aligned16(p.y) && aligned16(p.out);
    switch (dtype) {
        case P2P_BF16: return vec ? launch_rows<__nv_bfloat16, 8>(op, p, hidden, st, what)
                                  : launch_rows<__nv_bfloat16, 1>(op, p, hidden, st, what);
        case P2P_F16: return vec ? launch_rows<__half, 8>(op, p, hidden, st, what)
                                 : launch_rows<__half, 1>(op, p, hidden, st, what);
        default: return vec ? launch_rows<float, 4>(op, p, hidden, st, what)
                            : launch_rows<float, 1>(op, p, hidden, st, what);
    }
}

int check_rows(const char* what, int dtype, int64_t tokens, int k, int64_t hidden) {
    if (!dtype_ok(dtype)) return fail(P2P_EUNSUPPORTED, "%s: bf16, f16 or f32", what);
    // 2^30 columns: a column's number plus one step of the whole grid stays below 2^31
    P2P_REQUIRE(tokens >= 0 && k >= 1 && hidden >= 1 && hidden <= 0x40000000 && tokens <= 0x7fffffff / k,
                "%s: bad shape (%lld tokens, %d slots, %lld columns)", what, (long long)tokens, k, (long long)hidden);
    return P2P_OK;
}

}  // namespace
}  // namespace p2p

using namespace p2p;

extern "C" int p2p_moe_sort(const void* ids, int ids_bytes, int64_t n_pairs, int experts, int32_t* order,
                            int32_t* where, int32_t* offsets, int32_t* items, int64_t max_items, int item_tokens,
                            int32_t* n_items, void* stream) {
    P2P_REQUIRE(n_pairs >= 0 && n_pairs <= 0x7fffffff - 65536 && experts >= 1 && item_tokens >= 1 && item_tokens <= 65536,
                "p2p_moe_sort: %lld pairs, %d experts, items of %d", (long long)n_pairs, experts, item_tokens);
    if (experts > kSortExperts)
        return fail(P2P_EUNSUPPORTED, "p2p_moe_sort: %d experts, at most %d", experts, kSortExperts);
    P2P_REQUIRE(ids_bytes == 4 || ids_bytes == 8, "p2p_moe_sort: ids of %d bytes, not 4 or 8", ids_bytes);
    P2P_REQUIRE(offsets && n_items && items && (n_pairs == 0 || (ids && order && where)), "p2p_moe_sort: null pointer");
    P2P_REQUIRE(aligned16(items), "p2p_moe_sort: items must start on a 16-byte boundary");
    const int64_t full = (n_pairs + item_tokens - 1) / item_tokens;
    const int64_t need = n_pairs < full + experts ? n_pairs : full + experts;
    P2P_REQUIRE(max_items >= need && max_items <= 0x7fffffff, "p2p_moe_sort: room for %lld items, up to %lld needed",
                (long long)max_items, (long long)need);
    SortParams p = {ids, (int)n_pairs, experts, order, where, offsets, items, n_items, (int)max_items, item_tokens};
    const int ctas = n_pairs > kOneCtaPairs ? kClusterCtas : 1;
    // threads: one an expert at least, 8 pairs a thread at most until the block is full
    int threads = (experts + 31) / 32 * 32;
    const int64_t want = (n_pairs / ctas / 8 + 31) / 32 * 32;
    if (threads < want) threads = want < kSortThreads ? (int)want : kSortThreads;
    // one histogram a warp: fewer warps where the experts are many
    const size_t smem = ((size_t)(threads / 32) + 2) * experts * sizeof(int);
    const void* fn = ids_bytes == 4 ? (const void*)sort_kernel<int32_t> : (const void*)sort_kernel<int64_t>;
    if (int e = allow_smem(fn, (int)smem, "p2p_moe_sort")) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = as_stream(stream);
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, ids_bytes == 4 ? sort_kernel<int32_t> : sort_kernel<int64_t>, (const SortParams)p);
    return launch_status("p2p_moe_sort");
}

extern "C" int p2p_moe_spread(const void* x, int dtype, int64_t tokens, int k, int64_t hidden, int64_t ldx,
                              const int32_t* where, const int32_t* routed, void* out, int64_t ldo, void* stream) {
    if (int e = check_rows("p2p_moe_spread", dtype, tokens, k, hidden)) return e;
    if (tokens == 0) return P2P_OK;
    P2P_REQUIRE(x && where && routed && out && ldx >= hidden && ldo >= hidden, "p2p_moe_spread: null pointer or stride");
    RowParams p = {x, nullptr, out, ldx, 0, ldo, where, routed, nullptr, nullptr, P2P_F32, (int)tokens, k, 0};
    return run_rows(kSpread, p, dtype, hidden, as_stream(stream), "p2p_moe_spread");
}

extern "C" int p2p_moe_sum(const void* y, int dtype, int64_t tokens, int k, int64_t hidden, int64_t ldy,
                           const int32_t* where, const void* weights, int weights_dtype, void* out, int64_t ldo,
                           void* stream) {
    if (int e = check_rows("p2p_moe_sum", dtype, tokens, k, hidden)) return e;
    if (tokens == 0) return P2P_OK;
    P2P_REQUIRE(y && where && out && ldy >= hidden && ldo >= hidden && (!weights || dtype_ok(weights_dtype)),
                "p2p_moe_sum: null pointer, stride or weights' type");
    RowParams p = {nullptr, y, out, 0, ldy, ldo, where, nullptr, weights, nullptr, weights_dtype, (int)tokens, k, 0};
    return run_rows(kSum, p, dtype, hidden, as_stream(stream), "p2p_moe_sum");
}

extern "C" int p2p_moe_sum_back(const void* dout, const void* y, int dtype, int64_t tokens, int k, int64_t hidden,
                                int64_t ldd, int64_t ldy, const int32_t* where, const int32_t* routed,
                                const void* weights, int weights_dtype, void* dy, int64_t lddy, void* dweights,
                                void* stream) {
    if (int e = check_rows("p2p_moe_sum_back", dtype, tokens, k, hidden)) return e;
    if (tokens == 0) return P2P_OK;
    P2P_REQUIRE(dout && y && where && routed && weights && dy && dweights && dtype_ok(weights_dtype),
                "p2p_moe_sum_back: null pointer or weights' type");
    P2P_REQUIRE(ldd >= hidden && ldy >= hidden && lddy >= hidden, "p2p_moe_sum_back: a row stride below the row");
    RowParams p = {dout, y, dy, ldd, ldy, lddy, where, routed, weights, dweights, weights_dtype, (int)tokens, k, 0};
    return run_rows(kSumBack, p, dtype, hidden, as_stream(stream), "p2p_moe_sum_back");
}
