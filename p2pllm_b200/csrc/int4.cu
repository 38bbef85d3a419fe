// (2d) Products with 4-bit weights and group scales: y[t, r] = sum_c (code[r, c] - zero[r, g]) scale[r, g] x[t, c],
// g = c / group, on the layout of int4.cuh; its builder, the quantiser, and the same product for routed experts.
// No counterpart in the reference (p2p/compact.py stores a replica's weights pruned, 16 bits a kept one); it stands
// beside p2p_spmm_tc as another storage of a replica's projections.
//
//   p2p_int4_quantize   codes, scales and zero points of dense rows, each group of columns over its own range
//   p2p_int4_expand     the dense rows that codes stand for
//   p2p_int4_layout     codes and scales, row after row, into the layout
//   p2p_int4_mm         y = x W^T
//   p2p_int4_grouped    the same for the rows of one expert after the other, rows gathered by token or in place, with
//                       silu(gate) * up applied on the way out of a gated module
#include <atomic>

#include "int4.cuh"
#include "int4_run.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace p2p {
namespace {

// One warp a (row, group): the group's range by shuffles, then its codes. All arithmetic on the scale is in 64 bits
// before its one rounding to T, and a quotient of two 16-bit floats that is not a tie is further from it than fp32's
// rounding, so the codes are those of exact arithmetic.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T* __restrict__ w, int64_t ldw, int64_t rows, int cols,
                                                       int group, uint8_t* __restrict__ codes,
                                                       T* __restrict__ scales, uint8_t* __restrict__ zeros) {
    const int lane = threadIdx.x & 31;
    const int64_t groups = q4::div_up(cols, group), n_bytes = q4::div_up(cols, 2);
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x >> 5);
    for (int64_t i = blockIdx.x * (int64_t)(blockDim.x >> 5) + (threadIdx.x >> 5); i < rows * groups; i += warps) {
        const int64_t row = i / groups, g = i % groups;
        const T* p = w + row * ldw;
        float v[4];                                    // columns 2 lane, 2 lane + 1, and the same 64 further on
        float lo = 0.f, hi = 0.f;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int in = 2 * lane + (k & 1) + 64 * (k >> 1);
            const int64_t c = g * group + in;
            v[k] = in < group && c < cols ? to_f32(p[c]) : 0.f;
            lo = fminf(lo, v[k]);
            hi = fmaxf(hi, v[k]);
            bad |= v[k] != v[k];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        }
        bad = __any_sync(0xffffffffu, bad);
        const double span = zeros ? ((double)hi - (double)lo) / 15.0 : fmax((double)hi, -(double)lo) / 7.0;
        T s16 = from_f32<T>((float)span);
        if (bad) s16 = from_f32<T>(__int_as_float(0x7fffffff));   // a NaN weight makes its whole group NaN
        const float s = to_f32(s16);
        float z = 8.f;
        if (zeros) z = s > 0.f ? fminf(fmaxf(rintf(-lo / s), 0.f), 15.f) : 0.f;
        if (lane == 0) {
            scales[i] = s16;
            if (zeros) zeros[i] = (uint8_t)z;
        }
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
            const int in = 2 * lane + 32 * k;
            const int64_t c = g * group + in;
            if (in < group && c < cols) {
                int q[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float f = s > 0.f ? rintf(v[k + h] / s) + z : z;
                    q[h] = (int)fminf(fmaxf(f, 0.f), 15.f);
                }
                if (c + 1 >= cols) q[1] = 0;
                codes[row * n_bytes + c / 2] = (uint8_t)(q[0] | (q[1] << 4));
            }
        }
    }
}

// One thread two columns: (code - zero) scale, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) expand_kernel(const uint8_t* __restrict__ codes, const T* __restrict__ scales,
                                                     const uint8_t* __restrict__ zeros, int64_t rows, int cols,
                                                     int group, T* __restrict__ dense) {
    const int64_t n_bytes = q4::div_up(cols, 2), groups = q4::div_up(cols, group);
    const int64_t stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < rows * n_bytes; i += stride) {
        const int64_t row = i / n_bytes, c = i % n_bytes * 2, at = row * groups + c / group;
        const float s = to_f32(scales[at]), z = zeros ? (float)(zeros[at] & 15) : 8.f;
        dense[row * cols + c] = from_f32<T>(((float)(codes[i] & 15) - z) * s);
        if (c + 1 < cols) dense[row * cols + c + 1] = from_f32<T>(((float)(codes[i] >> 4) - z) * s);
    }
}

// One thread a 32-bit word of the layout: eight codes, four zero points or two scales.
__global__ void __launch_bounds__(256) layout_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scales,
                                                     const uint8_t* __restrict__ zeros, int64_t experts, int64_t rows,
                                                     int cols, int group, int gated, uint32_t* __restrict__ out) {
    const int64_t tiles = q4::row_tiles(rows, gated), units = q4::div_up(cols, q4::kUnitCols);
    const int64_t groups = q4::div_up(cols, group), n_bytes = q4::div_up(cols, 2), half = rows / 2;
    const int subs = q4::kUnitCols / group, zero_words = q4::unit_zero_bytes(group, zeros != nullptr) / 4;
    const int code_words = q4::kCodeBytes / 4, record = q4::unit_bytes(group, zeros != nullptr) / 4;
    // the source row of row `in` of row block rb, or -1 for padding
    auto source = [&](int64_t rb, int in) -> int64_t {
        const int64_t r = (gated ? rb / 2 : rb) * q4::kRows + in;
        if (gated) return r < half ? r + (rb & 1) * half : -1;
        return r < rows ? r : -1;
    };
    const int64_t n = experts * tiles * units * record, stride = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += stride) {
        const int64_t rec = i / record, unit = rec % units, tile = rec / units % tiles, e = rec / units / tiles;
        int w = (int)(i % record);
        uint32_t v = 0;
        if (w < code_words) {
            const int r = w & 3, lane = (w >> 2) & 31, kb = (w >> 7) & 1, blk = w >> 8;
            const int64_t k = unit * q4::kUnitCols + kb * q4::kCols + 16 * r + 4 * (lane & 3);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t row = source(tile * q4::kTileBlocks + blk, (lane >> 2) + 8 * h);
                if (row < 0) continue;
                const uint8_t* p = codes + (e * rows + row) * n_bytes;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (k + c >= cols) continue;
                    const uint32_t q = (p[(k + c) >> 1] >> (4 * (c & 1))) & 15u;
                    v |= q << (4 * (2 * h + (c >> 1)) + 16 * (c & 1));
                }
            }
        } else {
            w -= code_words;
            const bool is_zero = w < zero_words;
            if (!is_zero) w -= zero_words;
            const int per = is_zero ? 4 : 2;             // values a word; 16 values a row block
            for (int c = 0; c < per; ++c) {
                const int at = w * per + c, in = ((at >> 1) & 7) + 8 * (at & 1), blk = (at >> 4) & 7;
                const int64_t g = unit * subs + (at >> 7), row = source(tile * q4::kTileBlocks + blk, in);
                if (row < 0 || g >= groups) continue;
                const int64_t from = (e * rows + row) * groups + g;
                v |= (is_zero ? (uint32_t)(zeros[from] & 15) : (uint32_t)scales[from]) << (c * (32 / per));
            }
        }
        out[i] = v;
    }
}

using namespace sm100;

constexpr int kComputeWarps = 8;                       // one a row block of the tile
constexpr int kSmallThreads = (kComputeWarps + 1) * 32;
constexpr int kMaxSlots = 8;
constexpr int kRowPad = 132;                           // floats a token of the partial tile: 128 rows, padded

__device__ int g_small_error;            // site of the first wait that gave up since the last reset (0: none)
__device__ unsigned g_small_failed_seq;  // sequence number of the last launch in which a wait gave up

struct SmallParams {
    const uint8_t* layout;
    int record, zeros, scales_at;       // bytes of a unit's record; whether it holds zero points; where its scales start
    int units, row_tiles, group_shift, gated;
    int tokens, n_max, out_rows;        // n_max: tokens of a tile, at most
    int splits;                         // > 0: CTAs of a cluster, each with its share of one row tile; 0: runs
    float* partial;                     // runs: [ctas][2][n_max][128], the row tiles a run shares with its neighbours
    int slots, half_bytes, x_at, x_sub; // ring: slots of two units (a tile's last may hold one), half_bytes each: record,
                                        // then two x boxes of x_sub bytes at x_at
    void* y;
    int64_t ldy;
    const int32_t* items;               // routed: {expert, first place, places, 0}
    const int32_t* n_items;
    const int32_t* order;               // routed: place -> pair, x's row being pair / topk; null: the place itself
    int topk;
    int hold;                           // a test's withheld slot: neither its weights nor its x are loaded; -1: none
    const int32_t* routed;              // not null: output rows from *routed to pairs become zero
    int64_t pairs;
    uint64_t wait_ns;
    unsigned seq;
};
// With the tensor map 288 bytes of arguments: at 296 the host's launch took 0.4 us longer (a call of one token 4.1 us to 4.5).
static_assert(sizeof(CUtensorMap) + sizeof(SmallParams) <= 288, "a launch of more arguments takes the host longer");

// d = a b + c: c is four registers of their own, so that a zero one costs nothing.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint2 b, const float (&c)[4]) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// A value at byte `at` of shared memory: plain loads, which the compiler may move about between two barriers.
template <typename V> __device__ __forceinline__ V lds(const uint8_t* smem, uint32_t at) {
    return *reinterpret_cast<const V*>(smem + at);
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ int token_of(int column) { return 2 * column - (column >> 2) * 7; }

// Row tile `id` of a launch: whose rows, which tokens.
struct SmallTile {
    const uint8_t* records;
    int rt, first, n;
};
__device__ __forceinline__ SmallTile small_tile(const SmallParams& p, int id) {
    SmallTile t;
    const int item = id / p.row_tiles;                   // 0 of a dense call
    t.rt = id - item * p.row_tiles;
    int64_t expert = 0;
    if (p.items) {
        const int4 it = __ldcg(reinterpret_cast<const int4*>(p.items) + item);
        expert = it.x;
        t.first = it.y;
        t.n = min(it.z, p.n_max);
    } else {
        t.first = 0;
        t.n = p.tokens;
    }
    t.records = p.layout + (expert * p.row_tiles + t.rt) * p.units * p.record;
    return t;
}
__device__ __forceinline__ int small_tiles(const SmallParams& p) { return (p.items ? *p.n_items : 1) * p.row_tiles; }
// Runs of a launch: no more than it has units (routed launches learn that here), so that none is empty.
__device__ __forceinline__ uint32_t small_runs(uint32_t units_all, uint32_t ctas) { return max(1u, min(ctas, units_all)); }

// y of a finished pair of sums (gated) or sum.
template <typename T> __device__ __forceinline__ T gate_up(float g, float u) { return from_f32<T>(g / (1.f + expf(-g)) * u); }

// A CTA takes 128 x 128 units of a row tile and up to 8 NT tokens: its share of one row tile, the CTAs of a cluster adding
// theirs up over distributed shared memory in column order, or (runs) a contiguous run of units across row tiles, the
// sums of those it shares with its neighbours going to int4_small_join_kernel. One warp streams records and x tiles into
// a ring of shared memory; warp w multiplies row blocks 2 (w % 4) and + 1 of column block w / 4 (two row blocks share a
// fragment of x, whose reads would else bind): the codes become exact small integers, m16n8k16 products add a group's
// columns in fp32, and the group's scale multiplies that sum on its way into the fp32 accumulators: no weight is ever
// rounded. G32: groups of 32 columns, two a column block (else one holds the block or more).
//
// Measured: 4096 x 14336 at one f16 token (groups of 64, zero points; 31.7 MB) 12.5 us a call, 2.5 TB/s: a launch and a
// ring's first fill are 6 us of it. 28672 x 4096 at 17 tokens (61 MB) 27 us, 2.3 TB/s: bound by the warps' issue, 41 % of
// the slots at 9 warps a CTA and 25 % occupancy (a word of eight codes takes 20 cycles of the logic pipe, and a product of
// 8 tokens 9.5 of the tensor pipe). 128 experts of 2048 x 768 (f16, groups of 32, zero points, 123 MB) on 272 x 8 tokens
// 73 us, 1.7 TB/s: the same, with four groups a unit to scale.
template <typename T, int NT, bool G32>
__global__ void __launch_bounds__(kSmallThreads, 2) int4_small_kernel(const __grid_constant__ CUtensorMap tmap_x,
                                                                      const __grid_constant__ SmallParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    float* red = reinterpret_cast<float*>(smem_raw + (base - raw) + p.slots * 2 * p.half_bytes);   // [8 NT][kRowPad]
    const uint32_t bars = smem_u32(red) + NT * 8 * kRowPad * 4;
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kMaxSlots + s); };
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const WaitCtl wc{&g_small_error, &g_small_failed_seq, p.wait_ns, p.seq};
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.slots; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), kComputeWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    // The items are the previous kernel's. Dense weights wait for nobody; x (its input) and y (whose old values it may
    // still read) for that kernel's end.
    if (p.items || warp < kComputeWarps) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tiles = small_tiles(p), units_all = tiles * p.units;
    const bool clustered = p.splits > 0;
    int u0 = 0, u1 = 0, rank = 0;
    if (clustered) {
        const int tile = blockIdx.x / p.splits;
        rank = blockIdx.x - tile * p.splits;
        if (tile < tiles) {
            u0 = tile * p.units + p.units * rank / p.splits;
            u1 = tile * p.units + p.units * (rank + 1) / p.splits;
        }
    } else {
        const uint32_t n = small_runs(units_all, gridDim.x);
        const q4::Runs runs(units_all, n, 1u);
        if (blockIdx.x < n) {
            u0 = (int)runs.begin(blockIdx.x);
            u1 = (int)runs.begin(blockIdx.x + 1);
        }
    }

    if (warp == kComputeWarps) {
        if (elect_one()) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_x)) : "memory");
            const int n_slots = p.slots;
            const uint32_t w_bytes = (uint32_t)p.record;
            bool ok = true;
            // Units k and, if there is one, k + 1 of a tile into slot `slot`.
            auto load_w = [&](int slot, const SmallTile& t, int k, int n) {
                const uint32_t x_rows = p.order ? (uint32_t)t.n : (uint32_t)(NT * 8);
                mbar_expect_tx(full(slot), n * (w_bytes + 2u * 128u * x_rows));
                for (int i = 0; i < n; ++i)
                    bulk_load(base + (2 * slot + i) * p.half_bytes, t.records + (int64_t)(k + i) * p.record, w_bytes,
                              full(slot));
            };
            int rows[8];                                             // x's rows of a tile that picks them, at most 8
            auto pick = [&](const SmallTile& t) {
                if (!p.order) return;
#pragma unroll
                for (int i = 0; i < 8; ++i) rows[i] = i < t.n ? __ldcg(p.order + t.first + i) : 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) rows[i] /= p.topk;
            };
            auto load_x = [&](int slot, const SmallTile& t, int k, int n) {
                for (int h = 0; h < n; ++h) {
                    const uint32_t at = base + (2 * slot + h) * p.half_bytes + p.x_at;
                    if (p.order) {                                   // a row at a time, from wherever its token lies
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if (i < t.n) {
                                tma_load_2d(at + i * 128, &tmap_x, (k + h) * 128, rows[i], full(slot));
                                tma_load_2d(at + p.x_sub + i * 128, &tmap_x, (k + h) * 128 + 64, rows[i], full(slot));
                            }
                        }
                    } else {
                        tma_load_2d(at, &tmap_x, (k + h) * 128, t.first, full(slot));
                        tma_load_2d(at + p.x_sub, &tmap_x, (k + h) * 128 + 64, t.first, full(slot));
                    }
                }
            };
            int slot = 0, used = 0;
            uint32_t ph = 0;
            int u = u0;
            if (!p.items) {
                // the ring's first fill: weights, then, once the previous kernel has ended, x
                const int fill = p.hold >= 0 ? min(p.hold, n_slots) : n_slots;
                for (int pass = 0; pass < 2; ++pass) {
                    int i = 0;
                    for (u = u0; u < u1 && i < fill;) {
                        const SmallTile t = small_tile(p, u / p.units);
                        const int kz = min(p.units, u % p.units + (u1 - u));
                        for (int k = u % p.units; k < kz && i < fill; ++i) {
                            const int n = min(2, kz - k);
                            if (pass == 0) load_w(i, t, k, n); else load_x(i, t, k, n);
                            k += n;
                            u += n;
                        }
                    }
                    used = i;
                    if (pass == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
                }
                slot = used == n_slots ? 0 : used;
                ph = used == n_slots ? 1u : 0u;
            }
            while (u < u1 && ok) {
                const SmallTile t = small_tile(p, u / p.units);
                const int kz = min(p.units, u % p.units + (u1 - u));
                pick(t);
                for (int k = u % p.units; k < kz;) {
                    if (!(ok = used != p.hold)) break;               // a test withholds this load
                    if (used >= n_slots && !(ok = wait_one(empty(slot), ph ^ 1u, 1, wc))) break;
                    const int n = min(2, kz - k);
                    load_w(slot, t, k, n);
                    load_x(slot, t, k, n);
                    k += n;
                    u += n;
                    ++used;
                    advance(slot, ph, 1, n_slots);
                }
            }
            // every copy issued must have landed before the CTA may exit: each slot's last one
            for (int i = max(0, used - n_slots); i < used; ++i)
                mbar_drain(full(i % n_slots), (uint32_t)((i / n_slots) & 1), 2, wc);
        }
        __syncwarp();
    } else {
        const int j = lane & 3, n = lane >> 2, blk = 2 * (warp & 3), half = warp >> 2;
        // this lane's columns 4 j.. of a 16-column step, in the 128-byte swizzle: 16-byte chunk 2 r + j / 2, XOR token.
        // Column n of a product is token 2 n, or 2 n - 7 for n >= 4: a half warp then reads tokens 0, 2, 4, 6 or 1, 3, 5,
        // 7, whose chunks fill all banks once (tokens 0 to 3 share half of them).
        const int tok = token_of(n);
        uint32_t x_off[4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
            x_off[r] = (uint32_t)(p.x_at + half * p.x_sub + tok * 128 + (j & 1) * 8 + (((2 * r + (j >> 1)) ^ tok) << 4));
        const uint32_t code_off = (uint32_t)((blk * 2 + half) * q4::kBlockBytes + lane * 16);
        // the column block's first group in its unit, this lane's pair of rows in it
        const int group0 = G32 ? 2 * half : p.group_shift == 6 ? half : 0, mine = group0 * 64 + blk * 8 + n;
        const uint32_t zero_off = (uint32_t)(q4::kCodeBytes + mine * 2), scale_off = (uint32_t)(p.scales_at + mine * 4);
        int slot = 0;
        uint32_t ph = 0, rec = 0;
        bool ok = true;
        const uint8_t* ring = smem_raw + (base - raw);
        q4::Codes<T> codes[2];
        codes[0].zeros(8u, 8u);
        codes[1].zeros(8u, 8u);
        float zero[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) zero[i] = __uint_as_float(q4::opaque(0u));
        for (int u = u0; u < u1;) {
            const SmallTile t = small_tile(p, u / p.units);
            const int ka = u % p.units, kz = min(p.units, ka + (u1 - u));
            float acc[2][NT][4];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int c = 0; c < NT; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[b][c][i] = 0.f;
            // LIVE: 8-token columns of this tile that hold a token (an item may be a few of the tile's)
            auto multiply = [&](auto live) {
                constexpr int LIVE = decltype(live)::value;
                for (int k = ka; k < kz; k += 2) {
                    // a warp that gave up multiplies nothing more, but keeps meeting the others at every row tile's end
                    if (!ok || !(ok = __all_sync(0xffffffffu, wait_one(full(slot), ph, 3, wc)))) break;
                    const uint8_t* at = ring + rec;
                    const int n_units = min(2, kz - k);
#pragma unroll 1
                    for (int unit = 0; unit < n_units; ++unit, at += p.half_bytes) {
                        uint32_t w[2][4];
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const uint4 c = lds<uint4>(at, code_off + b * 2 * q4::kBlockBytes);
                            w[b][0] = c.x; w[b][1] = c.y; w[b][2] = c.z; w[b][3] = c.w;
                        }
                        // the two row blocks' products alternate: each waits for its own last one only
                        float part[2][LIVE][4];
                        auto begin = [&](int b, int g) {
                            if (p.zeros) {
                                const uint32_t z = lds<uint16_t>(at, zero_off + b * 16 + g * 128);
                                codes[b].zeros(z & 15u, z >> 8);
                            }
                        };
                        auto end = [&](int b, int g) {
                            const float2 s = unpack2<T>(lds<uint32_t>(at, scale_off + b * 32 + g * 256));
#pragma unroll
                            for (int c = 0; c < LIVE; ++c) {
                                acc[b][c][0] = fmaf(s.x, part[b][c][0], acc[b][c][0]);
                                acc[b][c][1] = fmaf(s.x, part[b][c][1], acc[b][c][1]);
                                acc[b][c][2] = fmaf(s.y, part[b][c][2], acc[b][c][2]);
                                acc[b][c][3] = fmaf(s.y, part[b][c][3], acc[b][c][3]);
                            }
                        };
                        begin(0, 0);
                        begin(1, 0);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (G32 && r == 2) {
                                end(0, 0);
                                end(1, 0);
                                begin(0, 1);
                                begin(1, 1);
                            }
                            uint2 xf[LIVE];
#pragma unroll
                            for (int c = 0; c < LIVE; ++c) xf[c] = lds<uint2>(at, x_off[r] + c * 1024);
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                uint32_t a[4];
                                codes[b].expand(w[b][r], a);
#pragma unroll
                                for (int c = 0; c < LIVE; ++c) {
                                    mma16816<T>(part[b][c], a, xf[c], r == 0 || (G32 && r == 2) ? zero : part[b][c]);
                                }
                            }
                        }
                        end(0, G32 ? 1 : 0);
                        end(1, G32 ? 1 : 0);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(empty(slot));
                    rec += 2u * (uint32_t)p.half_bytes;
                    if (++slot == p.slots) {
                        slot = 0;
                        ph ^= 1u;
                        rec = 0;
                    }
                }
            };
            if (NT > 3 && t.n > 24) multiply(std::integral_constant<int, NT>());
            else if (NT > 2 && t.n > 16) multiply(std::integral_constant<int, NT < 3 ? NT : 3>());
            else if (NT > 1 && t.n > 8) multiply(std::integral_constant<int, NT < 2 ? NT : 2>());
            else multiply(std::integral_constant<int, 1>());
            // The row tile's sums [token][row]: the second column block's first, the first one's added to them.
#pragma unroll
            for (int h = 1; h >= 0; --h) {
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (half == h) {
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int c = 0; c < NT; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                float* at = red + (c * 8 + token_of(2 * j + (i & 1))) * kRowPad + (blk + b) * 16 + n +
                                            8 * (i >> 1);
                                *at = h ? acc[b][c][i] : acc[b][c][i] + *at;
                            }
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (!clustered) {
                T* y = reinterpret_cast<T*>(p.y);
                if (kz - ka < p.units) {                             // shared with the neighbouring run
                    float* part = p.partial + ((int64_t)blockIdx.x * 2 + (u == u0 ? 0 : 1)) * p.n_max * 128;
                    for (int i = threadIdx.x; i < t.n * 32; i += 256)
                        *reinterpret_cast<float4*>(part + i * 4) =
                            *reinterpret_cast<const float4*>(red + (i >> 5) * kRowPad + (i & 31) * 4);
                } else if (p.gated) {
                    for (int i = threadIdx.x; i < t.n * 64; i += 256) {
                        const int in = i & 63, at = (i >> 6) * kRowPad + in / 16 * 32 + in % 16, row = t.rt * 64 + in;
                        if (row < p.out_rows)
                            y[(int64_t)(t.first + (i >> 6)) * p.ldy + row] = gate_up<T>(red[at], red[at + 16]);
                    }
                } else {
                    for (int i = threadIdx.x; i < t.n * 128; i += 256) {
                        const int row = t.rt * 128 + (i & 127);
                        if (row < p.out_rows)
                            y[(int64_t)(t.first + (i >> 7)) * p.ldy + row] = from_f32<T>(red[(i >> 7) * kRowPad + (i & 127)]);
                    }
                }
            }
            u += kz - ka;
        }
    }
    if (clustered) {
        // Sum over the cluster, in column order; CTA `rank` finishes its share of the outputs.
        cluster_sync_all();
        if (u0 < u1) {
            const SmallTile t = small_tile(p, u0 / p.units);
            auto total = [&](int tok, int row) {
                const uint32_t at = smem_u32(red + tok * kRowPad + row);
                float v[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c < p.splits) v[c] = ld_cluster_f32(cluster_addr(at, c));
                float sum = v[0];
#pragma unroll
                for (int c = 1; c < 8; ++c)
                    if (c < p.splits) sum += v[c];
                return sum;
            };
            T* y = reinterpret_cast<T*>(p.y);
            const int width = p.gated ? 64 : 128;
            const int begin = t.n * width * rank / p.splits, end = t.n * width * (rank + 1) / p.splits;
            for (int i = begin + threadIdx.x; i < end; i += kSmallThreads) {
                const int tok = i / width, in = i % width, row = t.rt * width + in;
                if (row >= p.out_rows) continue;
                y[(int64_t)(t.first + tok) * p.ldy + row] =
                    p.gated ? gate_up<T>(total(tok, in / 16 * 32 + in % 16), total(tok, in / 16 * 32 + 16 + in % 16))
                            : from_f32<T>(total(tok, in));           // even row blocks are gates, odd ones their ups
            }
        }
        cluster_sync_all();                                          // nobody leaves while its tile may still be read
    }
    if (p.routed && warp < kComputeWarps) {                          // what lies behind the last pair
        for (int64_t r = *p.routed + blockIdx.x; r < p.pairs; r += gridDim.x)
            for (int c = threadIdx.x; c < p.out_rows; c += 256) reinterpret_cast<T*>(p.y)[r * p.ldy + c] = from_f32<T>(0.f);
    }
}

// Row tiles that several runs share: their fp32 partials added in run order. A block takes a row tile, a warp a token at
// a time, a thread four rows.
template <typename T>
__global__ void __launch_bounds__(256) int4_small_join_kernel(const __grid_constant__ SmallParams p, int ctas) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // Every block waits, those without work too: this kernel's end stands for the end of the one before.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tile = blockIdx.x, tiles = small_tiles(p);
    if (tile >= tiles) return;
    const uint32_t units_all = (uint32_t)(tiles * p.units), a = (uint32_t)(tile * p.units);
    const q4::Runs runs(units_all, small_runs(units_all, ctas), 1u);
    const uint32_t b0 = runs.of(a), b1 = runs.of(a + p.units - 1);
    if (b0 == b1) return;                                            // one run wrote y itself
    const SmallTile t = small_tile(p, tile);
    const int lane = threadIdx.x & 31;
    const int64_t size = (int64_t)p.n_max * 128;
    // the tile is run b0's last row tile, unless b0 begins with it, and every other run's first
    const float* part = p.partial + ((int64_t)b0 * 2 + (runs.begin(b0) >= a ? 0 : 1)) * size + lane * 4;
    const float* next = p.partial + (int64_t)(b0 + 1) * 2 * size + lane * 4;
    T* y = reinterpret_cast<T*>(p.y);
    for (int tok = threadIdx.x >> 5; tok < t.n; tok += 8) {
        float4 sum = __ldcg(reinterpret_cast<const float4*>(part + tok * 128));
#pragma unroll 4
        for (uint32_t b = b0 + 1; b <= b1; ++b) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(next + (int64_t)(b - b0 - 1) * 2 * size + tok * 128));
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        T* out = y + (int64_t)(t.first + tok) * p.ldy;
        const float mine[4] = {sum.x, sum.y, sum.z, sum.w};
        if (p.gated) {                                               // lanes 8 i .. + 3 hold gates, + 4 .. + 7 their ups
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float up = __shfl_xor_sync(0xffffffffu, mine[c], 4);
                const int row = t.rt * 64 + (lane >> 3) * 16 + (lane & 3) * 4 + c;
                if (!(lane & 4) && row < p.out_rows) out[row] = gate_up<T>(mine[c], up);
            }
        } else {
            const int row = t.rt * 128 + lane * 4;
            q4::Quad<T> q;
#pragma unroll
            for (int c = 0; c < 4; ++c) q.v[c] = from_f32<T>(mine[c]);
            if (row + 3 < p.out_rows && (reinterpret_cast<uintptr_t>(out + row) & 7u) == 0) {
                *reinterpret_cast<q4::Quad<T>*>(out + row) = q;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (row + c < p.out_rows) out[row + c] = q.v[c];
            }
        }
    }
}

unsigned next_seq() {
    static std::atomic<unsigned> counter{0};
    unsigned v = ++counter;
    while (v == 0) v = ++counter;
    return v;
}

// How a call of up to 32 tokens a tile is cut: shares of a cluster's CTAs where they are all resident at once, else
// runs. Two CTAs an SM: three leave 72 registers, and measured slower (28672 x 4096 at 16 tokens the same, 24 to 33 us at
// 24; 128 experts on 17 tokens 78 to 100 us).
struct SmallPlan {
    int nt, splits, ctas, slots, half_bytes, x_at, x_sub, smem;
    int64_t tiles;
    size_t workspace;
};

SmallPlan plan_small(const Int4Call& c) {
    SmallPlan pl = {};
    const bool routed = c.items != nullptr;
    const int64_t most = routed ? c.item_tokens : c.tokens;
    pl.nt = (int)q4::div_up(most, 8);
    pl.tiles = q4::row_tiles(c.rows, c.gated) * (routed ? c.max_items : 1);
    const int64_t units = q4::div_up(c.cols, q4::kUnitCols), per_sm = 2, resident = per_sm * sm_count();
    if (pl.tiles * 2 <= resident) {
        // a power of two: clusters of three leave SMs empty
        int s = 2;
        while (s < 8 && pl.tiles * s * 2 <= resident && units / (2 * s) >= 2) s *= 2;
        pl.splits = units >= 2 * s ? s : 1;
        pl.ctas = (int)(pl.tiles * pl.splits);
    } else {
        const int64_t all = pl.tiles * units;
        pl.ctas = (int)(all < resident ? all : resident);
        pl.workspace = (size_t)pl.ctas * 2 * pl.nt * 8 * 128 * sizeof(float);
    }
    const int record = q4::unit_bytes(c.group, c.has_zeros);
    pl.x_at = (int)q4::div_up(record, 1024) * 1024;
    pl.x_sub = pl.nt * 8 * 128;
    pl.half_bytes = pl.x_at + 2 * pl.x_sub;
    const int fixed = 1024 + pl.nt * 8 * kRowPad * 4 + 8 * 2 * kMaxSlots;
    pl.slots = (int)((226 * 1024 / per_sm - 1024 - fixed) / (2 * pl.half_bytes));
    if (pl.slots > kMaxSlots) pl.slots = kMaxSlots;
    pl.smem = fixed + pl.slots * 2 * pl.half_bytes;
    return pl;
}

template <typename T, int NT, bool G32>
int launch_small(const CUtensorMap& map, const SmallParams& p, const SmallPlan& pl, cudaStream_t st, const char* what) {
    auto kernel = int4_small_kernel<T, NT, G32>;
    if (int e = allow_smem((const void*)kernel, pl.smem, what)) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = pl.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)pl.ctas);
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = pl.smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = pl.splits > 0 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, map, p);
    if (int e = launch_status(what)) return e;
    if (pl.splits > 0) return P2P_OK;
    cfg.gridDim = dim3((unsigned)pl.tiles);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, int4_small_join_kernel<T>, p, pl.ctas);
    return launch_status(what);
}

template <typename T>
int run_small(const Int4Call& c, const int32_t* order, int topk, void* workspace, cudaStream_t st, const char* what) {
    const SmallPlan pl = plan_small(c);
    const int64_t all = pl.tiles * q4::div_up(c.cols, q4::kUnitCols);
    if (all > 0x7fffffff)
        return fail(P2P_EUNSUPPORTED, "%s: %lld units of 128 x 128 weights, below 2^31", what, (long long)all);
    SmallParams p = {};
    p.layout = reinterpret_cast<const uint8_t*>(c.layout);
    p.record = q4::unit_bytes(c.group, c.has_zeros);
    p.zeros = c.has_zeros;
    p.scales_at = q4::kCodeBytes + q4::unit_zero_bytes(c.group, c.has_zeros);
    p.units = (int)q4::div_up(c.cols, q4::kUnitCols);
    p.row_tiles = (int)q4::row_tiles(c.rows, c.gated);
    p.group_shift = c.group == 32 ? 5 : c.group == 64 ? 6 : 7;
    p.gated = c.gated;
    p.tokens = (int)c.tokens;
    p.n_max = pl.nt * 8;
    p.out_rows = (int)(c.gated ? c.rows / 2 : c.rows);
    p.splits = pl.splits;
    p.partial = reinterpret_cast<float*>(workspace);
    p.slots = pl.slots;
    p.half_bytes = pl.half_bytes;
    p.x_at = pl.x_at;
    p.x_sub = pl.x_sub;
    p.y = c.y;
    p.ldy = c.ldy;
    p.items = c.items;
    p.n_items = c.n_items;
    p.order = order;
    p.topk = topk;
    p.routed = c.routed;
    p.pairs = c.pairs;
    p.hold = c.hold;
    p.wait_ns = c.wait_ns;
    p.seq = next_seq();
    const int64_t x_rows = order ? c.pairs / topk : c.items ? c.pairs : c.tokens;
    CUtensorMap map;
    if (int e = encode_x_map(&map, c.x, c.dtype, x_rows, c.cols, c.ldx, order ? 1 : pl.nt * 8)) return e;
    const bool g32 = c.group == 32;
    switch (pl.nt) {
        case 1: return g32 ? launch_small<T, 1, true>(map, p, pl, st, what) : launch_small<T, 1, false>(map, p, pl, st, what);
        case 2: return g32 ? launch_small<T, 2, true>(map, p, pl, st, what) : launch_small<T, 2, false>(map, p, pl, st, what);
        case 3: return g32 ? launch_small<T, 3, true>(map, p, pl, st, what) : launch_small<T, 3, false>(map, p, pl, st, what);
        default: return g32 ? launch_small<T, 4, true>(map, p, pl, st, what) : launch_small<T, 4, false>(map, p, pl, st, what);
    }
}

int group_shift(int group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

}  // namespace
}  // namespace p2p

using namespace p2p;

extern "C" int p2p_int4_quantize(const void* w, int dtype, int64_t rows, int64_t cols, int64_t ldw, int group,
                                 uint8_t* codes, void* scales, uint8_t* zeros, void* stream) {
    P2P_REQUIRE(rows >= 0 && cols >= 1 && cols <= 0x7fffffff && ldw >= cols, "p2p_int4_quantize: bad shape");
    P2P_REQUIRE(group_shift(group) > 0, "p2p_int4_quantize: groups of %d columns, not 32, 64 or 128", group);
    if (dtype != P2P_BF16 && dtype != P2P_F16) return fail(P2P_EUNSUPPORTED, "p2p_int4_quantize: bf16 or f16");
    if (rows == 0) return P2P_OK;
    P2P_REQUIRE(w && codes && scales, "p2p_int4_quantize: null pointer");
    const int64_t warps = rows * q4::div_up(cols, group), most = (int64_t)sm_count() * 32;
    const int grid = (int)(q4::div_up(warps, 8) < most ? q4::div_up(warps, 8) : most);
    if (dtype == P2P_BF16)
        quantize_kernel<<<grid, 256, 0, as_stream(stream)>>>(reinterpret_cast<const __nv_bfloat16*>(w), ldw, rows,
                                                             (int)cols, group, codes,
                                                             reinterpret_cast<__nv_bfloat16*>(scales), zeros);
    else
        quantize_kernel<<<grid, 256, 0, as_stream(stream)>>>(reinterpret_cast<const __half*>(w), ldw, rows, (int)cols,
                                                             group, codes, reinterpret_cast<__half*>(scales), zeros);
    return launch_status("p2p_int4_quantize");
}

extern "C" int p2p_int4_expand(const uint8_t* codes, const void* scales, const uint8_t* zeros, int dtype, int64_t rows,
                               int64_t cols, int group, void* dense, void* stream) {
    P2P_REQUIRE(rows >= 0 && cols >= 1 && cols <= 0x7fffffff, "p2p_int4_expand: bad shape");
    P2P_REQUIRE(group_shift(group) > 0, "p2p_int4_expand: groups of %d columns, not 32, 64 or 128", group);
    if (dtype != P2P_BF16 && dtype != P2P_F16) return fail(P2P_EUNSUPPORTED, "p2p_int4_expand: bf16 or f16");
    if (rows == 0) return P2P_OK;
    P2P_REQUIRE(codes && scales && dense, "p2p_int4_expand: null pointer");
    const int grid = sm_count() * 16;
    if (dtype == P2P_BF16)
        expand_kernel<<<grid, 256, 0, as_stream(stream)>>>(codes, reinterpret_cast<const __nv_bfloat16*>(scales), zeros,
                                                           rows, (int)cols, group,
                                                           reinterpret_cast<__nv_bfloat16*>(dense));
    else
        expand_kernel<<<grid, 256, 0, as_stream(stream)>>>(codes, reinterpret_cast<const __half*>(scales), zeros, rows,
                                                           (int)cols, group, reinterpret_cast<__half*>(dense));
    return launch_status("p2p_int4_expand");
}

extern "C" int64_t p2p_int4_layout_bytes(int64_t experts, int64_t rows, int64_t cols, int group, int has_zeros,
                                         int gated) {
    if (experts < 1 || rows < 1 || cols < 1 || (gated && rows % 2) || group_shift(group) < 0) return -1;
    return q4::layout_bytes(experts, rows, cols, group, has_zeros != 0, gated);
}

extern "C" int p2p_int4_layout(const uint8_t* codes, const void* scales, const uint8_t* zeros, int64_t experts,
                               int64_t rows, int64_t cols, int group, int gated, void* layout, void* stream) {
    P2P_REQUIRE(experts >= 1 && rows >= 1 && cols >= 1 && cols <= 0x7fffffff && !(gated && rows % 2),
                "p2p_int4_layout: bad shape");
    P2P_REQUIRE(group_shift(group) > 0, "p2p_int4_layout: groups of %d columns, not 32, 64 or 128", group);
    P2P_REQUIRE(codes && scales && layout, "p2p_int4_layout: null pointer");
    P2P_REQUIRE(aligned16(layout), "p2p_int4_layout: the layout must start on a 16-byte boundary");
    layout_kernel<<<sm_count() * 16, 256, 0, as_stream(stream)>>>(codes, reinterpret_cast<const uint16_t*>(scales), zeros,
                                                                  experts, rows, (int)cols, group, gated,
                                                                  reinterpret_cast<uint32_t*>(layout));
    return launch_status("p2p_int4_layout");
}

namespace {
// Calls of up to this many tokens take the kernel above, which multiplies on the warps' own tensor path, so that nothing
// changes hands; above, that path's rate binds. Both sides, us at 32 tokens here and at 33 on tcgen05, which takes the same
// up to 48 (bf16; groups of 128, 64 and 32):
//   28672 x 4096     34.4, 34.6    34.3, 48.2    38.3, 75.5
//    6912 x 5120     18.2, 18.4    18.2, 22.2    19.4, 30.0    (zero points)
//    4096 x 14336    20.7, 24.8    20.9, 31.5    23.2, 45.0
//    1024 x 4096      8.4, 25.4     8.6, 22.4     8.4, 24.9
// The switch is where the two meet for large modules with groups of 128. Below it tcgen05 never wins; above it, small
// modules and finer groups would take two tiles of tokens here in less, which the kernel above does not cut.
constexpr int64_t kSmallTokens = 32;

int check_int4(const Int4Call& c, const char* what) {
    if (c.dtype != P2P_BF16 && c.dtype != P2P_F16) return fail(P2P_EUNSUPPORTED, "%s: bf16 or f16", what);
    P2P_REQUIRE(c.rows <= 0x7fffffff - 256 && c.cols >= 1 && c.cols <= 0x7fffffff - 256, "%s: bad shape", what);
    P2P_REQUIRE(group_shift(c.group) > 0, "%s: groups of %d columns, not 32, 64 or 128", what, c.group);
    P2P_REQUIRE(!(c.gated && c.rows % 2), "%s: a gated module has as many gate rows as up rows", what);
    P2P_REQUIRE(c.x && c.layout && c.y, "%s: null pointer", what);
    P2P_REQUIRE(aligned16(c.layout), "%s: the layout must start on a 16-byte boundary", what);
    P2P_REQUIRE(c.ldx >= c.cols && c.ldy >= (c.gated ? c.rows / 2 : c.rows), "%s: a row stride below the row", what);
    P2P_REQUIRE(aligned16(c.x) && c.ldx % 8 == 0, "%s: x's rows must start on 16-byte boundaries", what);
    return P2P_OK;
}
}  // namespace

extern "C" size_t p2p_int4_workspace(int64_t tokens, int64_t rows, int64_t cols, int gated) {
    if (tokens <= 0 || rows <= 0 || cols <= 0 || (gated && rows % 2)) return 0;
    if (tokens > kSmallTokens) return int4_tc_workspace(tokens, rows, cols, gated);
    Int4Call c = {};
    c.tokens = tokens; c.rows = rows; c.cols = cols; c.gated = gated != 0; c.group = 128;
    return plan_small(c).workspace;
}

extern "C" size_t p2p_int4_grouped_workspace(int64_t max_items, int64_t item_tokens, int64_t rows, int64_t cols, int gated) {
    if (max_items <= 0 || item_tokens <= 0 || item_tokens > kSmallTokens || rows <= 0 || cols <= 0 || (gated && rows % 2))
        return 0;
    Int4Call c = {};
    static const int32_t some = 0;
    c.items = &some; c.max_items = max_items; c.item_tokens = item_tokens;
    c.rows = rows; c.cols = cols; c.gated = gated != 0; c.group = 128;
    return plan_small(c).workspace;
}

namespace {
// p2p_int4_mm on a call that brings a test's withheld load and wait limit, or their defaults.
int int4_mm(Int4Call c, const void* x, int dtype, int64_t tokens, int64_t cols, int64_t ldx, const void* layout,
            int has_zeros, int64_t rows, int group, int gated, void* y, int64_t ldy, void* workspace,
            size_t workspace_bytes, void* stream) {
    P2P_REQUIRE(tokens >= 0 && rows >= 0 && tokens <= 0x7fffffff, "p2p_int4_mm: bad shape");
    if (tokens == 0 || rows == 0) return P2P_OK;
    c.x = x; c.dtype = dtype; c.tokens = tokens; c.cols = cols; c.ldx = ldx;
    c.layout = layout; c.has_zeros = has_zeros != 0;
    c.rows = rows; c.group = group; c.gated = gated != 0; c.y = y; c.ldy = ldy;
    if (int e = check_int4(c, "p2p_int4_mm")) return e;
    cudaStream_t st = as_stream(stream);
    const size_t need = p2p_int4_workspace(tokens, rows, cols, gated);
    P2P_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                "p2p_int4_mm: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (tokens <= kSmallTokens)
        return dtype == P2P_BF16 ? run_small<__nv_bfloat16>(c, nullptr, 1, workspace, st, "p2p_int4_mm")
                                 : run_small<__half>(c, nullptr, 1, workspace, st, "p2p_int4_mm");
    return int4_tc_run(c, workspace, st, "p2p_int4_mm");
}
}  // namespace

extern "C" int p2p_int4_mm(const void* x, int dtype, int64_t tokens, int64_t cols, int64_t ldx, const void* layout,
                           int has_zeros, int64_t rows, int group, int gated, void* y, int64_t ldy, void* workspace,
                           size_t workspace_bytes, void* stream) {
    return int4_mm({}, x, dtype, tokens, cols, ldx, layout, has_zeros, rows, group, gated, y, ldy, workspace,
                   workspace_bytes, stream);
}

extern "C" int p2p_int4_withhold(const void* x, int dtype, int64_t tokens, int64_t cols, int64_t ldx, const void* layout,
                                 int has_zeros, int64_t rows, int group, int gated, void* y, int64_t ldy,
                                 void* workspace, size_t workspace_bytes, int64_t hold, int64_t wait_us, void* stream) {
    P2P_REQUIRE(hold >= 0 && hold < 4096, "p2p_int4_withhold: load %lld", (long long)hold);
    P2P_REQUIRE(wait_us >= 1000 && wait_us <= 2000000, "p2p_int4_withhold: a limit of 1 ms to 2 s (%lld us)",
                (long long)wait_us);
    Int4Call c = {};
    c.hold = (int)hold;
    c.wait_ns = (uint64_t)wait_us * 1000ull;
    return int4_mm(c, x, dtype, tokens, cols, ldx, layout, has_zeros, rows, group, gated, y, ldy, workspace,
                   workspace_bytes, stream);
}

extern "C" int p2p_int4_grouped(const void* x, int dtype, int64_t cols, int64_t ldx, const void* layout,
                                int has_zeros, int64_t rows, int group, int gated,
                                const int32_t* items, const int32_t* n_items, int64_t max_items, int64_t item_tokens,
                                const int32_t* order, int topk, const int32_t* routed, int64_t pairs, void* y,
                                int64_t ldy, void* workspace, size_t workspace_bytes, void* stream) {
    P2P_REQUIRE(max_items >= 0 && rows >= 0 && item_tokens >= 0 && pairs >= 0 && pairs <= 0x7fffffff,
                "p2p_int4_grouped: bad shape");
    if (max_items == 0 || rows == 0 || item_tokens == 0 || pairs == 0) return P2P_OK;
    P2P_REQUIRE(item_tokens <= kInt4TileTokens, "p2p_int4_grouped: items of up to %lld tokens, at most %d",
                (long long)item_tokens, kInt4TileTokens);
    P2P_REQUIRE(items && n_items && topk >= 1, "p2p_int4_grouped: null pointer or topk %d", topk);
    P2P_REQUIRE(aligned16(items), "p2p_int4_grouped: items must start on a 16-byte boundary");
    P2P_REQUIRE(!order || item_tokens <= 8, "p2p_int4_grouped: items of more than 8 tokens take x in the order's places");
    Int4Call c = {};
    c.x = x; c.dtype = dtype; c.cols = cols; c.ldx = ldx;
    c.layout = layout; c.has_zeros = has_zeros != 0;
    c.rows = rows; c.group = group; c.gated = gated != 0; c.y = y; c.ldy = ldy;
    c.items = items; c.n_items = n_items; c.max_items = max_items; c.item_tokens = item_tokens; c.pairs = pairs;
    c.routed = routed;
    if (int e = check_int4(c, "p2p_int4_grouped")) return e;
    cudaStream_t st = as_stream(stream);
    const size_t need = p2p_int4_grouped_workspace(max_items, item_tokens, rows, cols, gated);
    P2P_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                "p2p_int4_grouped: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (item_tokens <= kSmallTokens)
        return dtype == P2P_BF16 ? run_small<__nv_bfloat16>(c, order, topk, workspace, st, "p2p_int4_grouped")
                                 : run_small<__half>(c, order, topk, workspace, st, "p2p_int4_grouped");
    return int4_tc_run(c, nullptr, st, "p2p_int4_grouped");
}

extern "C" int p2p_int4_status(int reset, void* stream) {
    cudaStream_t st = as_stream(stream);
    int v[2] = {0, 0};
    if (cudaMemcpyFromSymbolAsync(&v[0], g_small_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaStreamSynchronize(st) != cudaSuccess)
        return fail(P2P_ECUDA, "p2p_int4_status: %s", cudaGetErrorString(cudaGetLastError()));
    if (int e = int4_tc_error(&v[1], reset, st)) return e;
    if (reset && v[0]) {
        const int zero = 0;
        cudaMemcpyToSymbolAsync(g_small_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
        cudaStreamSynchronize(st);
    }
    if (v[0] || v[1]) return fail(P2P_ECUDA, "p2p_int4: a pipeline wait timed out (sites %d, %d)", v[0], v[1]);
    return P2P_OK;
}
