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
        const float s = to_f32(scales[at]), z = zeros ? (float)zeros[at] : 8.f;
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
constexpr uint64_t kSmallWaitNs = 2000000000ull;

__device__ int g_small_error;            // site of the first wait that gave up since the last reset (0: none)
__device__ unsigned g_small_failed_seq;  // sequence number of the last launch in which a wait gave up

struct SmallParams {
    const uint8_t* layout;
    int record, zeros, scales_at;       // bytes of a unit's record; whether it holds zero points; where its scales start
    int units, row_tiles, group_shift, gated;
    int tokens, out_rows;
    int splits;                         // CTAs of a cluster, each with its share of the units
    int slots, slot_bytes, x_at, x_sub; // ring: record, then two x boxes of x_sub bytes at x_at
    void* y;
    int64_t ldy;
    const int32_t* items;               // routed: {expert, first place, places, 0}
    const int32_t* n_items;
    const int32_t* order;               // routed: place -> pair, x's row being pair / topk; null: the place itself
    int topk;
    const int32_t* routed;              // not null: output rows from *routed to pairs become zero
    int64_t pairs;
    uint64_t wait_ns;
    unsigned seq;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint2 b, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint2 b, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}
__device__ __forceinline__ uint2 lds_v2(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t lds_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// A CTA takes a row tile (128 rows), up to 8 NT tokens and a share of the columns; the CTAs of a cluster hold the row
// tile's shares and add them up over distributed shared memory, in column order. One warp streams the share's records
// and x tiles into a ring of shared memory; warp w multiplies row block w: the codes become exact small integers, eight
// m16n8k16 products a unit and 8 tokens add a group's columns in fp32, and the group's scale multiplies that sum on its
// way into the fp32 accumulators: no weight is ever rounded.
template <typename T, int NT>
__global__ void __launch_bounds__(kSmallThreads, NT <= 2 ? 4 : 3) int4_small_kernel(const __grid_constant__ CUtensorMap tmap_x,
                                                                                   const __grid_constant__ SmallParams p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    const uint32_t bars = base + (uint32_t)(p.slots * p.slot_bytes);
    auto full = [&](int s) { return bars + 8u * s; };
    auto empty = [&](int s) { return bars + 8u * (kMaxSlots + s); };
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
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
    int64_t expert = 0, first = (int64_t)blockIdx.y * (NT * 8);
    int count = 0;
    if (p.items) {
        asm volatile("griddepcontrol.wait;" ::: "memory");           // the items are the previous kernel's
        const int n_items = *p.n_items;
        if ((int)blockIdx.y >= n_items) {                            // no item left: zero what lies behind the last pair
            const int64_t col = (int64_t)tile * (p.gated ? 64 : 128) + threadIdx.x;
            if (p.routed && rank == 0 && threadIdx.x < (p.gated ? 64 : 128) && col < p.out_rows)
                for (int64_t r = *p.routed + (blockIdx.y - n_items); r < p.pairs; r += gridDim.y - n_items)
                    reinterpret_cast<T*>(p.y)[r * p.ldy + col] = from_f32<T>(0.f);
            return;
        }
        const int4 it = reinterpret_cast<const int4*>(p.items)[blockIdx.y];
        expert = it.x;
        first = it.y;
        count = min(it.z, NT * 8);
    } else {
        count = (int)min((int64_t)(NT * 8), p.tokens - first);
    }
    const int k0 = (int)((int64_t)p.units * rank / p.splits), k1 = (int)((int64_t)p.units * (rank + 1) / p.splits);
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;

    if (warp == kComputeWarps) {
        if (elect_one()) {
            const uint8_t* src = p.layout + ((expert * p.row_tiles + tile) * p.units + k0) * p.record;
            const int n_slots = p.slots;
            const uint32_t x_rows = p.order ? (uint32_t)count : (uint32_t)(NT * 8);
            bool ok = true, first_x = true;
            auto load_x = [&](int slot, int k) {
                const uint32_t at = base + slot * p.slot_bytes + p.x_at;
                if (p.order) {                                       // a row at a time, from wherever its token lies
                    for (int i = 0; i < count; ++i) {
                        const int row = __ldcg(p.order + first + i) / p.topk;
                        tma_load_2d(at + i * 128, &tmap_x, k * 128, row, full(slot));
                        tma_load_2d(at + p.x_sub + i * 128, &tmap_x, k * 128 + 64, row, full(slot));
                    }
                } else {
                    tma_load_2d(at, &tmap_x, k * 128, (int)first, full(slot));
                    tma_load_2d(at + p.x_sub, &tmap_x, k * 128 + 64, (int)first, full(slot));
                }
            };
            // the ring's first fill: all weights, then, once x is there, all x tiles
            const int head = min(n_slots, k1 - k0);
            for (int i = 0; i < head; ++i) {
                mbar_expect_tx(full(i), (uint32_t)p.record + 2u * 128u * x_rows);
                bulk_load(base + i * p.slot_bytes, src + (int64_t)i * p.record, (uint32_t)p.record, full(i));
            }
            if (!p.items) asm volatile("griddepcontrol.wait;" ::: "memory");   // x may be the previous kernel's output
            for (int i = 0; i < head; ++i) load_x(i, k0 + i);
            int slot = 0, used = head;
            uint32_t ph = 0;
            for (int k = k0 + head; k < k1; ++k) {
                if (!(ok = wait_one(empty(slot), ph, 1, wc))) break;
                mbar_expect_tx(full(slot), (uint32_t)p.record + 2u * 128u * x_rows);
                bulk_load(base + slot * p.slot_bytes, src + (int64_t)(k - k0) * p.record, (uint32_t)p.record, full(slot));
                load_x(slot, k);
                ++used;
                advance(slot, ph, 1, n_slots);
            }
            // every copy issued must have landed before the CTA may exit: each slot's last one
            for (int i = max(0, used - n_slots); i < used; ++i)
                mbar_drain(full(i % n_slots), (uint32_t)((i / n_slots) & 1), 2, wc);
        }
        __syncwarp();
    } else {
        if (!p.items) asm volatile("griddepcontrol.wait;" ::: "memory");       // y may be the previous kernel's input
        const int j = lane & 3, n = lane >> 2;
        // this lane's columns 4 j.. of a 16-column step, in the 128-byte swizzle: 16-byte chunk 2 r + j / 2, XOR row
        const uint32_t x_row = (uint32_t)(p.x_at + n * 128 + (j & 1) * 8);
        int slot = 0;
        uint32_t ph = 0;
        for (int k = k0; k < k1; ++k) {
            if (!__all_sync(0xffffffffu, wait_one(full(slot), ph, 3, wc))) break;
            const uint32_t rec = base + slot * p.slot_bytes;
            const uint32_t mine = (uint32_t)(warp * 8 + n);           // of a group's 64 pairs of rows
            q4::Codes<T> codes;
            float part[NT][4];
            auto clear = [&] {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[t][i] = 0.f;
            };
            auto begin = [&](int g) {                                 // group g of the unit
                const uint32_t z = p.zeros ? lds_u16(rec + q4::kCodeBytes + (g * 64 + mine) * 2) : 0x0808u;
                codes.zeros(z & 15u, z >> 8);
                clear();
            };
            auto end = [&](int g) {
                const float2 s = unpack2<T>(lds_u32(rec + p.scales_at + (g * 64 + mine) * 4));
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    acc[t][0] = fmaf(s.x, part[t][0], acc[t][0]);
                    acc[t][1] = fmaf(s.x, part[t][1], acc[t][1]);
                    acc[t][2] = fmaf(s.y, part[t][2], acc[t][2]);
                    acc[t][3] = fmaf(s.y, part[t][3], acc[t][3]);
                }
            };
            begin(0);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint4 c = lds_v4(rec + (warp * 2 + half) * q4::kBlockBytes + lane * 16);
                const uint32_t w[4] = {c.x, c.y, c.z, c.w};
                if (half == 1 && p.group_shift < 7) {
                    end(p.group_shift == 6 ? 0 : 1);
                    begin(p.group_shift == 6 ? 1 : 2);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (r == 2 && p.group_shift == 5) {
                        end(2 * half);
                        begin(2 * half + 1);
                    }
                    uint32_t a[4];
                    codes.expand(w[r], a);
                    const uint32_t at = rec + x_row + half * p.x_sub + (((2 * r + (j >> 1)) ^ n) << 4);
#pragma unroll
                    for (int t = 0; t < NT; ++t) mma16816(part[t], a, lds_v2(at + t * 1024), T());
                }
            }
            end(p.group_shift == 7 ? 0 : p.group_shift == 6 ? 1 : 3);
            __syncwarp();
            if (lane == 0) mbar_arrive(empty(slot));
            advance(slot, ph, 1, p.slots);
        }
    }
    // Each CTA's partial tile [token][row] goes to the front of its own ring, all of whose copies have been read.
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem_raw + (base - raw));
    if (warp < kComputeWarps) {
        const int j = lane & 3, n = lane >> 2;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                red[(t * 8 + 2 * j + (i & 1)) * kRowPad + warp * 16 + n + 8 * (i >> 1)] = acc[t][i];
    }
    if (p.splits > 1) cluster_sync_all(); else __syncthreads();
    // Sum over the cluster, in column order: CTA `rank` finishes every splits-th token... of all rows.
    auto total = [&](int tok, int row) {
        const uint32_t at = smem_u32(red + tok * kRowPad + row);
        if (p.splits == 1) return __uint_as_float(lds_u32(at));
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
    const int begin = count * width * rank / p.splits, end = count * width * (rank + 1) / p.splits;
    for (int i = begin + threadIdx.x; i < end; i += kSmallThreads) {
        const int tok = i / width, in = i % width;
        const int64_t row = (int64_t)tile * width + in;
        if (row >= p.out_rows) continue;
        float v;
        if (p.gated) {                                               // even row blocks are gates, odd ones their ups
            const float g = total(tok, in / 16 * 32 + in % 16), u = total(tok, in / 16 * 32 + 16 + in % 16);
            v = g / (1.f + expf(-g)) * u;
        } else {
            v = total(tok, in);
        }
        y[(first + tok) * p.ldy + row] = from_f32<T>(v);
    }
    if (p.splits > 1) cluster_sync_all();                            // nobody leaves while its tile may still be read
}

unsigned next_seq() {
    static std::atomic<unsigned> counter{0};
    unsigned v = ++counter;
    while (v == 0) v = ++counter;
    return v;
}

template <typename T, int NT>
int launch_small(const CUtensorMap& map, SmallParams& p, int64_t col_tiles, cudaStream_t st, const char* what) {
    auto kernel = int4_small_kernel<T, NT>;
    const int smem = 1024 + p.slots * p.slot_bytes + 8 * 2 * kMaxSlots;
    if (int e = allow_smem((const void*)kernel, smem, what)) return e;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(p.row_tiles * p.splits), (unsigned)col_tiles);
    cfg.blockDim = dim3(kSmallThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = p.splits > 1 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, map, (const SmallParams)p);
    return launch_status(what);
}

// Up to 32 tokens (an item, or a tile of the tokens).
template <typename T>
int run_small(const Int4Call& c, const int32_t* order, int topk, cudaStream_t st, const char* what) {
    SmallParams p = {};
    const bool routed = c.items != nullptr;
    const int64_t most = routed ? c.item_tokens : c.tokens < 32 ? c.tokens : 32;
    const int nt = (int)q4::div_up(most, 8);
    const int64_t col_tiles = routed ? c.max_items : q4::div_up(c.tokens, nt * 8);
    if (col_tiles > 65535) return fail(P2P_EUNSUPPORTED, "%s: %lld tiles of tokens, at most 65535", what, (long long)col_tiles);
    p.layout = reinterpret_cast<const uint8_t*>(c.layout);
    p.record = q4::unit_bytes(c.group, c.has_zeros);
    p.zeros = c.has_zeros;
    p.scales_at = q4::kCodeBytes + q4::unit_zero_bytes(c.group, c.has_zeros);
    p.units = (int)q4::div_up(c.cols, q4::kUnitCols);
    p.row_tiles = (int)q4::row_tiles(c.rows, c.gated);
    p.group_shift = c.group == 32 ? 5 : c.group == 64 ? 6 : 7;
    p.gated = c.gated;
    p.tokens = (int)c.tokens;
    p.out_rows = (int)(c.gated ? c.rows / 2 : c.rows);
    p.x_at = (int)q4::div_up(p.record, 1024) * 1024;
    p.x_sub = nt * 8 * 128;
    p.slot_bytes = p.x_at + 2 * p.x_sub;
    const int64_t ctas = p.row_tiles * col_tiles;
    p.splits = 1;
    while (p.splits < 8 && ctas * p.splits < 3 * sm_count() && p.units / (2 * p.splits) >= 2) p.splits *= 2;
    const int share = (int)q4::div_up(p.units, p.splits);
    p.slots = (72 * 1024 - 1024) / p.slot_bytes;
    if (p.slots > kMaxSlots) p.slots = kMaxSlots;
    if (p.slots > share) p.slots = share;
    // the partial tile reuses the ring
    const int tile_bytes = nt * 8 * kRowPad * 4;
    while (p.slots * p.slot_bytes < tile_bytes) ++p.slots;
    p.y = c.y;
    p.ldy = c.ldy;
    p.items = c.items;
    p.n_items = c.n_items;
    p.order = order;
    p.topk = topk;
    p.routed = c.routed;
    p.pairs = c.pairs;
    p.wait_ns = kSmallWaitNs;
    p.seq = next_seq();
    const int64_t x_rows = order ? c.pairs / topk : routed ? c.pairs : c.tokens;
    CUtensorMap map;
    if (int e = encode_x_map(&map, c.x, c.dtype, x_rows, c.cols, c.ldx, order ? 1 : nt * 8)) return e;
    switch (nt) {
        case 1: return launch_small<T, 1>(map, p, col_tiles, st, what);
        case 2: return launch_small<T, 2>(map, p, col_tiles, st, what);
        case 3: return launch_small<T, 3>(map, p, col_tiles, st, what);
        default: return launch_small<T, 4>(map, p, col_tiles, st, what);
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
// Calls of up to this many tokens take the kernel above, which streams weights at the memory's rate and multiplies on
// the warps' own tensor path; above, that path's rate would bind.
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
    if (tokens <= kSmallTokens || rows <= 0 || cols <= 0 || (gated && rows % 2)) return 0;
    return int4_tc_workspace(tokens, rows, cols, gated);
}

extern "C" int p2p_int4_mm(const void* x, int dtype, int64_t tokens, int64_t cols, int64_t ldx, const void* layout,
                           int has_zeros, int64_t rows, int group, int gated, void* y, int64_t ldy, void* workspace,
                           size_t workspace_bytes, void* stream) {
    P2P_REQUIRE(tokens >= 0 && rows >= 0 && tokens <= 0x7fffffff, "p2p_int4_mm: bad shape");
    if (tokens == 0 || rows == 0) return P2P_OK;
    Int4Call c = {};
    c.x = x; c.dtype = dtype; c.tokens = tokens; c.cols = cols; c.ldx = ldx;
    c.layout = layout; c.has_zeros = has_zeros != 0;
    c.rows = rows; c.group = group; c.gated = gated != 0; c.y = y; c.ldy = ldy;
    if (int e = check_int4(c, "p2p_int4_mm")) return e;
    cudaStream_t st = as_stream(stream);
    if (tokens <= kSmallTokens)
        return dtype == P2P_BF16 ? run_small<__nv_bfloat16>(c, nullptr, 1, st, "p2p_int4_mm")
                                 : run_small<__half>(c, nullptr, 1, st, "p2p_int4_mm");
    const size_t need = p2p_int4_workspace(tokens, rows, cols, gated);
    P2P_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                "p2p_int4_mm: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return int4_tc_run(c, workspace, st, "p2p_int4_mm");
}

extern "C" int p2p_int4_grouped(const void* x, int dtype, int64_t cols, int64_t ldx, const void* layout,
                                int has_zeros, int64_t rows, int group, int gated,
                                const int32_t* items, const int32_t* n_items, int64_t max_items, int64_t item_tokens,
                                const int32_t* order, int topk, const int32_t* routed, int64_t pairs, void* y,
                                int64_t ldy, void* stream) {
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
    if (item_tokens <= kSmallTokens)
        return dtype == P2P_BF16 ? run_small<__nv_bfloat16>(c, order, topk, st, "p2p_int4_grouped")
                                 : run_small<__half>(c, order, topk, st, "p2p_int4_grouped");
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
