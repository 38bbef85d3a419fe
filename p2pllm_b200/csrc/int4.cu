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
#include <stdlib.h>
#include "int4.cuh"
#include "int4_run.cuh"

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

struct Int4Params {
    const void* x;
    int64_t ldx;
    int vec;                          // x's rows start on 8 bytes and cols is a multiple of 4: 8-byte loads
    const uint8_t* layout;
    int record, scales_at;            // bytes of a unit's record, and where its scales start
    int zeros;                        // it holds zero points (else 8 everywhere)
    int tokens, cols, kbs, units, group_shift;
    int64_t rows, rbs, tiles;         // rows (a gated module's: both halves), row blocks and row tiles of one expert
    int gated;
    void* y;
    int64_t ldy;
    const int32_t* items;             // routed: {expert, first place, places, 0}
    const int32_t* n_items;
    const int32_t* order;             // routed: place -> pair, x's row being pair / topk; null: the place itself
    int topk;
    const int32_t* routed;            // not null: output rows from *routed to pairs become zero
    int64_t pairs;
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

// Four columns k.. of an x row (null: a row past the tokens), zero past the module's columns.
template <typename T>
__device__ __forceinline__ uint2 load_x(const T* row, int k, int cols, int vec) {
    if (row == nullptr) return make_uint2(0u, 0u);
    if (vec) return k < cols ? __ldg(reinterpret_cast<const uint2*>(row + k)) : make_uint2(0u, 0u);
    const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + k;
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < cols ? __ldg(p + i) : 0u;
    return make_uint2(v[0] | (v[1] << 16), v[2] | (v[3] << 16));
}

// A CTA takes RB row blocks (16 RB rows) and up to 8 NT tokens; its warps take column blocks in turn, U at a step, and
// add up their sums in shared memory, in warp order. Within a warp the codes become exact small integers, four
// m16n8k16 products add a group's 32 or 64 columns in fp32, and the group's scale multiplies that sum on its way into
// the fp32 accumulators: no weight is ever rounded.
template <typename T, int NT, int RB, int WARPS>
__global__ void __launch_bounds__(WARPS * 32) int4_kernel(const __grid_constant__ Int4Params p) {
    constexpr int U = RB == 1 ? 4 : 2;                               // column blocks in flight a warp
    __shared__ float red[WARPS][RB * 16][NT * 8 + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, j = lane & 3, n = lane >> 2;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int64_t expert = 0, first = (int64_t)blockIdx.y * (NT * 8);
    int count = 0;
    if (p.items) {
        asm volatile("griddepcontrol.wait;" ::: "memory");           // the items are the previous kernel's
        const int n_items = *p.n_items;
        if ((int)blockIdx.y >= n_items) {                            // no item left: zero what lies behind the last pair
            if (p.routed) {
                const int64_t out_rows = p.gated ? p.rows / 2 : p.rows, width = (p.gated ? RB / 2 : RB) * 16;
                const int64_t col = blockIdx.x * width + threadIdx.x;
                if (threadIdx.x < width && col < out_rows)
                    for (int64_t r = *p.routed + (blockIdx.y - n_items); r < p.pairs; r += gridDim.y - n_items)
                        reinterpret_cast<T*>(p.y)[r * p.ldy + col] = from_f32<T>(0.f);
            }
            return;
        }
        const int4 it = reinterpret_cast<const int4*>(p.items)[blockIdx.y];
        expert = it.x;
        first = it.y;
        count = min(it.z, NT * 8);
    } else {
        count = (int)min((int64_t)(NT * 8), p.tokens - first);
    }
    const int64_t rb0 = (int64_t)blockIdx.x * RB;                    // RB divides a tile's 8 blocks
    const uint8_t* base = p.layout + (expert * p.tiles + rb0 / 8) * p.units * p.record;
    const int blk = (int)(rb0 & 7);
    const int n_rb = (int)min((int64_t)RB, p.rbs - rb0);
    struct Stage {
        uint4 w[U][RB];
        uint32_t s[U][RB][2];
        uint16_t z[U][RB][2];
    };
    auto load = [&](Stage& st, int step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kb = step * U + u;
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                st.w[u][b] = make_uint4(0u, 0u, 0u, 0u);
                st.s[u][b][0] = st.s[u][b][1] = 0u;
                st.z[u][b][0] = st.z[u][b][1] = 0x0808;
                if (kb < p.kbs && b < n_rb) {
                    const uint8_t* rec = base + (int64_t)(kb >> 1) * p.record;
                    st.w[u][b] = __ldg(reinterpret_cast<const uint4*>(rec + ((blk + b) * 2 + (kb & 1)) * q4::kBlockBytes) + lane);
                    // the block's first group in its unit, and with groups of 32 the next
                    const int g = p.group_shift == 7 ? 0 : p.group_shift == 6 ? kb & 1 : 2 * (kb & 1);
                    const int at = (g * 8 + blk + b) * 8 + n;
                    const uint32_t* sc = reinterpret_cast<const uint32_t*>(rec + p.scales_at) + at;
                    const uint16_t* ze = reinterpret_cast<const uint16_t*>(rec + q4::kCodeBytes) + at;
                    st.s[u][b][0] = __ldg(sc);
                    if (p.zeros) st.z[u][b][0] = __ldg(ze);
                    if (p.group_shift == 5) {
                        st.s[u][b][1] = __ldg(sc + 64);
                        if (p.zeros) st.z[u][b][1] = __ldg(ze + 64);
                    }
                }
            }
        }
    };
    const int steps = (p.kbs + U - 1) / U;
    Stage cur, nxt;
    if (warp < steps) load(cur, warp);                               // weights wait for nobody
    if (!p.items) asm volatile("griddepcontrol.wait;" ::: "memory"); // x may be the previous kernel's output
    const T* xrow[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int i = t * 8 + n;
        xrow[t] = nullptr;
        if (i < count) {
            int64_t row = first + i;
            if (p.order) row = p.order[row] / p.topk;
            xrow[t] = reinterpret_cast<const T*>(p.x) + row * p.ldx;
        }
    }
    float acc[RB][NT][4];
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[b][t][i] = 0.f;
    for (int step = warp; step < steps; step += WARPS) {
        if (step + WARPS < steps) load(nxt, step + WARPS);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = (step * U + u) * 64 + 4 * j;
            uint2 xf[4][NT];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < NT; ++t) xf[r][t] = load_x(xrow[t], k0 + 16 * r, p.cols, p.vec);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                const uint32_t w[4] = {cur.w[u][b].x, cur.w[u][b].y, cur.w[u][b].z, cur.w[u][b].w};
                q4::Codes<T> codes;
                float part[NT][4];
                auto clear = [&] {
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) part[t][i] = 0.f;
                };
                auto promote = [&](int h) {
                    const float2 s = unpack2<T>(cur.s[u][b][h]);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        acc[b][t][0] = fmaf(s.x, part[t][0], acc[b][t][0]);
                        acc[b][t][1] = fmaf(s.x, part[t][1], acc[b][t][1]);
                        acc[b][t][2] = fmaf(s.y, part[t][2], acc[b][t][2]);
                        acc[b][t][3] = fmaf(s.y, part[t][3], acc[b][t][3]);
                    }
                };
                codes.zeros(cur.z[u][b][0] & 15u, cur.z[u][b][0] >> 8);
                clear();
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (r == 2 && p.group_shift == 5) {              // a group of 32 ends inside the block
                        promote(0);
                        clear();
                        codes.zeros(cur.z[u][b][1] & 15u, cur.z[u][b][1] >> 8);
                    }
                    uint32_t a[4];
                    codes.expand(w[r], a);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        if (t * 8 < count) mma16816(part[t], a, xf[r][t], T());
                }
                promote(p.group_shift == 5 ? 1 : 0);
            }
        }
        cur = nxt;
    }
#pragma unroll
    for (int b = 0; b < RB; ++b)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) red[warp][b * 16 + n + 8 * (i >> 1)][t * 8 + 2 * j + (i & 1)] = acc[b][t][i];
    __syncthreads();
    auto total = [&](int row, int tok) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) v += red[w][row][tok];
        return v;
    };
    T* y = reinterpret_cast<T*>(p.y);
    if (RB % 2 == 0 && p.gated) {
        constexpr int kUnits = RB < 2 ? 1 : RB / 2 * 16;
        const int64_t half = p.rows / 2;
        for (int i = threadIdx.x; i < kUnits * count; i += WARPS * 32) {
            const int in = i % kUnits, tok = i / kUnits;
            const int64_t row = rb0 / 2 * 16 + in;
            if (row >= half) continue;
            const float g = total(in / 16 * 32 + in % 16, tok), u = total(in / 16 * 32 + 16 + in % 16, tok);
            y[(first + tok) * p.ldy + row] = from_f32<T>(g / (1.f + expf(-g)) * u);
        }
    } else {
        for (int i = threadIdx.x; i < RB * 16 * count; i += WARPS * 32) {
            const int in = i % (RB * 16), tok = i / (RB * 16);
            const int64_t row = rb0 * 16 + in;
            if (row < p.rows) y[(first + tok) * p.ldy + row] = from_f32<T>(total(in, tok));
        }
    }
}

template <typename T, int NT, int RB, int WARPS>
int launch_int4(const Int4Params& p, int64_t row_tiles, int64_t col_tiles, cudaStream_t st, const char* what) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)row_tiles, (unsigned)col_tiles);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, int4_kernel<T, NT, RB, WARPS>, p);
    return launch_status(what);
}

template <typename T> int run_int4(const Int4Params& p, int64_t most, int64_t n_items, cudaStream_t st, const char* what) {
    const int nt = (int)q4::div_up(most < 32 ? most : 32, 8);
    const int64_t tiles = p.items ? n_items : q4::div_up(p.tokens, nt * 8);
    const int64_t rb = p.gated ? 2 : 1, row_tiles = q4::div_up(p.rbs, rb);
    if (tiles > 65535) return fail(P2P_EUNSUPPORTED, "%s: %lld tiles of tokens, at most 65535", what, (long long)tiles);
    if (rb == 1) switch (nt) {
        case 1: return launch_int4<T, 1, 1, 8>(p, row_tiles, tiles, st, what);
        case 2: return launch_int4<T, 2, 1, 8>(p, row_tiles, tiles, st, what);
        case 3: return launch_int4<T, 3, 1, 8>(p, row_tiles, tiles, st, what);
        default: return launch_int4<T, 4, 1, 8>(p, row_tiles, tiles, st, what);
    }
    switch (nt) {
        case 1: return launch_int4<T, 1, 2, 8>(p, row_tiles, tiles, st, what);
        case 2: return launch_int4<T, 2, 2, 8>(p, row_tiles, tiles, st, what);
        case 3: return launch_int4<T, 3, 2, 8>(p, row_tiles, tiles, st, what);
        default: return launch_int4<T, 4, 2, 8>(p, row_tiles, tiles, st, what);
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
// What both products check and fill in.
int int4_params(Int4Params& p, const char* what, const void* x, int dtype, int64_t cols, int64_t ldx, const void* layout,
                int has_zeros, int64_t rows, int group, int gated, void* y, int64_t ldy) {
    if (dtype != P2P_BF16 && dtype != P2P_F16) return fail(P2P_EUNSUPPORTED, "%s: bf16 or f16", what);
    P2P_REQUIRE(rows <= 0x7fffffff && cols >= 1 && cols <= 0x7fffff00, "%s: bad shape", what);
    P2P_REQUIRE(group_shift(group) > 0, "%s: groups of %d columns, not 32, 64 or 128", what, group);
    P2P_REQUIRE(!(gated && rows % 2), "%s: a gated module has as many gate rows as up rows", what);
    P2P_REQUIRE(x && layout && y, "%s: null pointer", what);
    P2P_REQUIRE(aligned16(layout), "%s: the layout must start on a 16-byte boundary", what);
    P2P_REQUIRE(ldx >= cols && ldy >= (gated ? rows / 2 : rows), "%s: a row stride below the row", what);
    p.x = x;
    p.ldx = ldx;
    p.vec = cols % 4 == 0 && ldx % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 7u) == 0;
    p.layout = reinterpret_cast<const uint8_t*>(layout);
    p.record = q4::unit_bytes(group, has_zeros != 0);
    p.scales_at = q4::kCodeBytes + q4::unit_zero_bytes(group, has_zeros != 0);
    p.zeros = has_zeros != 0;
    p.tokens = 0;
    p.cols = (int)cols;
    p.kbs = (int)q4::div_up(cols, q4::kCols);
    p.units = (int)q4::div_up(cols, q4::kUnitCols);
    p.group_shift = group_shift(group);
    p.rows = rows;
    p.rbs = q4::row_blocks(rows, gated);
    p.tiles = q4::row_tiles(rows, gated);
    p.gated = gated;
    p.y = y;
    p.ldy = ldy;
    p.items = p.n_items = p.order = nullptr;
    p.topk = 1;
    p.routed = nullptr;
    p.pairs = 0;
    return P2P_OK;
}
}  // namespace

namespace {
// Calls of up to this many tokens stay with the kernel above.
bool use_tc(int64_t tokens, int64_t rows, int64_t cols) {
    static const char* e = getenv("P2P_INT4_TC");
    if (e) return tokens >= atoi(e);
    return tokens > 8;
}
bool tc_aligned(const void* x, int64_t ldx) { return aligned16(x) && ldx % 8 == 0; }
}  // namespace

extern "C" size_t p2p_int4_workspace(int64_t tokens, int64_t rows, int64_t cols, int gated) {
    if (tokens <= 0 || rows <= 0 || cols <= 0 || !use_tc(tokens, rows, cols)) return 0;
    return int4_tc_workspace(tokens, rows, cols, gated);
}

extern "C" int p2p_int4_mm(const void* x, int dtype, int64_t tokens, int64_t cols, int64_t ldx, const void* layout,
                           int has_zeros, int64_t rows, int group, int gated, void* y, int64_t ldy, void* workspace,
                           size_t workspace_bytes, void* stream) {
    P2P_REQUIRE(tokens >= 0 && rows >= 0 && tokens <= 0x7fffffff, "p2p_int4_mm: bad shape");
    if (tokens == 0 || rows == 0) return P2P_OK;
    Int4Params p;
    if (int e = int4_params(p, "p2p_int4_mm", x, dtype, cols, ldx, layout, has_zeros, rows, group, gated, y, ldy))
        return e;
    cudaStream_t st = as_stream(stream);
    if (use_tc(tokens, rows, cols)) {
        P2P_REQUIRE(tc_aligned(x, ldx), "p2p_int4_mm: %lld tokens need x rows of 16-byte alignment", (long long)tokens);
        const size_t need = p2p_int4_workspace(tokens, rows, cols, gated);
        P2P_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && aligned16(workspace)),
                    "p2p_int4_mm: workspace of %zu bytes, %zu needed", workspace_bytes, need);
        Int4Call c = {};
        c.x = x; c.dtype = dtype; c.tokens = tokens; c.cols = cols; c.ldx = ldx;
        c.layout = layout; c.has_zeros = has_zeros != 0;
        c.rows = rows; c.group = group; c.gated = gated; c.y = y; c.ldy = ldy;
        return int4_tc_run(c, workspace, st, "p2p_int4_mm");
    }
    p.tokens = (int)tokens;
    return dtype == P2P_BF16 ? run_int4<__nv_bfloat16>(p, tokens, 0, st, "p2p_int4_mm")
                             : run_int4<__half>(p, tokens, 0, st, "p2p_int4_mm");
}

extern "C" int p2p_int4_grouped(const void* x, int dtype, int64_t cols, int64_t ldx, const void* layout,
                                int has_zeros, int64_t rows, int group, int gated,
                                const int32_t* items, const int32_t* n_items, int64_t max_items, int64_t item_tokens,
                                const int32_t* order, int topk, const int32_t* routed, int64_t pairs, void* y,
                                int64_t ldy, void* stream) {
    P2P_REQUIRE(max_items >= 0 && rows >= 0 && item_tokens >= 0 && pairs >= 0 && pairs <= 0x7fffffff,
                "p2p_int4_grouped: bad shape");
    if (max_items == 0 || rows == 0 || item_tokens == 0 || pairs == 0) return P2P_OK;
    const bool tc = item_tokens > 8;
    P2P_REQUIRE(item_tokens <= kInt4TileTokens, "p2p_int4_grouped: items of up to %lld tokens, at most %d",
                (long long)item_tokens, kInt4TileTokens);
    P2P_REQUIRE(items && n_items && topk >= 1, "p2p_int4_grouped: null pointer or topk %d", topk);
    P2P_REQUIRE(aligned16(items), "p2p_int4_grouped: items must start on a 16-byte boundary");
    Int4Params p;
    if (int e = int4_params(p, "p2p_int4_grouped", x, dtype, cols, ldx, layout, has_zeros, rows, group, gated, y, ldy))
        return e;
    cudaStream_t st = as_stream(stream);
    if (tc) {
        P2P_REQUIRE(!order, "p2p_int4_grouped: items of more than 8 tokens take x in the order's places");
        P2P_REQUIRE(tc_aligned(x, ldx), "p2p_int4_grouped: items of more than 8 tokens need x rows of 16-byte alignment");
        Int4Call c = {};
        c.x = x; c.dtype = dtype; c.cols = cols; c.ldx = ldx;
        c.layout = layout; c.has_zeros = has_zeros != 0;
        c.rows = rows; c.group = group; c.gated = gated; c.y = y; c.ldy = ldy;
        c.items = items; c.n_items = n_items; c.max_items = max_items; c.item_tokens = item_tokens; c.pairs = pairs;
        c.routed = routed;
        return int4_tc_run(c, nullptr, st, "p2p_int4_grouped");
    }
    p.items = items;
    p.n_items = n_items;
    p.order = order;
    p.topk = topk;
    p.routed = routed;
    p.pairs = pairs;
    return dtype == P2P_BF16 ? run_int4<__nv_bfloat16>(p, item_tokens, max_items, st, "p2p_int4_grouped")
                             : run_int4<__half>(p, item_tokens, max_items, st, "p2p_int4_grouped");
}
