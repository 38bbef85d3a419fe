// (2d) The 4-bit product on tcgen05 tensor cores: y[t, r] = sum_c (code[r, c] - zero[r, g]) scale[r, g] x[t, c] for more
// than 32 tokens, or items of more than 32 places (int4.cu keeps the others and says why), dense or for routed experts.
//
// Scales stay out of the tensor cores: a group's sum of exact small integers times x goes to TMEM in fp32, and the
// warps that read it out multiply it by the group's scale on the way into fp32 registers, so no weight is rounded (one
// scaled weight rounded to bf16 would double the squared error of the result). A CTA, one an SM, takes a contiguous run
// of units (128 rows x 128 columns), row tile after row tile:
//
//   warps 0-3, 4-7      read the even and the odd pieces' accumulators out, group after group, acc += scale * sum (packed
//                       fp32 pairs), while other pieces multiply, and write the finished row tile: y itself,
//                       silu(gate) * up of it, or, where the tile is shared with the neighbouring run, an fp32 partial
//                       that int4_join_kernel adds in run order
//   from warp 8 (build) a warp turns the codes of one 16-row block (of two above 160 tokens) into bf16 / f16 integers and
//                       stores them into the unit's A tile in tensor memory (two tcgen05.st.16x256b.x4 a block: the
//                       layout is that store's order): 16 warps, two groups on alternate units, up to 64 tokens, where
//                       the codes' turn binds; 8 up to 160; 4 above, where the accumulators take the registers
//   weights             streams the run's records, 8.4 KB a unit and one linear range of the layout a row tile, into
//                       rings in shared memory by bulk copies (codes and zero points in one, scales, which are used
//                       later, in another), ahead of the previous kernel's end and up to 12 units ahead of their use
//   x                   TMA of each unit's x tile [tokens x 128] (two 64-column boxes, 128-byte swizzle)
//   two warps (MMA)     one thread each issues tcgen05.mma kind::f16, A from TMEM, M = 128: a group's columns times a
//                       piece of the tokens (quarters or halves) into a zeroed accumulator, then a commit. The warps take
//                       the even and the odd pieces: a look at a barrier costs an issuing thread 130 cycles even when it
//                       has nothing to wait for
//
// Measured (bf16, groups of 128): 28672 x 4096 at 272 tokens 88 us a call and 80 us replayed from a graph (724 and 794
// TFLOP/s; the product alone would take 39 us at the measured rate); 128 experts of 1536 x 2048 on 2048 x 8 tokens 240 us
// (429 TFLOP/s; items of up to 160 places, whose products are of their own places in steps of 16, their accumulators 160
// columns apart). Groups of 32 take longer, a hand-over a group: 6913 x 5119 at 33 tokens 37 us, 4096 x 14336 at 40, 160 and
// 272 tokens 45, 74 and 108. What binds is the way of a unit from hand to hand, with 130 to 220 cycles for each look at a
// barrier, and the partials and their join: with products, read-out and building all left out of a copy, 272 tokens took 60
// us of 85. A unit takes some 3,100 and 2,500 cycles where its products are 1,088 and 640: the tensor pipe is busy 37 % and
// 21 % of the time. Half of x's traffic (6 TB/s from L2) or twice the builders change nothing.
//
// Every wait is bounded (2 s, and a millisecond of tests before the clock is looked at): a launch that gives up records
// where, issues nothing more, drains what it issued and exits (p2p_int4_status reads the site, p2p_int4_withhold tests it).
#include <atomic>

#include "int4.cuh"
#include "int4_run.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace p2p {
namespace {

using namespace sm100;

constexpr int kPromoteWarps = 8;
constexpr int kBuildWarp = kPromoteWarps;               // 8..
// Warps that build one unit, and groups of them taking alternate units: up to 64 tokens the codes' turn binds; above 160
// the promoting warps' accumulators leave registers for four builders only.
constexpr int group_warps(int acc) { return acc >= 96 ? 4 : 8; }
constexpr int build_groups(int acc) { return acc <= 32 ? 2 : 1; }
constexpr int threads_of(int acc) { return (kPromoteWarps + build_groups(acc) * group_warps(acc) + 4) * 32; }
// Registers a thread of promoting, building and other warps: what the launch gives (a whole register file over the
// threads, in eights), dealt anew. 0: as launched.
constexpr int promote_regs(int acc) { return acc >= 96 ? 200 : acc >= 64 ? 136 : 0; }
constexpr int kBuildRegs = 64;
constexpr int other_regs(int acc) { return acc >= 96 ? 40 : 48; }
constexpr int dealt_regs(int acc) {
    return kPromoteWarps * 32 * promote_regs(acc) + build_groups(acc) * group_warps(acc) * 32 * kBuildRegs +
           128 * other_regs(acc);
}
constexpr int kWSlotBytes = q4::kCodeBytes + 512;       // codes and up to four groups' zero points
constexpr int kSSlotBytes = 1024;                       // up to four groups' scales
constexpr int kACols = 64;                              // TMEM columns of one unit's A tile
constexpr int kTmemCols = 512;
constexpr int kMaxW = 12, kMaxX = 8, kMaxA = 6, kMaxBuf = 4, kMaxPieces = 4;
constexpr int kSSlots = 16;                             // scales wait for the rings before them: more than W + A slots hold
constexpr int kSmemLimit = 227 * 1024 - 1024;

__device__ int g_int4_error;            // site of the first wait that gave up since the last reset (0: none)
__device__ unsigned g_int4_failed_seq;  // sequence number of the last launch in which a wait gave up

struct TcParams {
    const uint8_t* layout;
    int record, zero_bytes, scale_bytes;                // of a unit
    int out_rows, row_tiles, units, group_shift, gated; // units: 128-column steps a row tile
    int tokens, tile_tokens, token_tiles;                                         // dense
    const int32_t* items;                                                         // routed
    const int32_t* n_items;
    void* y;
    int64_t ldy;
    const int32_t* routed;              // not null: output rows from *routed to pairs become zero
    int64_t pairs;
    float* partial;                     // [ctas][2][n_max][128]; null: every CTA takes whole row tiles
    int n_max, ctas;
    int x_rows, box_rows, w_slots, x_slots, a_slots, bufs, a_col0;
    int hold;                           // a test's withheld x tile; -1: none
    uint64_t wait_ns;
    unsigned seq;
};

__device__ __forceinline__ void ld16_async(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
        "[%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// Waits for this thread's TMEM loads; r passes through so that nothing reads it earlier.
__device__ __forceinline__ void ld16_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void st16(uint32_t taddr, const uint64_t* v) {
    asm volatile(
        "{\n\t.reg .b32 r<16>;\n\t"
        "mov.b64 {r0, r1}, %1;\n\tmov.b64 {r2, r3}, %2;\n\tmov.b64 {r4, r5}, %3;\n\tmov.b64 {r6, r7}, %4;\n\t"
        "mov.b64 {r8, r9}, %5;\n\tmov.b64 {r10, r11}, %6;\n\tmov.b64 {r12, r13}, %7;\n\tmov.b64 {r14, r15}, %8;\n\t"
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {r0, r1, r2, r3, r4, r5, r6, r7, r8, r9, r10, r11, r12, r13, r14, "
        "r15};\n\t}" ::"r"(taddr),
        "l"(v[0]), "l"(v[1]), "l"(v[2]), "l"(v[3]), "l"(v[4]), "l"(v[5]), "l"(v[6]), "l"(v[7])
        : "memory");
}
// Two fp32 products and sums at once: acc.{lo,hi} += s.{lo,hi} * {lo, hi}.
__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t s, uint32_t lo, uint32_t hi) {
    asm("{\n\t.reg .b64 v;\n\tmov.b64 v, {%2, %3};\n\tfma.rn.f32x2 %0, %1, v, %0;\n\t}" : "+l"(acc) : "l"(s), "r"(lo), "r"(hi));
}
__device__ __forceinline__ float half_of(uint64_t v, int i) { return __uint_as_float((uint32_t)(v >> (32 * i))); }

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}
// Up to three barriers at once: their looks overlap.
__device__ __forceinline__ bool wait_three(uint32_t b0, uint32_t p0, uint32_t b1, uint32_t p1, uint32_t b2, uint32_t p2,
                                           bool third, int site, const WaitCtl& wc) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i) {
        const bool r0 = mbar_test(b0, p0), r1 = mbar_test(b1, p1), r2 = mbar_test(third ? b2 : b0, third ? p2 : p0);
        if (r0 && r1 && r2) return true;
    }
    return wait_one(b0, p0, site, wc) && wait_one(b1, p1, site + 1, wc) && (!third || wait_one(b2, p2, site + 2, wc));
}

__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity, int site, const WaitCtl& wc) {
    return __all_sync(0xffffffffu, wait_one(bar, parity, site, wc));
}

// A row tile of the run: its row blocks, its tokens, the steps of it that this CTA takes.
struct Tile {
    const uint8_t* records;             // its units' records
    int rt;                             // row tile within the module
    int first, n;                       // first x row (and y row), tokens
    int k0, k1;                         // steps [k0, k1) of p.units
};

__device__ __forceinline__ Tile tile_at(const TcParams& p, int u, int u1) {
    Tile t;
    const int id = u / p.units;
    t.k0 = u - id * p.units;
    t.k1 = min(p.units, t.k0 + (u1 - u));
    if (p.items) {
        const int item = id / p.row_tiles;
        t.rt = id - item * p.row_tiles;
        const int4 it = __ldcg(reinterpret_cast<const int4*>(p.items) + item);
        t.records = p.layout + ((int64_t)it.x * p.row_tiles + t.rt) * p.units * p.record;
        t.first = it.y;
        t.n = min(it.z, p.n_max);
    } else {
        t.rt = id / p.token_tiles;
        t.first = (id - t.rt * p.token_tiles) * p.tile_tokens;
        t.n = min(p.tile_tokens, p.tokens - t.first);
        t.records = p.layout + (int64_t)t.rt * p.units * p.record;
    }
    return t;
}
// Pieces of the tokens, each a multiple of 16: halves up to 160 tokens, quarters above. (An accumulator that is read out
// cannot take products: with four pieces three multiply meanwhile.)
__host__ __device__ constexpr int n_total(int n) { return (n + 15) & ~15; }
template <int PIECES> __device__ __forceinline__ int piece_size(int n, int i) {
    return (n_total(n) / 16 - i + PIECES - 1) / PIECES * 16;
}
template <int PIECES> __device__ __forceinline__ int piece_begin(int n, int i) {
    int at = 0;
#pragma unroll
    for (int k = 0; k < PIECES; ++k) at += k < i ? piece_size<PIECES>(n, k) : 0;
    return at;
}

// PIECES of the tokens; W0, W1: the most columns of a promoting warp's first and second piece, whose sums it holds in
// registers (W1 = 0: it has one).
template <typename T, int PIECES, int W0, int W1>
__global__ void __launch_bounds__(threads_of(W0 + W1), 1) int4_tc_kernel(const __grid_constant__ CUtensorMap tmap_x,
                                                              const __grid_constant__ TcParams p) {
    // The promoting warps need an accumulator of up to 144 registers and take what the others give back.
    static_assert(PIECES == 2 || (PIECES == 4 && W1 > 0), "one or two pieces for each half of the promoting warps");
    constexpr int kAcc = W0 + W1, kGroups = build_groups(kAcc), kGroupWarps = group_warps(kAcc);
    constexpr bool kSplitRegs = promote_regs(kAcc) > 0;
    constexpr bool kStaged = kAcc > 32;                  // sums leave through tensor memory
    constexpr int kWeightWarp = kBuildWarp + kGroups * kGroupWarps;
    constexpr int kXWarp = kWeightWarp + 1, kMmaWarp = kWeightWarp + 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint32_t s_tmem;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int SW = p.w_slots, SX = p.x_slots, SA = p.a_slots, NB = p.bufs;
    const uint32_t sub_bytes = (uint32_t)p.x_rows * 128u, x_bytes = 2u * sub_bytes;
    const uint32_t x_ring = base, w_ring = x_ring + SX * x_bytes, s_ring = w_ring + SW * kWSlotBytes;
    const uint32_t bars = s_ring + kSSlots * kSSlotBytes;
    auto wfull = [&](int s) { return bars + 8u * s; };
    auto wempty = [&](int s) { return bars + 8u * (kMaxW + s); };
    auto xfull = [&](int s) { return bars + 8u * (2 * kMaxW + s); };
    auto xempty = [&](int s) { return bars + 8u * (2 * kMaxW + kMaxX + s); };
    auto afull = [&](int s) { return bars + 8u * (2 * kMaxW + 2 * kMaxX + s); };
    auto aempty = [&](int s) { return bars + 8u * (2 * kMaxW + 2 * kMaxX + kMaxA + s); };
    constexpr int kDBar = 2 * kMaxW + 2 * kMaxX + 2 * kMaxA, kSBar = kDBar + 2 * kMaxBuf * kMaxPieces;
    auto dfull = [&](int piece, int b) { return bars + 8u * (kDBar + kMaxPieces * b + piece); };
    auto dempty = [&](int piece, int b) { return bars + 8u * (kDBar + kMaxPieces * (kMaxBuf + b) + piece); };
    auto sfull = [&](int s) { return bars + 8u * (kSBar + s); };
    auto sempty = [&](int s) { return bars + 8u * (kSBar + kSSlots + s); };
    const uint32_t done = bars + 8u * (kSBar + 2 * kSSlots);

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const WaitCtl wc{&g_int4_error, &g_int4_failed_seq, p.wait_ns, p.seq};
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        for (int s = 0; s < SW; ++s) { mbar_init(wfull(s), 1); mbar_init(wempty(s), kGroupWarps); }
        for (int s = 0; s < SX; ++s) { mbar_init(xfull(s), 1); mbar_init(xempty(s), 2); }
        for (int s = 0; s < SA; ++s) { mbar_init(afull(s), kGroupWarps); mbar_init(aempty(s), 2); }
        for (int b = 0; b < NB; ++b)
            for (int i = 0; i < kMaxPieces; ++i) { mbar_init(dfull(i, b), 1); mbar_init(dempty(i, b), 4); }
        for (int s = 0; s < kSSlots; ++s) { mbar_init(sfull(s), 1); mbar_init(sempty(s), kPromoteWarps); }
        mbar_init(done, 2);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == kXWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
    // The items are the previous kernel's; dense weights wait for nobody, and everything else for that kernel's end.
    if (p.items || (warp != kWeightWarp && (warp < kBuildWarp || warp >= kWeightWarp)))
        asm volatile("griddepcontrol.wait;" ::: "memory");
    const uint32_t tiles = (uint32_t)(p.items ? *p.n_items * p.row_tiles : p.row_tiles * p.token_tiles);
    const q4::Runs runs(p.partial ? tiles * (uint32_t)p.units : tiles, (uint32_t)p.ctas, p.partial ? 1u : (uint32_t)p.units);
    const int u0 = (int)runs.begin(blockIdx.x), u1 = (int)runs.begin(blockIdx.x + 1);
    const int subs = 128 >> p.group_shift;               // groups a unit
    // TMEM column of buffer b of a piece: the same for every tile, so that one piece may run ahead into the next tile
    auto d_col = [&](int piece, int b) { return (uint32_t)(b * p.n_max + piece_begin<PIECES>(p.n_max, piece)); };

    if (warp >= kWeightWarp) {
        if (kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(other_regs(kAcc)));
        if (warp == kWeightWarp) {
            if (elect_one()) {
                int slot = 0, ss = 0, used = 0;
                uint32_t ph = 0, phs = 0;
                bool ok = true;
                const uint32_t w_bytes = (uint32_t)(q4::kCodeBytes + p.zero_bytes);
                for (int u = u0; u < u1 && ok;) {
                    const Tile t = tile_at(p, u, u1);
                    const uint8_t* src = t.records + (int64_t)t.k0 * p.record;
                    for (int k = t.k0; k < t.k1; ++k, src += p.record) {
                        if (used >= SW && !(ok = wait_one(wempty(slot), ph ^ 1u, 1, wc))) break;
                        if (used >= kSSlots && !(ok = wait_one(sempty(ss), phs ^ 1u, 12, wc))) break;
                        mbar_expect_tx(wfull(slot), w_bytes);
                        bulk_load(w_ring + slot * kWSlotBytes, src, w_bytes, wfull(slot));
                        mbar_expect_tx(sfull(ss), (uint32_t)p.scale_bytes);
                        bulk_load(s_ring + ss * kSSlotBytes, src + w_bytes, (uint32_t)p.scale_bytes, sfull(ss));
                        ++used;
                        advance(slot, ph, 1, SW);
                        advance(ss, phs, 1, kSSlots);
                    }
                    u += t.k1 - t.k0;
                }
                // every copy issued must have landed before the CTA may exit: each slot's last one
                for (int i = max(0, used - SW); i < used; ++i) mbar_drain(wfull(i % SW), (uint32_t)((i / SW) & 1), 2, wc);
                for (int i = max(0, used - kSSlots); i < used; ++i)
                    mbar_drain(sfull(i % kSSlots), (uint32_t)((i / kSSlots) & 1), 2, wc);
            }
            __syncwarp();
        } else if (warp == kXWarp) {
            if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmap_x)) : "memory");
            if (elect_one()) {
                int slot = 0, used = 0;
                uint32_t ph = 0;
                bool ok = true;
                for (int u = u0; u < u1 && ok;) {
                    const Tile t = tile_at(p, u, u1);
                    const int boxes = (n_total(t.n) + p.box_rows - 1) / p.box_rows;
                    for (int k = t.k0; k < t.k1; ++k) {
                        if (!(ok = used != p.hold)) break;           // a test withholds this load
                        if (used >= SX && !(ok = wait_one(xempty(slot), ph ^ 1u, 3, wc))) break;
                        mbar_expect_tx(xfull(slot), (uint32_t)(2 * boxes * p.box_rows) * 128u);
                        for (int b = 0; b < boxes; ++b)
#pragma unroll
                            for (int s = 0; s < 2; ++s)
                                tma_load_2d(x_ring + slot * x_bytes + s * sub_bytes + b * p.box_rows * 128, &tmap_x,
                                            k * 128 + s * 64, t.first + b * p.box_rows, xfull(slot));
                        ++used;
                        advance(slot, ph, 1, SX);
                    }
                    u += t.k1 - t.k0;
                }
                for (int i = max(0, used - SX); i < used; ++i) mbar_drain(xfull(i % SX), (uint32_t)((i / SX) & 1), 4, wc);
            }
            __syncwarp();
        } else {
            const int h = warp - kMmaWarp;
            if (elect_one()) {
                int sa = 0, sx = 0, sb = 0, jobs = 0;
                uint32_t pha = 0, phx = 0, phb = 0;
                bool ok = true;
                const uint64_t x_desc = sw128_desc(x_ring);
                const uint32_t d0 = tmem + d_col(h, 0), d1 = tmem + d_col(h + 2, 0);
                // one unit: SUBS groups of 8 / SUBS products of K = 16 for each of this warp's pieces
                auto unit = [&](auto subs_, uint32_t id0, uint32_t id1, uint32_t row0, uint32_t row1) {
                    constexpr int SUBS = decltype(subs_)::value, STEPS = 8 / SUBS;
                    const uint32_t a = tmem + (uint32_t)(p.a_col0 + sa * kACols);
                    const uint64_t b0 = x_desc + (uint64_t)((uint32_t)(sx * x_bytes) >> 4);
                    const uint64_t b1 = b0 + (uint64_t)(sub_bytes >> 4);
#pragma unroll
                    for (int s = 0; s < SUBS; ++s) {
                        if (s == 0) {
                            if (!(ok = wait_three(afull(sa), pha, xfull(sx), phx, dempty(h, sb), phb ^ 1u, jobs >= NB, 5, wc)))
                                return;
                        } else {
                            if (jobs >= NB && !(ok = wait_one(dempty(h, sb), phb ^ 1u, 7, wc))) return;
                        }
                        tc_fence_after();
                        auto piece = [&](uint32_t d, uint32_t row, uint32_t id) {
                            if (id == 0) return;
#pragma unroll
                            for (int k = 0; k < STEPS; ++k) {
                                const int kk = s * STEPS + k;
                                umma_f16_ts(d, a + 8u * kk, (kk < 4 ? b0 : b1) + row + 2 * (kk & 3), id, k ? 1u : 0u);
                            }
                        };
                        piece(d0 + sb * p.n_max, row0, id0);
                        umma_commit(dfull(h, sb));
                        if constexpr (PIECES == 4) {
                            if (jobs >= NB && !(ok = wait_one(dempty(h + 2, sb), phb ^ 1u, 7, wc))) return;
                            tc_fence_after();
                            piece(d1 + sb * p.n_max, row1, id1);
                            umma_commit(dfull(h + 2, sb));
                        }
                        ++jobs;
                        advance(sb, phb, 1, NB);
                    }
                };
                for (int u = u0; u < u1 && ok;) {
                    const Tile t = tile_at(p, u, u1);
                    const int n0 = piece_size<PIECES>(t.n, h), n1 = PIECES == 4 ? piece_size<PIECES>(t.n, h + 2) : 0;
                    const uint32_t id0 = n0 > 0 ? idesc_f16<T>(n0) : 0u, id1 = n1 > 0 ? idesc_f16<T>(n1) : 0u;
                    const uint32_t row0 = (uint32_t)(piece_begin<PIECES>(t.n, h) * 128) >> 4;
                    const uint32_t row1 = (uint32_t)(piece_begin<PIECES>(t.n, h + 2) * 128) >> 4;
                    for (int k = t.k0; k < t.k1; ++k) {
                        if (subs == 1) unit(std::integral_constant<int, 1>(), id0, id1, row0, row1);
                        else if (subs == 2) unit(std::integral_constant<int, 2>(), id0, id1, row0, row1);
                        else unit(std::integral_constant<int, 4>(), id0, id1, row0, row1);
                        if (!ok) break;
                        umma_commit(aempty(sa));
                        umma_commit(xempty(sx));
                        advance(sa, pha, 1, SA);
                        advance(sx, phx, 1, SX);
                    }
                    u += t.k1 - t.k0;
                }
                umma_commit(done);
                mbar_drain(done, 0, 8, wc);              // both issuers' products complete before TMEM is freed
            }
            __syncwarp();
        }
    } else if (warp >= kBuildWarp) {
        if (kSplitRegs) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kBuildRegs));
        const int group = (warp - kBuildWarp) / kGroupWarps, w = (warp - kBuildWarp) % kGroupWarps;
        constexpr int kBlocks = 8 / kGroupWarps;                                // row blocks a warp builds
        const int blk0 = 2 * (w & 3) + (kBlocks == 1 ? w >> 2 : 0);             // lanes 32 (w % 4).. are this warp's
        int sw = group, sa = group, used = group;
        uint32_t phw = 0, pha = 0;
        bool ok = true;
        q4::Codes<T> codes;
        codes.zeros(8u, 8u);
        for (int u = u0 + group; u < u1 && ok; u += kGroups) {
            {
                if (!(ok = wait_all(wfull(sw), phw, 9, wc))) break;
                const uint32_t rec = w_ring + sw * kWSlotBytes;
                if (used >= SA && !(ok = wait_all(aempty(sa), pha ^ 1u, 10, wc))) break;
                tc_fence_after();
#pragma unroll
                for (int i = 0; i < 2 * kBlocks; ++i) {
                    const int blk = blk0 + i / 2, half = i & 1;
                    const uint4 c = lds_v4(rec + (blk * 2 + half) * q4::kBlockBytes + lane * 16);
                    const uint32_t words[4] = {c.x, c.y, c.z, c.w};
                    // this column block's groups: one holds it, or (32 columns) two do
                    auto zeros = [&](int g) {
                        if (p.zero_bytes) {
                            const uint32_t z = lds_u16(rec + q4::kCodeBytes + ((g * 8 + blk) * 8 + (lane >> 2)) * 2);
                            codes.zeros(z & 15u, z >> 8);
                        }
                    };
                    zeros(p.group_shift == 5 ? 2 * half : p.group_shift == 6 ? half : 0);
                    uint32_t r[16];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (k == 2 && p.group_shift == 5) zeros(2 * half + 1);
                        uint32_t a[4];
                        codes.expand(words[k], a);
                        r[4 * k] = a[0]; r[4 * k + 1] = a[2]; r[4 * k + 2] = a[1]; r[4 * k + 3] = a[3];
                    }
                    const uint32_t col = (uint32_t)(p.a_col0 + sa * kACols + half * 32);
                    tmem_st_16x256b_x4(tmem + ((uint32_t)(16 * blk) << 16) + col, r);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(wempty(sw));
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(afull(sa));
                used += kGroups;
                advance(sw, phw, kGroups, SW);
                advance(sa, pha, kGroups, SA);
            }
        }
    } else {
        if constexpr (kSplitRegs) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(promote_regs(kAcc)));
        const int h = warp >> 2, q = warp & 3, row_in = 32 * q + lane;
        T* y = reinterpret_cast<T*>(p.y);
        const uint32_t scale_at = (uint32_t)(((row_in >> 4) * 8 + (row_in & 7)) * 2 + ((row_in >> 3) & 1)) * 2u;
        const uint32_t lanes = tmem + ((uint32_t)(32 * q) << 16);
        const uint32_t d_at[2] = {lanes + d_col(h, 0), lanes + d_col(h + 2, 0)};
        int sb = 0, ss = 0;
        uint32_t phb = 0, phs = 0;
        bool ok = true;
        for (int u = u0; u < u1 && ok;) {
            const Tile t = tile_at(p, u, u1);
            const int size[2] = {piece_size<PIECES>(t.n, h), W1 ? piece_size<PIECES>(t.n, h + 2) : 0};
            uint64_t acc[(W0 + W1) / 2];
#pragma unroll
            for (int i = 0; i < (W0 + W1) / 2; ++i) acc[i] = 0;
            // one group of the run's next unit; the tile's last sums are kept for the way out
            int sub = 0;
            auto step = [&](auto kept) {
                if (sub == 0 && !(ok = wait_all(sfull(ss), phs, 13, wc))) return;
                const uint16_t bits = (uint16_t)lds_u16(s_ring + ss * kSSlotBytes + sub * 256 + scale_at);
                uint64_t s2;
                asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "r"(__float_as_uint(to_f32(*reinterpret_cast<const T*>(&bits)))));
                auto promote = [&](auto which) {
                    constexpr int I = decltype(which)::value, kWidth = I ? W1 : W0;
                    const int piece = h + 2 * I;
                    if (!ok || !(ok = wait_all(dfull(piece, sb), phb, 11, wc))) return;
                    tc_fence_after();
                    const uint32_t d = d_at[I] + sb * p.n_max;
#pragma unroll
                    for (int c = 0; c < kWidth / 16; ++c) {
                        if (c * 16 < size[I]) {
                            uint32_t v[16];
                            ld16_async(d + c * 16, v);
                            ld16_wait(v);
#pragma unroll
                            for (int e = 0; e < 8; ++e) fma2(acc[I * W0 / 2 + c * 8 + e], s2, v[2 * e], v[2 * e + 1]);
                        }
                    }
                    if constexpr (!decltype(kept)::value) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(dempty(piece, sb));
                    }
                };
                promote(std::integral_constant<int, 0>());
                if constexpr (W1 > 0) promote(std::integral_constant<int, 1>());
                if constexpr (!decltype(kept)::value) advance(sb, phb, 1, NB);
                if (++sub == subs) {
                    sub = 0;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(sempty(ss));
                    advance(ss, phs, 1, kSSlots);
                }
            };
#pragma unroll 1
            for (int jobs = (t.k1 - t.k0) * subs - 1; jobs > 0 && ok; --jobs) step(std::false_type());
            const bool whole = t.k1 - t.k0 == p.units;
            if (ok) {
                if (kStaged && whole) step(std::integral_constant<bool, kStaged>());
                else step(std::false_type());
            }
            if (!ok) break;
            if (!whole) {                                // shared with the neighbouring run: all of the piece's columns
                float* part = p.partial + ((int64_t)blockIdx.x * 2 + (u == u0 ? 0 : 1)) * p.n_max * 128 + row_in;
                auto leave = [&](auto which) {
                    constexpr int I = decltype(which)::value, kWidth = I ? W1 : W0;
                    float* at = part + piece_begin<PIECES>(t.n, h + 2 * I) * 128;
#pragma unroll
                    for (int c0 = 0; c0 < kWidth; c0 += 16) {
                        if (c0 < size[I]) {
#pragma unroll
                            for (int c = c0; c < c0 + 16; ++c) at[c * 128] = half_of(acc[I * W0 / 2 + c / 2], c & 1);
                        }
                    }
                };
                leave(std::integral_constant<int, 0>());
                if constexpr (W1 > 0) leave(std::integral_constant<int, 1>());
            } else if constexpr (!kStaged) {
                auto store = [&](auto which) {
                    constexpr int I = decltype(which)::value, kWidth = I ? W1 : W0, kAt = I * W0 / 2;
                    const int col0 = piece_begin<PIECES>(t.n, h + 2 * I);
                    const int left = min(size[I], t.n - col0);                               // this piece's tokens
                    if (p.gated) {
                        // even row blocks are gates, odd ones the same units' ups: lanes i and i + 16 of a warp. Each pair
                        // of lanes exchanges one of two columns and finishes the other.
                        const int row = t.rt * 64 + 16 * q + (lane & 15);
                        T* out = y + (int64_t)(t.first + col0 + (lane >> 4)) * p.ldy + row;
#pragma unroll
                        for (int c = 0; c < kWidth; c += 2) {
                            if (c >= left) continue;
                            const float even = half_of(acc[kAt + c / 2], 0), odd = half_of(acc[kAt + c / 2], 1);
                            const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? odd : even, 16);
                            const float gate = lane < 16 ? even : other, up = lane < 16 ? other : odd;
                            if (c + (lane >> 4) < left && row < p.out_rows)
                                out[c * p.ldy] = from_f32<T>(gate / (1.f + expf(-gate)) * up);
                        }
                    } else {
                        const int row = t.rt * 128 + row_in;
                        if (row < p.out_rows) {
                            T* out = y + (int64_t)(t.first + col0) * p.ldy + row;
#pragma unroll
                            for (int c = 0; c < kWidth; ++c)
                                if (c < left) out[c * p.ldy] = from_f32<T>(half_of(acc[kAt + c / 2], c & 1));
                        }
                    }
                };
                store(std::integral_constant<int, 0>());
            } else {
                // The way out, through the accumulator just read: a loop over 16 columns at a time. (Straight from the
                // registers every column would be code of its own, fetched anew each time: 21,000 cycles a row tile of 272
                // tokens.)
                auto stage = [&](auto which) {
                    constexpr int I = decltype(which)::value, kWidth = I ? W1 : W0;
#pragma unroll
                    for (int c = 0; c < kWidth / 16; ++c)
                        if (c * 16 < size[I]) st16(d_at[I] + sb * p.n_max + c * 16, acc + I * W0 / 2 + c * 8);
                };
                stage(std::integral_constant<int, 0>());
                if constexpr (W1 > 0) stage(std::integral_constant<int, 1>());
                tmem_wait_st();
#pragma unroll 1
                for (int i = 0; i < (W1 > 0 ? 2 : 1); ++i) {
                    const int piece = h + 2 * i, col0 = piece_begin<PIECES>(t.n, piece), n = i ? size[1] : size[0];
                    const int left = min(n, t.n - col0);     // this piece's tokens
                    const uint32_t d = (i ? d_at[1] : d_at[0]) + sb * p.n_max;
#pragma unroll 1
                    for (int c0 = 0; c0 < n; c0 += 16) {
                        uint32_t v[16];
                        ld16_async(d + c0, v);
                        ld16_wait(v);
                        if (p.gated) {
                            // even row blocks are gates, odd ones the same units' ups: lanes i and i + 16 of a warp. Each
                            // pair of lanes exchanges one of two columns and finishes the other.
                            const int row = t.rt * 64 + 16 * q + (lane & 15);
                            T* out = y + (int64_t)(t.first + col0 + c0 + (lane >> 4)) * p.ldy + row;
#pragma unroll
                            for (int c = 0; c < 16; c += 2) {
                                const uint32_t other = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[c + 1] : v[c], 16);
                                const float gate = __uint_as_float(lane < 16 ? v[c] : other);
                                const float up = __uint_as_float(lane < 16 ? other : v[c + 1]);
                                if (c0 + c + (lane >> 4) < left && row < p.out_rows)
                                    out[c * p.ldy] = from_f32<T>(gate / (1.f + expf(-gate)) * up);
                            }
                        } else {
                            const int row = t.rt * 128 + row_in;
                            T* out = y + (int64_t)(t.first + col0 + c0) * p.ldy + row;
                            if (row < p.out_rows) {
#pragma unroll
                                for (int c = 0; c < 16; ++c)
                                    if (c0 + c < left) out[c * p.ldy] = from_f32<T>(__uint_as_float(v[c]));
                            }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(dempty(piece, sb));
                }
                advance(sb, phb, 1, NB);
            }
            u += t.k1 - t.k0;
        }
        if (p.routed) {                                  // what lies behind the last pair
            for (int64_t r = *p.routed + blockIdx.x; r < p.pairs; r += p.ctas)
                for (int c = threadIdx.x; c < p.out_rows; c += kPromoteWarps * 32) y[r * p.ldy + c] = from_f32<T>(0.f);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kXWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// Row tiles that several runs share: their fp32 partials added in run order. A block takes a row tile and 32 tokens, a
// warp a token at a time, a thread four rows.
constexpr int kJoinTokens = 32;
template <typename T> __global__ void __launch_bounds__(256) int4_join_kernel(const __grid_constant__ TcParams p) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const q4::Runs runs((uint32_t)(p.row_tiles * p.token_tiles * p.units), (uint32_t)p.ctas, 1u);
    const uint32_t a = blockIdx.x * (uint32_t)p.units, b0 = runs.of(a), b1 = runs.of(a + p.units - 1);
    // Every block waits, those without work too: this kernel's end stands for the end of the one before.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (b0 == b1) return;                                // one run wrote y itself
    const Tile t = tile_at(p, (int)a, (int)a + p.units);
    const int lane = threadIdx.x & 31, last = min(t.n, (int)(blockIdx.y + 1) * kJoinTokens);
    // the tile is run b0's last row tile, unless b0 begins with it, and every other run's first
    const float* part = p.partial + ((int64_t)b0 * 2 + (runs.begin(b0) >= a ? 0 : 1)) * p.n_max * 128 + lane * 4;
    const float* next = p.partial + (int64_t)(b0 + 1) * 2 * p.n_max * 128 + lane * 4;
    T* y = reinterpret_cast<T*>(p.y);
#pragma unroll 2
    for (int tok = blockIdx.y * kJoinTokens + (threadIdx.x >> 5); tok < last; tok += 8) {
        float4 sum = __ldcg(reinterpret_cast<const float4*>(part + (int64_t)tok * 128));
#pragma unroll 4
        for (uint32_t b = b0 + 1; b <= b1; ++b) {
            const float4 v = __ldcg(reinterpret_cast<const float4*>(next + ((int64_t)(b - b0 - 1) * 2 * p.n_max + tok) * 128));
            sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
        }
        T* out = y + (int64_t)(t.first + tok) * p.ldy;
        const float mine[4] = {sum.x, sum.y, sum.z, sum.w};
        if (p.gated) {                                   // lanes 8 i .. + 3 hold gates, + 4 .. + 7 their ups
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float up = __shfl_xor_sync(0xffffffffu, mine[c], 4);
                const int row = t.rt * 64 + (lane >> 3) * 16 + (lane & 3) * 4 + c;
                if (!(lane & 4) && row < p.out_rows) out[row] = from_f32<T>(mine[c] / (1.f + expf(-mine[c])) * up);
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

// What a launch of at most `most` tokens a tile takes: accumulator columns, rings.
struct TcPlan {
    int n_max, x_rows, box_rows, bufs, a_col0, a_slots, x_slots, w_slots, smem;
};

TcPlan plan_tc(int most, bool routed) {
    TcPlan pl;
    const int total = n_total(most);
    pl.n_max = total;
    pl.x_rows = total;
    // a routed item's x rows end anywhere: boxes of 16 rows follow it; a dense tile is one box, or two above 256 rows
    pl.box_rows = routed ? 16 : total <= 256 ? total : total / 2;
    pl.bufs = kMaxBuf;                                   // accumulators in turn, as far as two A tiles leave room
    while (pl.bufs > 1 && pl.bufs * total + (pl.bufs > 2 ? 4 : 2) * kACols > kTmemCols) --pl.bufs;
    pl.a_col0 = (pl.bufs * total + 31) / 32 * 32;
    pl.a_slots = (kTmemCols - pl.a_col0) / kACols;
    if (pl.a_slots > kMaxA) pl.a_slots = kMaxA;
    const int x_bytes = 2 * pl.x_rows * 128;
    const int barriers = 2 * kMaxW + 2 * kMaxX + 2 * kMaxA + 2 * kMaxBuf * kMaxPieces + 2 * kSSlots + 1;
    const int fixed = 1024 + kSSlots * kSSlotBytes + 8 * barriers;
    // eight units of weights in flight at least, then x, then as much again as is left for weights
    pl.x_slots = (kSmemLimit - fixed - 8 * kWSlotBytes) / x_bytes;
    if (pl.x_slots > kMaxX) pl.x_slots = kMaxX;
    pl.w_slots = (kSmemLimit - fixed - pl.x_slots * x_bytes) / kWSlotBytes;
    if (pl.w_slots > kMaxW) pl.w_slots = kMaxW;
    pl.smem = fixed + pl.x_slots * x_bytes + pl.w_slots * kWSlotBytes;
    return pl;
}

template <typename T, int PIECES, int W0, int W1>
int launch_tc(const CUtensorMap& map, const TcParams& p, int smem, cudaStream_t st, const char* what) {
    auto kernel = int4_tc_kernel<T, PIECES, W0, W1>;
    constexpr int kThreads = threads_of(W0 + W1);
    if (int e = allow_smem((const void*)kernel, smem, what)) return e;
    if (promote_regs(W0 + W1) > 0) {                     // the register split needs what it was written for
        static std::atomic<int> regs{0};
        if (regs == 0) {
            cudaFuncAttributes a;
            if (cudaFuncGetAttributes(&a, kernel) != cudaSuccess)
                return fail(P2P_ECUDA, "%s: %s", what, cudaGetErrorString(cudaGetLastError()));
            regs = a.numRegs;
        }
        if (regs * kThreads < dealt_regs(W0 + W1))
            return fail(P2P_EUNSUPPORTED, "%s: built with %d registers a thread for %d in all", what, regs.load(),
                        dealt_regs(W0 + W1));
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)p.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, kernel, map, p);
    if (int e = launch_status(what)) return e;
    if (!p.partial) return P2P_OK;
    cfg.gridDim = dim3((unsigned)(p.row_tiles * p.token_tiles), (unsigned)((p.tile_tokens + kJoinTokens - 1) / kJoinTokens));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    cudaLaunchKernelEx(&cfg, int4_join_kernel<T>, p);
    return launch_status(what);
}

template <typename T>
int launch_width(const CUtensorMap& map, const TcParams& p, int smem, cudaStream_t st, const char* what) {
    if (p.n_max <= 64) return launch_tc<T, 2, 32, 0>(map, p, smem, st, what);
    if (p.n_max <= 128) return launch_tc<T, 2, 64, 0>(map, p, smem, st, what);
    if (p.n_max <= 160) return launch_tc<T, 2, 80, 0>(map, p, smem, st, what);
    if (p.n_max <= 192) return launch_tc<T, 4, 48, 48>(map, p, smem, st, what);
    return launch_tc<T, 4, 80, 64>(map, p, smem, st, what);
}

// Token tiles of a dense call: as even as they divide, at most 272 tokens each.
int64_t token_tiles(int64_t tokens) { return (tokens + kInt4TileTokens - 1) / kInt4TileTokens; }
int tile_tokens(int64_t tokens) {
    const int64_t n = token_tiles(tokens);
    return (int)((tokens + n - 1) / n);
}
// CTAs of a dense call, and whether they split row tiles: not where whole tiles leave at most a tenth of them idle.
int dense_ctas(int64_t tiles, int64_t units, bool* split) {
    const int64_t sms = sm_count(), waves = (tiles + sms - 1) / sms;
    *split = waves * sms * 10 > tiles * 11;
    const int64_t most = *split ? tiles * units : tiles;
    return (int)(most < sms ? most : sms);
}

}  // namespace

size_t int4_tc_workspace(int64_t tokens, int64_t rows, int64_t cols, int gated) {
    const int64_t row_tiles = q4::row_tiles(rows, gated), units = q4::div_up(cols, q4::kUnitCols);
    bool split;
    const int ctas = dense_ctas(row_tiles * token_tiles(tokens), units, &split);
    if (!split) return 0;
    return (size_t)ctas * 2 * ((tile_tokens(tokens) + 15) / 16 * 16) * 128 * sizeof(float);
}

int int4_tc_run(const Int4Call& c, void* workspace, cudaStream_t st, const char* what) {
    TcParams p = {};
    const bool routed = c.items != nullptr;
    const int most = routed ? (int)c.item_tokens : tile_tokens(c.tokens);
    const TcPlan pl = plan_tc(most, routed);
    p.layout = reinterpret_cast<const uint8_t*>(c.layout);
    p.record = q4::unit_bytes(c.group, c.has_zeros);
    p.zero_bytes = q4::unit_zero_bytes(c.group, c.has_zeros);
    p.scale_bytes = q4::unit_scale_bytes(c.group);
    p.out_rows = (int)(c.gated ? c.rows / 2 : c.rows);
    p.row_tiles = (int)q4::row_tiles(c.rows, c.gated);
    p.units = (int)q4::div_up(c.cols, q4::kUnitCols);
    p.group_shift = c.group == 32 ? 5 : c.group == 64 ? 6 : 7;
    p.gated = c.gated;
    p.tokens = (int)c.tokens;
    p.tile_tokens = routed ? most : tile_tokens(c.tokens);
    p.token_tiles = routed ? 1 : (int)token_tiles(c.tokens);
    p.items = c.items;
    p.n_items = c.n_items;
    p.routed = c.routed;
    p.pairs = c.pairs;
    p.y = c.y;
    p.ldy = c.ldy;
    p.n_max = pl.n_max;
    bool split = false;
    if (routed) {
        const int64_t tiles = c.max_items * p.row_tiles;
        p.ctas = (int)(tiles < sm_count() ? tiles : sm_count());
    } else {
        p.ctas = dense_ctas((int64_t)p.row_tiles * p.token_tiles, p.units, &split);
    }
    p.partial = split ? reinterpret_cast<float*>(workspace) : nullptr;
    const int64_t tiles = (int64_t)p.row_tiles * (routed ? c.max_items : p.token_tiles);
    if (tiles * p.units > 0x7fffffff || tiles > 0x7fffffff / 2)
        return fail(P2P_EUNSUPPORTED, "%s: %lld units of 128 x 128 weights, below 2^31", what, (long long)(tiles * p.units));
    p.x_rows = pl.x_rows;
    p.box_rows = pl.box_rows;
    p.w_slots = pl.w_slots;
    p.x_slots = pl.x_slots;
    p.a_slots = pl.a_slots;
    p.bufs = pl.bufs;
    p.a_col0 = pl.a_col0;
    p.hold = c.hold;
    p.wait_ns = c.wait_ns;
    p.seq = next_seq();
    CUtensorMap map;
    if (int e = encode_x_map(&map, c.x, c.dtype, routed ? c.pairs : c.tokens, c.cols, c.ldx, pl.box_rows)) return e;
    return c.dtype == P2P_BF16 ? launch_width<__nv_bfloat16>(map, p, pl.smem, st, what)
                               : launch_width<__half>(map, p, pl.smem, st, what);
}

int int4_tc_error(int* site, int reset, cudaStream_t st) {
    if (cudaMemcpyFromSymbolAsync(site, g_int4_error, sizeof(int), 0, cudaMemcpyDeviceToHost, st) != cudaSuccess ||
        cudaStreamSynchronize(st) != cudaSuccess)
        return fail(P2P_ECUDA, "p2p_int4_status: %s", cudaGetErrorString(cudaGetLastError()));
    if (reset && *site) {
        const int zero = 0;
        cudaMemcpyToSymbolAsync(g_int4_error, &zero, sizeof(int), 0, cudaMemcpyHostToDevice, st);
        cudaStreamSynchronize(st);
    }
    return P2P_OK;
}

}  // namespace p2p
