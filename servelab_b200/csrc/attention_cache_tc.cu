// Attention over a paged cache in bfloat16 or 8 bits for many query rows a kv head (trees of drafted tokens, portions of
// prompts) on the 5th-generation tensor cores, bfloat16 queries, head sizes 64 and 128, any page size.
//
// Work unit: (128 query rows of a request, kv head, share of the keys).  Per 64 keys, accumulators in tensor memory:
//
//   loader warps   rows of the pages: bfloat16 by asynchronous 16-byte copies, codes through registers, where they become
//                  float16 (cache_codes.cuh), into two-stage rings in the 128-byte swizzle        -> k_full, v_full
//   MMA warp       S = Q.K^T   (M=128 N=64, K=16 x D/16)                                          -> s_full
//                  O += P.V    (M=128 N=D,  K=16 x 4)                                             -> pv_done
//   softmax warps  32 rows each: 64 scores times their keys' scales, running maximum and sum in float32, probabilities times
//                  the values' scales in 16 bits back to tensor memory; four rows a lane where all keys are seen, a row a
//                  lane and a mask where not, where scores are huge or query rows have factors of their own   -> p_full
//
// A scout warp runs ahead of the loaders: it looks pages up, asks for their rows and brings the scales.
// Scores are double buffered.  A barrier is one of a pair indexed by the tile's parity.  The running maximum is only raised
// when it is exceeded by 2^8.  int8 codes come out in the order 0, 2, 1, 3: the queries are laid out so too, and the columns of O
// are put back when they are stored.
//
// Few tiles leave SMs idle: then blocks (`parts`, or one more) share a tile's keys and a second kernel adds their results up.
// (Through the shared memory of a cluster of eight that took 7,500 cycles a block, and clusters left half of the SMs' places empty.)
//
// What bounds it: the chain of the roles.  A tile takes 3,700 cycles with two blocks an SM, whose issue slots are busy to 53 % and
// tensor pipe to 24 %; a block's start (tile, pages, queries, first keys) takes 7,500.  28 heads over 4 of 128: two portions of 257
// tokens over 2,043 keys in int8 40.2 us, eight trees of 32 drafts over 2,040 keys 28.2, one of 64 over 16,380 keys in bfloat16 32.4.
//
// Over a bfloat16 cache probabilities are rounded to bfloat16 (both operands of a product have one type): at most 2^-8 of a weight;
// the last case is 2.3e-3 of its results' size away from 64 bits, where rounding the results alone makes 1.7e-3.
//
// Every wait is bounded; a role that gives up sets the status word and leaves its loop, the block frees its tensor memory
// and has no result (its part: NaN).
#include <cuda.h>

#include "cache_codes.cuh"
#include "mma_util.cuh"
#include "softmax_util.cuh"
#include "umma_util.cuh"

#if (SLB_HEAD_DIM != 64 && SLB_HEAD_DIM != 128)
#error "compile with -DSLB_HEAD_DIM=64 or 128"
#endif

SLB_DEFINE_STATUS_WORD(cache_tc_status, slb_cache_attention_tc_status)

namespace {

using namespace slb_umma;

constexpr int D = SLB_HEAD_DIM;
constexpr int PANELS = D / 64;                 // 64-element (128-byte) column panels
constexpr int BM = 128, BN = 64;
constexpr int SOFTMAX_WARPS = 4, LOADER_WARPS = 4, MMA_WARP = SOFTMAX_WARPS + LOADER_WARPS, SCOUT_WARP = MMA_WARP + 1;
constexpr int THREADS = 32 * (SCOUT_WARP + 1);
constexpr int TMEM_COLS = 256;                 // two score buffers at columns 0 and 64, O from 128 on
constexpr int O_COL = 128;
constexpr int Q_PANEL = BM * 128, KV_PANEL = BN * 128, KV_TILE = PANELS * KV_PANEL;
constexpr int OFF_K = PANELS * Q_PANEL;
constexpr int OFF_V = OFF_K + 2 * KV_TILE;
constexpr int AHEAD = 8;                       // tiles whose rows and scales the scout may know
constexpr int OFF_SCALE = OFF_V + 2 * KV_TILE;         // [AHEAD][SCALES][BN] floats: keys' scales, values', log2 of the values'
constexpr int SCALES = 3;
constexpr int OFF_ROW = OFF_SCALE + AHEAD * SCALES * BN * 4;   // [AHEAD][BN] cache rows, -1: none
constexpr int OFF_LOG = OFF_ROW + AHEAD * BN * 4;      // [AHEAD] log2 of a power of two above a tile's value scales
constexpr int OFF_BAR = OFF_LOG + AHEAD * 4;
constexpr int OFF_TOP = OFF_BAR + 320;                 // [BM] largest magnitude of each row of the queries, 16 bits
constexpr int OFF_SPREAD = OFF_TOP + 2 * BM;           // [MMA_WARP] largest and least of what a warp stages, 16 bits each
constexpr int OFF_FIELD = OFF_SPREAD + 4 * MMA_WARP;   // the queries' factor
constexpr size_t SMEM = OFF_FIELD + 16;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_THRESHOLD = 8.f;       // log2 of the largest probability tolerated
// References up to here go with scores in one multiply-add.  It takes the product as it is and the reference as the product
// that was rounded: an exponent is off by up to half a unit in the last place, 2^-5 here, but 128 and more from 2^31 on.
constexpr float FUSED_REFERENCE = 1048576.f;

__device__ __forceinline__ void gave_up(int code) {
    if ((threadIdx.x & 31) == 0) atomicCAS(&cache_tc_status, 0, code);
}

// The step's `unit`-th tile of 128 rows (requests in order): its request, first row and what the request's arrays say, found
// by a warp, whose lanes look at a request each; s = -1: no such tile.
struct Tile {
    int s, row0, q0, q_len, ctx;
};
__device__ __forceinline__ Tile find_tile(const CacheAttnArgs& a, int g, int unit) {
    const int lane = threadIdx.x & 31;
    Tile t = {-1, 0, 0, 0, 0};
    int before = 0;
    int i = min(lane, a.S - 1), from = a.cu_q[i], to = a.cu_q[i + 1], ctx = a.ctx_len[i];
    for (int s0 = 0; s0 < a.S; s0 += 32) {
        clamp_span(a.T, from, to);
        const int n = s0 + lane < a.S ? (int)(((long long)(to - from) * g + BM - 1) / BM) : 0;
        const int q0 = from, q_len = to - from, c = ctx;
        if (s0 + 32 < a.S) {                                // (the next 32 are on their way meanwhile)
            i = min(s0 + 32 + lane, a.S - 1);
            from = a.cu_q[i];
            to = a.cu_q[i + 1];
            ctx = a.ctx_len[i];
        }
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + upto > unit);
        if (past != 0) {
            const int l = __ffs(past) - 1;
            t.s = s0 + l;
            t.row0 = (unit - before - __shfl_sync(0xffffffffu, upto - n, l)) * BM;
            t.q0 = __shfl_sync(0xffffffffu, q0, l);
            t.q_len = __shfl_sync(0xffffffffu, q_len, l);
            t.ctx = __shfl_sync(0xffffffffu, c, l);
            return t;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return t;
}

// Bits 0 .. 63 of the keys k0 .. k0 + 63 that a row sees (kend: behind the last key of the tile's rows).
__device__ __forceinline__ unsigned long long seen_keys(const CacheAttnArgs& a, const RowView& r, int k0, int kend, int base, int q0) {
    auto below = [](int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull; };     // bits 0 .. n - 1
    if (r.bits == nullptr) return below(min(kend, r.hi + 1) - k0) & ~below(r.lo - k0);
    unsigned long long m = below(min(kend, base) - k0) & ~below(r.lo - k0);
    const int j0 = k0 - base;                          // drafted token of bit 0 (may be negative)
    unsigned long long drafts = 0;
    for (int w = max(0, j0 >> 5); w < a.mask_words && 32 * w < j0 + 64; ++w) {
        const unsigned long long word = (unsigned)r.bits[w];
        const int at = 32 * w - j0;                    // bit that the word's first token has, -31 .. 63 + 31
        drafts |= at >= 0 ? word << at : word >> -at;
    }
    drafts &= below(kend - k0) & ~below(base - k0);
    if (a.window > 0) {
        for (unsigned long long left = drafts; left != 0; left &= left - 1) {
            const int i = __ffsll((long long)left) - 1;
            if (r.pos - a.pos[q0 + j0 + i] >= a.window) drafts &= ~(1ull << i);
        }
    }
    return m | drafts;
}

// Scores where all keys are seen are worked on in fragments: lane l holds columns 8 i + 2 (l % 4) and the next of the rows
// l / 4 + 8 r, r = 0 .. 3, of a warp's 32, so that it needs 16 keys' scales rather than 64 (a row a lane, scales took
// 512 of 1,300 cycles that the shared memory was busy with a tile).  16 columns: scores[8 (r / 2) + 4 (i % 2) + 2 (r % 2) + ..].
__device__ __forceinline__ void load_fragment(uint32_t s_col, uint32_t (&s)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(s[0]), "=r"(s[1]), "=r"(s[2]), "=r"(s[3]), "=r"(s[4]), "=r"(s[5]), "=r"(s[6]), "=r"(s[7]) : "r"(s_col));
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(s[8]), "=r"(s[9]), "=r"(s[10]), "=r"(s[11]), "=r"(s[12]), "=r"(s[13]), "=r"(s[14]), "=r"(s[15])
                 : "r"(s_col + (16u << 16)));
}
// 16-bit pairs of 64 columns of 16 rows: p[2 i + r % 2]
__device__ __forceinline__ void store_pairs(uint32_t col, const uint32_t (&p)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(col), "r"(p[0]), "r"(p[1]), "r"(p[2]), "r"(p[3]), "r"(p[4]), "r"(p[5]), "r"(p[6]), "r"(p[7]), "r"(p[8]),
                 "r"(p[9]), "r"(p[10]), "r"(p[11]), "r"(p[12]), "r"(p[13]), "r"(p[14]), "r"(p[15]) : "memory");
}
// A number of each of the warp's rows, from a lane a row to fragments (lane l: rows l / 4 + 8 r) and back (every lane of
// four has the same).
__device__ __forceinline__ void rows_to_fragments(float x, float (&f)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = __shfl_sync(0xffffffffu, x, 8 * r + ((threadIdx.x & 31) >> 2));
}
__device__ __forceinline__ float fragments_to_rows(const float (&f)[4]) {
    const int lane = threadIdx.x & 31;
    float x = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float y = __shfl_sync(0xffffffffu, f[r], 4 * (lane & 7));
        if (lane >> 3 == r) x = y;
    }
    return x;
}

// 16 columns, QUARTER of 64: 16-bit 2^(s kscale - ref) times the values' scales (CODES) or 2^(s scale - ref); float32 sums of the
// probabilities are added to sum[].  kscale, vscale: of the lane's first column.
template <bool CODES, int QUARTER>
__device__ __forceinline__ void exponentials(const uint32_t (&s)[16], float scale, const float* kscale, const float* vscale,
                                             const float (&ref)[4], uint32_t (&p)[2][16], uint64_t (&sum)[4]) {
    using namespace slb_softmax;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float2 k = make_float2(scale, scale), v = k;
        if constexpr (CODES) {
            k = *reinterpret_cast<const float2*>(kscale + 16 * QUARTER + 8 * i);
            v = *reinterpret_cast<const float2*>(vscale + 16 * QUARTER + 8 * i);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int at = 8 * (r >> 1) + 4 * i + 2 * (r & 1);
            const float2 x = pair_of(fma2(pair_bits(__uint_as_float(s[at]), __uint_as_float(s[at + 1])), pair_bits(k.x, k.y),
                                          pair_bits(-ref[r], -ref[r])));
            const uint64_t e = pair_bits(fast_exp2(x.x), fast_exp2(x.y));
            sum[r] = add2(sum[r], e);
            const float2 y = pair_of(CODES ? mul2(e, pair_bits(v.x, v.y)) : e);
            p[r >> 1][2 * (2 * QUARTER + i) + (r & 1)] = CODES ? slb_codes::half_pair(y.x, y.y) : pack2(y.x, y.y);
        }
    }
}
// A warp's rows, every quarter's scores on their way while the one before is worked on.
template <bool CODES>
__device__ __forceinline__ void all_exponentials(uint32_t s_col, float scale, const float* kscale, const float* vscale,
                                                 const float (&ref)[4], uint32_t (&p)[2][16], float (&sums)[4]) {
    uint32_t a[16], b[16];
    uint64_t sum[4] = {0, 0, 0, 0};
    load_fragment(s_col, a);
    wait_ld16(a);
    load_fragment(s_col + 16, b);
    exponentials<CODES, 0>(a, scale, kscale, vscale, ref, p, sum);
    wait_ld16(b);
    load_fragment(s_col + 32, a);
    exponentials<CODES, 1>(b, scale, kscale, vscale, ref, p, sum);
    wait_ld16(a);
    load_fragment(s_col + 48, b);
    exponentials<CODES, 2>(a, scale, kscale, vscale, ref, p, sum);
    wait_ld16(b);
    exponentials<CODES, 3>(b, scale, kscale, vscale, ref, p, sum);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float2 t = slb_softmax::pair_of(sum[r]);
        sums[r] = t.x + t.y;
    }
}
// The largest score of each row (a lane a row), with codes the largest sum of a key's score and log2 of its value's scale: of one
// key, so that a large scale whose key has no weight leaves the others' bits alone.  klog: as kscale, of those logarithms.
template <bool CODES> __device__ __forceinline__ float row_maximum(uint32_t s_col, float scale, const float* kscale, const float* klog) {
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
    for (int quarter = 0; quarter < 4; ++quarter) {
        uint32_t s[16];
        load_fragment(s_col + 16 * quarter, s);
        wait_ld16(s);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float2 k = make_float2(scale, scale), w = make_float2(0.f, 0.f);
            if constexpr (CODES) {
                k = *reinterpret_cast<const float2*>(kscale + 16 * quarter + 8 * i);
                w = *reinterpret_cast<const float2*>(klog + 16 * quarter + 8 * i);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int at = 8 * (r >> 1) + 4 * i + 2 * (r & 1);
                m[r] = fmaxf(m[r], fmaxf(fmaf(__uint_as_float(s[at]), k.x, w.x), fmaf(__uint_as_float(s[at + 1]), k.y, w.y)));
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 1));
        m[r] = fmaxf(m[r], __shfl_xor_sync(0xffffffffu, m[r], 2));
    }
    return fragments_to_rows(m);
}
// Powers of two that bring the tile's queries into float16, as exponent fields.  One for all rows (`field`) where each row's
// largest element lies within 2^16 of the tile's: then an element is off by at most 2^-22 of its row's largest.  Otherwise
// (`wide`) a row has its own, at most 2^126 above the tile's.
struct QueryFactors {
    int field;
    bool wide;
};
// 16-bit magnitudes: the largest, and one less than the least that is not zero
struct Spread {
    unsigned top, least;
    __device__ __forceinline__ bool wide() const { return least != 0xffffu && (int)(top >> 7) - (int)((least + 1) >> 7) > 16; }
};
__device__ __forceinline__ Spread spread_of(unsigned tops, unsigned leasts) {      // of pairs, over a warp
    return {__reduce_max_sync(0xffffffffu, max(tops & 0xffffu, tops >> 16)), __reduce_min_sync(0xffffffffu, min(leasts & 0xffffu, leasts >> 16))};
}
__device__ __forceinline__ int row_field(const unsigned char* smem, int row, const QueryFactors& f) {
    if (!f.wide) return f.field;
    const unsigned top = reinterpret_cast<const unsigned short*>(smem + OFF_TOP)[row];
    return min(slb_codes::query_field(__uint_as_float(top << 16)), f.field + 126);
}

// grid: units of 128 rows and kv head, each with its shares of the keys
template <int KIND>
__global__ void __launch_bounds__(THREADS, 2) cache_attention_tc_kernel(const CacheAttnArgs a) {
    constexpr bool CODES = KIND != CACHE_PLAIN;
    constexpr int ROW_BYTES = D * (CODES ? 1 : 2);
    extern __shared__ __align__(1024) unsigned char smem[];
    // s_full[b]: Q.K^T of a tile is done (scores ready, keys replaceable); pv_done[b]: its P.V (values replaceable, O final)
    uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + OFF_BAR);     // [2] each
    uint64_t* v_full = k_full + 2;
    uint64_t* s_full = v_full + 2;
    uint64_t* p_full = s_full + 2;
    uint64_t* pv_done = p_full + 2;
    uint64_t* scouted = pv_done + 2;                        // [AHEAD] each: a tile's rows, its scales are known; its place is free
    uint64_t* scaled = scouted + AHEAD;
    uint64_t* vacated = scaled + AHEAD;
    uint64_t* q_full = vacated + AHEAD;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);
    float* scales = reinterpret_cast<float*>(smem + OFF_SCALE);
    int* key_rows = reinterpret_cast<int*>(smem + OFF_ROW);
    int* scale_logs = reinterpret_cast<int*>(smem + OFF_LOG);

    // (what needs no data goes before the wait for the kernels before this one)
    const int warp = slb_warp(), lane = threadIdx.x & 31;
    const bool aligned = (smem_u32(smem) & 1023u) == 0;     // the swizzle needs 1024-byte alignment
    if (!aligned) { gave_up(0x900); return; }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], CODES ? LOADER_WARPS : 32 * LOADER_WARPS);
            mbar_init(&v_full[i], CODES ? LOADER_WARPS : 32 * LOADER_WARPS);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], SOFTMAX_WARPS);
            mbar_init(&pv_done[i], 1);
        }
        for (int i = 0; i < AHEAD; ++i) {
            mbar_init(&scouted[i], 1);
            mbar_init(&scaled[i], 1);
            mbar_init(&vacated[i], LOADER_WARPS + SOFTMAX_WARPS);
        }
        mbar_init(q_full, MMA_WARP);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_wait();
    // the units' blocks one behind the other, the last `more` units with a part more each
    const int units = a.tiles * a.Hkv, plain = (units - a.more) * a.parts, behind = (int)blockIdx.x - plain;
    const int parts = a.parts + (behind >= 0 ? 1 : 0);
    const int unit = behind >= 0 ? units - a.more + behind / parts : (int)blockIdx.x / parts;
    const int part = behind >= 0 ? behind % parts : (int)blockIdx.x % parts;
    const int kvh = unit % a.Hkv, g = a.H / a.Hkv;
    // (tiles from the last to the first: a request's last tile has the most keys)
    const int tile = units / a.Hkv - 1 - unit / a.Hkv;
    const Tile t = find_tile(a, g, tile);
    const int row0 = t.row0, q0 = t.q0, ctx = t.ctx, base = ctx - t.q_len;
    const int nrows = min(BM, t.q_len * g - row0);
    const int* table = a.table + (size_t)max(t.s, 0) * a.max_pages;
    // keys that some row of the tile sees: from kbeg on (with a mask a token's position is at least base) to kend
    const int first_local = row0 / g, last_local = (row0 + nrows - 1) / g;
    int kbeg = 0;
    if (a.window > 0) kbeg = max(0, (a.mask != nullptr ? base : base + first_local) - a.window + 1);
    if (a.mask != nullptr) kbeg = min(kbeg, max(0, base));
    kbeg = kbeg / BN * BN;
    int kend = a.mask != nullptr ? ctx : min(ctx, base + last_local + 1);
    int ntiles = max(0, kend - kbeg + BN - 1) / BN;
    if (parts > 1) {                                        // this block's share of the keys (maybe none)
        const int per = ntiles / parts, more = ntiles - per * parts;
        kbeg += (part * per + min(part, more)) * BN;
        ntiles = per + (part < more ? 1 : 0);
        kend = min(kend, kbeg + ntiles * BN);
    }
    const int shift = page_shift(a.ps);
    auto page_of = [&](int j, int i) {                      // the scout's look-ups, the first before the block's barrier
        const int at = kbeg + j * BN + lane + 32 * i;
        return table_entry(table, a.max_pages, at, a.ps, shift, j < ntiles && at < kend);
    };
    int next[2] = {-1, -1};
    if (warp == SCOUT_WARP && t.s >= 0) {
        next[0] = page_of(0, 0);
        next[1] = page_of(0, 1);
    }

    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    if (t.s < 0) {                                          // no such tile
        if (warp == MMA_WARP)
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
        return;
    }

    if (warp < MMA_WARP) {
        // Queries: softmax and loader warps (whose rows are being looked up) stage 16 rows each, D / 8 lanes a row.  With codes
        // they become float16 by powers of two (QueryFactors).
        constexpr int LANES = D / 8, AT_ONCE = 32 / LANES, MINE = BM / MMA_WARP, ROUNDS = MINE / AT_ONCE;
        const int c = lane % LANES, rho = row0 + min(MINE * warp + lane % MINE, nrows - 1), local = rho / g;
        const bf16* mine = reinterpret_cast<const bf16*>(a.q) + (size_t)(q0 + local) * a.ldq + (size_t)(kvh * g + rho - local * g) * D;
        uint4 x[ROUNDS];
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {                  // (rows of padding repeat the last one)
            const unsigned long long row = __shfl_sync(0xffffffffu, (unsigned long long)(uintptr_t)mine, i * AT_ONCE + lane / LANES);
            x[i] = reinterpret_cast<const uint4*>((uintptr_t)row)[c];
        }
        QueryFactors factors = {};
        if constexpr (CODES) {
            // Of every 16 bytes the largest magnitude (bfloat16 bits), in pairs of rounds: if those lie near enough to one another,
            // rows do.
            unsigned tops[ROUNDS / 2], most = 0, leasts = 0xffffffffu;
#pragma unroll
            for (int i = 0; i < ROUNDS; ++i) {
                const unsigned both = __vmaxu2(__vmaxu2(x[i].x & 0x7fff7fffu, x[i].y & 0x7fff7fffu), __vmaxu2(x[i].z & 0x7fff7fffu, x[i].w & 0x7fff7fffu));
                const unsigned top = max(both & 0xffffu, both >> 16);
                tops[i / 2] = i % 2 ? tops[i / 2] | top << 16 : top;
            }
#pragma unroll
            for (int i = 0; i < ROUNDS / 2; ++i) {
                most = __vmaxu2(most, tops[i]);
                leasts = __vminu2(leasts, __vsub2(tops[i], 0x00010001u));
            }
            Spread s = spread_of(most, leasts);
            if (lane == 0) reinterpret_cast<unsigned*>(smem + OFF_SPREAD)[warp] = s.top | s.least << 16;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * MMA_WARP) : "memory");
            const uint4 u = *reinterpret_cast<const uint4*>(smem + OFF_SPREAD), w = *reinterpret_cast<const uint4*>(smem + OFF_SPREAD + 16);
            s.top = __vmaxu2(__vmaxu2(__vmaxu2(u.x, u.y), __vmaxu2(u.z, u.w)), __vmaxu2(__vmaxu2(w.x, w.y), __vmaxu2(w.z, w.w))) & 0xffffu;
            s.least = __vminu2(__vminu2(__vminu2(u.x, u.y), __vminu2(u.z, u.w)), __vminu2(__vminu2(w.x, w.y), __vminu2(w.z, w.w))) >> 16;
            if (s.wide() || s.top >= 0x7f80u) {             // (in all of these warps) row by row
#pragma unroll
                for (int i = 0; i < ROUNDS; i += 2) {
                    unsigned rows = tops[i / 2];
#pragma unroll
                    for (int o = LANES / 2; o > 0; o >>= 1) rows = __vmaxu2(rows, __shfl_xor_sync(0xffffffffu, rows, o));
                    if (c < 2) {                            // (a row with an infinity or NaN does not count: it has no result)
                        const unsigned top = c == 0 ? rows & 0xffffu : rows >> 16;
                        reinterpret_cast<unsigned short*>(smem + OFF_TOP)[warp * MINE + (i + c) * AT_ONCE + lane / LANES] =
                            (unsigned short)(top < 0x7f80u ? top : 0);
                    }
                }
                asm volatile("bar.sync 1, %0;" ::"n"(32 * MMA_WARP) : "memory");
                const uint2 t4 = reinterpret_cast<const uint2*>(smem + OFF_TOP)[lane];
                s = spread_of(__vmaxu2(t4.x, t4.y), __vminu2(__vsub2(t4.x, 0x00010001u), __vsub2(t4.y, 0x00010001u)));
                factors.wide = s.wide();
            }
            factors.field = slb_codes::query_field(__uint_as_float(s.top << 16));
            if (threadIdx.x == 0) *reinterpret_cast<QueryFactors*>(smem + OFF_FIELD) = factors;
        }
#pragma unroll
        for (int i = 0; i < ROUNDS; ++i) {
            const int qr = warp * MINE + i * AT_ONCE + lane / LANES;
            uint4 y = x[i];
            if constexpr (CODES) {
                const float factor = slb_codes::power(row_field(smem, qr, factors));
                if (slb_codes::swaps<KIND>())
                    y = make_uint4(__byte_perm(y.x, y.y, 0x5410), __byte_perm(y.x, y.y, 0x7632),
                                   __byte_perm(y.z, y.w, 0x5410), __byte_perm(y.z, y.w, 0x7632));
                y = make_uint4(slb_codes::half_pair(y.x, factor), slb_codes::half_pair(y.y, factor),
                               slb_codes::half_pair(y.z, factor), slb_codes::half_pair(y.w, factor));
            }
            *reinterpret_cast<uint4*>(smem + (c >> 3) * Q_PANEL + qr * 128 + (((c & 7) ^ (qr & 7)) << 4)) = y;
        }
        fence_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
    }
    if (warp >= SOFTMAX_WARPS && warp < MMA_WARP) {
        // ---------------------------------------------------------------- loaders
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // In round i a warp takes PER keys, a lane a 16-byte piece of one: key 4 PER i + PER w + sub, whose place in the
        // swizzle is the same in every round.  (Codes of 128 elements: neighbouring lanes hold four pieces of two keys, so
        // that eight lanes store to eight different banks of 16 bytes.)
        const int w = warp - SOFTMAX_WARPS;
        constexpr int PIECES = ROW_BYTES / 16, PER = 32 / PIECES, ROUNDS = BN / (LOADER_WARPS * PER);
        const int piece = CODES && PIECES == 8 ? (lane & 3) | (lane >> 3 & 1) << 2 : lane % PIECES;
        const int sub = CODES && PIECES == 8 ? (lane >> 2 & 1) | (lane >> 4 & 1) << 1 : lane / PIECES;
        const int key0 = PER * w + sub;
        // where piece c of 16 bytes of this lane's key goes (its key in round i: 512 PER i bytes further)
        auto place = [&](int c) { return (c >> 3) * KV_PANEL + key0 * 128 + (((c & 7) ^ (key0 & 7)) << 4); };
        const char* kbase = reinterpret_cast<const char*>(a.k) + 16 * piece;
        const char* vbase = reinterpret_cast<const char*>(a.v) + 16 * piece;
        int rows[ROUNDS];
        auto get_rows = [&](int j) -> bool {                // the tile's rows, from the scout
            if (j >= ntiles) return true;
            if (!mbar_wait(&scouted[j % AHEAD], (j / AHEAD) & 1)) { gave_up(0x103); return false; }
#pragma unroll
            for (int i = 0; i < ROUNDS; ++i) rows[i] = key_rows[(j % AHEAD) * BN + LOADER_WARPS * PER * i + key0];
            __syncwarp();
            if (lane == 0) mbar_arrive(&vacated[j % AHEAD]);
            return true;
        };
        if constexpr (CODES) {
            uint4 kx[ROUNDS], vx[ROUNDS];
            auto fetch = [&](const char* from, uint4 (&x)[ROUNDS]) {
#pragma unroll
                for (int i = 0; i < ROUNDS; ++i) {
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (rows[i] >= 0)
                        asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x[i].x), "=r"(x[i].y), "=r"(x[i].z), "=r"(x[i].w)
                                     : "l"(from + (size_t)rows[i] * ROW_BYTES));
                }
            };
            const int lo = place(2 * piece), hi = place(2 * piece + 1);
            auto put = [&](unsigned char* tile, const uint4 (&x)[ROUNDS]) {
#pragma unroll
                for (int i = 0; i < ROUNDS; ++i) {
                    uint4 u, v;
                    slb_codes::four<KIND>(x[i].x, u.x, u.y);
                    slb_codes::four<KIND>(x[i].y, u.z, u.w);
                    slb_codes::four<KIND>(x[i].z, v.x, v.y);
                    slb_codes::four<KIND>(x[i].w, v.z, v.w);
                    *reinterpret_cast<uint4*>(tile + lo + i * (LOADER_WARPS * PER * 128)) = u;
                    *reinterpret_cast<uint4*>(tile + hi + i * (LOADER_WARPS * PER * 128)) = v;
                }
            };
            auto hand_over = [&](uint64_t* full) {          // a warp's stores, to the tensor core
                fence_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full);
            };
            bool ok = get_rows(0);
            if (ok && ntiles > 0) {
                fetch(kbase, kx);
                fetch(vbase, vx);
            }
            for (int j = 0; j < ntiles && ok; ++j) {
                const int st = j & 1;
                const uint32_t turn = ((j >> 1) & 1) ^ 1;
                if (!mbar_wait(&s_full[st], turn)) { gave_up(0x101); break; }
                put(smem + OFF_K + st * KV_TILE, kx);
                hand_over(&k_full[st]);
                ok = get_rows(j + 1);
                if (j + 1 < ntiles && ok) fetch(kbase, kx);
                if (!mbar_wait(&pv_done[st], turn)) { gave_up(0x102); break; }
                put(smem + OFF_V + st * KV_TILE, vx);
                hand_over(&v_full[st]);
                if (j + 1 < ntiles && ok) fetch(vbase, vx);
            }
        } else {
            auto copy_rows = [&](unsigned char* tile, const char* from, uint64_t* full) {
#pragma unroll
                for (int i = 0; i < ROUNDS; ++i)
                    slb_mma::cp_async16(tile + place(piece) + i * (LOADER_WARPS * PER * 128),
                                        from + (size_t)max(rows[i], 0) * ROW_BYTES, rows[i] >= 0);
                // the barrier counts this thread when its copies have landed
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
            };
            for (int j = 0; j < ntiles; ++j) {
                const int st = j & 1;
                const uint32_t turn = ((j >> 1) & 1) ^ 1;
                if (!get_rows(j)) break;
                if (!mbar_wait(&s_full[st], turn)) { gave_up(0x101); break; }
                copy_rows(smem + OFF_K + st * KV_TILE, kbase, &k_full[st]);
                if (!mbar_wait(&pv_done[st], turn)) { gave_up(0x102); break; }
                copy_rows(smem + OFF_V + st * KV_TILE, vbase, &v_full[st]);
            }
            asm volatile("cp.async.wait_all;" ::: "memory");        // (no copy is in flight when the block leaves)
        }
    } else if (warp == SCOUT_WARP) {
        // ---------------------------------------------------------------- scout
        // Looks the rows of up to AHEAD tiles up (lane l: keys l and l + 32), asks for them and brings their scales: loaders and
        // softmax warps find both in shared memory, and the rows in the L2 cache.  (Done by the loaders themselves,
        // look-ups and scales took 1,700 cycles of their 3,000 a tile.)
        float ksc[2], vsc[2], factor = 0.f;
        auto hand_scales = [&](int j) -> bool {             // (a tile later: they have arrived by then)
            if constexpr (CODES) {
                const int place = j % AHEAD;
                if (j == 0) {
                    if (!mbar_wait(q_full, 0)) { gave_up(0x402); return false; }
                    factor = a.scale * LOG2E * slb_codes::power(254 - reinterpret_cast<const QueryFactors*>(smem + OFF_FIELD)->field);
                }
                int top = -100;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float* to = scales + place * SCALES * BN + lane + 32 * i;
                    const int log = slb_codes::scale_log2(vsc[i]);
                    to[0] = ksc[i] * factor;
                    to[BN] = vsc[i] * slb_codes::VALUE_FACTOR;
                    to[2 * BN] = (float)log;
                    top = max(top, log);
                }
                top = __reduce_max_sync(0xffffffffu, top);
                if (lane == 0) scale_logs[place] = top;
                __syncwarp();
                if (lane == 0) mbar_arrive(&scaled[place]);
            }
            return true;
        };
        for (int j = 0; j < ntiles; ++j) {
            const int place = j % AHEAD;
            int row[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                row[i] = cache_row(next[i], kbeg + j * BN + lane + 32 * i, a.ps, shift, a.num_pages, a.Hkv, kvh, &cache_tc_status);
            if (!mbar_wait(&vacated[place], ((j / AHEAD) & 1) ^ 1)) { gave_up(0x401); break; }
#pragma unroll
            for (int i = 0; i < 2; ++i) key_rows[place * BN + lane + 32 * i] = row[i];
            __syncwarp();
            if (lane == 0) mbar_arrive(&scouted[place]);
            if (j > 0 && !hand_scales(j - 1)) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                next[i] = page_of(j + 1, i);
                ksc[i] = CODES && row[i] >= 0 ? a.ks[row[i]] : 0.f;
                vsc[i] = CODES && row[i] >= 0 ? a.vs[row[i]] : 0.f;
                if (j > 0 && row[i] >= 0) {                 // (the first tile's rows are fetched at once)
#pragma unroll
                    for (int c = 0; c < ROW_BYTES; c += 128) {
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(a.k) + (size_t)row[i] * ROW_BYTES + c));
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char*>(a.v) + (size_t)row[i] * ROW_BYTES + c));
                    }
                }
            }
            if (j == ntiles - 1) hand_scales(j);
        }
    } else if (warp == MMA_WARP) {
        // ---------------------------------------------------------------- MMA issuer
        constexpr uint32_t TYPES = (1u << 4) | (CODES ? 0u : (1u << 7) | (1u << 10));     // float32 sums of float16 or bfloat16
        const uint32_t idesc_qk = TYPES | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
        const uint32_t idesc_pv = TYPES | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
                                  ((uint32_t)(BM >> 4) << 24);
        const uint64_t q_desc = desc_128b(smem_u32(smem), 1);
        const uint64_t k_desc = desc_128b(smem_u32(smem + OFF_K), 1);
        const uint64_t v_desc = desc_128b(smem_u32(smem + OFF_V), KV_PANEL >> 4);
        // S = Q.K^T of tile t into score buffer t & 1 (its P.V of tile t - 2 has been issued before)
        auto issue_qk = [&](int t) -> bool {
            const int st = t & 1;
            if (!mbar_spin(&k_full[st], (t >> 1) & 1)) { gave_up(0x201); return false; }
            if (!CODES) fence_smem();                       // (asynchronous copies are fenced here, stores by the loaders)
            fence_after();
            if (leader()) {
#pragma unroll
                for (int p = 0; p < PANELS; ++p)
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)          // 16 elements of D = 32 bytes per step
                        mma_ss(tmem + 64 * st, q_desc + ((p * Q_PANEL + kk * 32) >> 4),
                               k_desc + ((st * KV_TILE + p * KV_PANEL + kk * 32) >> 4), idesc_qk, (p > 0 || kk > 0) ? 1u : 0u);
                commit(&s_full[st]);
            }
            return true;
        };
        bool ok = true;
        if (ntiles > 0 && !mbar_spin(q_full, 0)) { gave_up(0x204); ok = false; }
        if (ok && ntiles > 0) ok = issue_qk(0);
        if (ok && ntiles > 1) ok = issue_qk(1);
        for (int j = 0; j < ntiles && ok; ++j) {
            const int st = j & 1;
            if (!mbar_spin(&p_full[st], (j >> 1) & 1)) { gave_up(0x202); break; }
            if (!mbar_spin(&v_full[st], (j >> 1) & 1)) { gave_up(0x203); break; }
            if (!CODES) fence_smem();
            fence_after();
            if (leader()) {
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)              // 16 keys per step: P 8 columns, V 16 rows
                    mma_ts(tmem + O_COL, tmem + 64 * st + kk * 8, v_desc + ((st * KV_TILE + kk * 16 * 128) >> 4), idesc_pv,
                           (j > 0 || kk > 0) ? 1u : 0u);
                commit(&pv_done[st]);
            }
            if (j + 2 < ntiles) ok = issue_qk(j + 2);
        }
    } else {
        // ---------------------------------------------------------------- softmax, epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 128;");
        const int r = threadIdx.x;
        const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
        const int rho = row0 + min(r, nrows - 1), local = rho / g;
        const bool live = warp * 32 < nrows;                // (a warp whose rows are all padding only hands tiles on)
        const float scale = a.scale * LOG2E;                // (with codes it is in the keys' scales)
        const RowView view = row_view(a, base, q0 + local, local);
        int row_hi = view.bits != nullptr ? base - 1 : view.hi;           // every key up to here and from view.lo on is seen
        if (CODES && ntiles > 0) {                          // (rows with factors of their own go the way of masked tiles)
            if (!mbar_wait(q_full, 0)) gave_up(0x305);
            if (reinterpret_cast<const QueryFactors*>(smem + OFF_FIELD)->wide) row_hi = -1;
        }
        // A row's reference and the sum of its probabilities, of the latter what came from fragments by itself.
        // m_low: the second number of a reference (cache_codes.cuh), 0 but for scores that reach 2^24.
        float m_ref = -INFINITY, m_low = 0.f, l = 0.f, ref[4] = {0.f, 0.f, 0.f, 0.f}, l_frag[4] = {0.f, 0.f, 0.f, 0.f};
        bool ok = true;
        for (int j = 0; j < ntiles && ok; ++j) {
            if (!(live ? mbar_spin(&s_full[j & 1], (j >> 1) & 1) : mbar_wait(&s_full[j & 1], (j >> 1) & 1))) {
                gave_up(0x301);
                ok = false;
                break;
            }
            if (!live) {
                if (lane == 0) {
                    mbar_arrive(&p_full[j & 1]);
                    mbar_arrive(&vacated[j % AHEAD]);
                }
                continue;
            }
            fence_after();
            const float* kscale = scales + (j % AHEAD) * SCALES * BN;
            const float* vscale = kscale + BN;
            const float* vlog = kscale + 2 * BN;
            const uint32_t s_col = tmem + lane_base + 64 * (j & 1);
            const int k0 = kbeg + j * BN;
            bool open = __all_sync(0xffffffffu, k0 >= view.lo && k0 + BN - 1 <= row_hi && k0 + BN <= kend &&
                                                    (m_ref == -INFINITY || fabsf(m_ref) <= FUSED_REFERENCE));
            // Where every key is seen the exponentials are taken against the reference as it is.  The maximum is looked for
            // first only where a row has none yet, or where their sum says that one times its scale may be above 2^8 (as it may
            // if that key has the tile's largest scale: the search then tells).
            float alpha = 1.f, sum = 0.f, sums[4] = {0.f, 0.f, 0.f, 0.f};
            auto raise = [&](float mt) {
                if (mt > m_ref + RESCALE_THRESHOLD || (m_ref == -INFINITY && mt != -INFINITY)) {
                    alpha = m_ref == -INFINITY ? 0.f : exp2f(m_ref - mt);
                    m_ref = mt;
                }
            };
            if (CODES && !mbar_spin(&scaled[j % AHEAD], (j / AHEAD) & 1)) { gave_up(0x304); ok = false; break; }
            if (open) {
                const int top = CODES ? scale_logs[j % AHEAD] : 0;  // log2 of a power of two above the tile's value scales
                const float limit = slb_codes::power(127 + 8 - top);
                const int frag = 2 * (lane & 3);
                bool again = __any_sync(0xffffffffu, m_ref == -INFINITY);
                uint32_t p[2][16];
#pragma unroll 1
                for (int attempt = 0; attempt < 2; ++attempt) {
                    if (again) {
                        const float mt = row_maximum<CODES>(s_col, scale, kscale + frag, vlog + frag);
                        open = __all_sync(0xffffffffu, mt == -INFINITY || fabsf(mt) <= FUSED_REFERENCE);
                        if (!open) break;
                        raise(mt);
                        rows_to_fragments(m_ref == -INFINITY ? 0.f : m_ref, ref);
                    }
                    all_exponentials<CODES>(s_col, scale, kscale + frag, vscale + frag, ref, p, sums);
                    if (again) break;
                    again = __any_sync(0xffffffffu, !(fmaxf(fmaxf(sums[0], sums[1]), fmaxf(sums[2], sums[3])) <= limit) || sums[0] != sums[0] ||
                                                    sums[1] != sums[1] || sums[2] != sums[2] || sums[3] != sums[3]);
                    if (!again) break;
                }
                // P: 64 numbers of 16 bits = 32 columns, over the first half of this tile's scores
                if (open) {
                    store_pairs(s_col, p[0]);
                    store_pairs(s_col + (16u << 16), p[1]);
                }
            }
            if (!open) {
                // (sums of an attempt that was given up do not count)
                sums[0] = sums[1] = sums[2] = sums[3] = 0.f;
                uint32_t v[32];
                // (in halves and rarely: short code rather than fast)
                const unsigned long long seen = seen_keys(a, view, k0, kend, base, q0);
                // (scores are rounded before their reference is taken off: see FUSED_REFERENCE)
                float mt = -INFINITY, ms = -INFINITY, row_scale = 1.f;
                if constexpr (CODES) {                      // what the row's scores have besides the tile's factor
                    const QueryFactors f = *reinterpret_cast<const QueryFactors*>(smem + OFF_FIELD);
                    row_scale = slb_codes::power(127 + f.field - row_field(smem, r, f));
                }
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    const unsigned bits = (unsigned)(seen >> (32 * half));
                    tmem_ld32(s_col + 32 * half, v);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 k = CODES ? *reinterpret_cast<const float4*>(kscale + 32 * half + i) : make_float4(scale, scale, scale, scale);
                        const float4 w = CODES ? *reinterpret_cast<const float4*>(vlog + 32 * half + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                        const float ks[4] = {k.x, k.y, k.z, k.w}, logs[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = bits >> (i + e) & 1u ? __fmul_rn(__uint_as_float(v[i + e]), ks[e] * row_scale) : -INFINITY;
                            ms = fmaxf(ms, x);
                            if (CODES) mt = fmaxf(mt, x + logs[e]);
                        }
                    }
                }
                const bool coarse = CODES && (slb_codes::coarse_score(ms) || slb_codes::coarse_score(m_ref));
                if (CODES && __any_sync(0xffffffffu, coarse)) {
                    const float hi = fmaxf(ms, m_ref), old = (m_ref - hi) + m_low;
                    float low = old;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {
                        const unsigned bits = (unsigned)(seen >> (32 * half));
                        tmem_ld32(s_col + 32 * half, v);
                        wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float x = __fmul_rn(__uint_as_float(v[i]), kscale[32 * half + i] * row_scale) - hi + vlog[32 * half + i];
                            low = fmaxf(low, bits >> i & 1u ? x : -INFINITY);
                        }
                    }
                    if (coarse) {
                        const bool still = slb_codes::coarse_score(hi);
                        alpha = exp2f(old - low);
                        m_ref = still ? hi : hi + low;
                        m_low = still ? low : 0.f;
                    }
                }
                if (!coarse) raise(CODES ? mt : ms);
                const float row_ref = m_ref == -INFINITY ? 0.f : m_ref;
                rows_to_fragments(row_ref, ref);
                // (each half of P goes behind its scores)
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    const unsigned bits = (unsigned)(seen >> (32 * half));
                    uint32_t few[16];
                    tmem_ld32(s_col + 32 * half, v);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        const float4 k = CODES ? *reinterpret_cast<const float4*>(kscale + 32 * half + i) : make_float4(scale, scale, scale, scale);
                        const float4 w = CODES ? *reinterpret_cast<const float4*>(vscale + 32 * half + i) : make_float4(1.f, 1.f, 1.f, 1.f);
                        const float ks[4] = {k.x, k.y, k.z, k.w}, vs[4] = {w.x, w.y, w.z, w.w};
                        float p[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = __fmul_rn(__uint_as_float(v[i + e]), CODES ? ks[e] * row_scale : ks[e]);
                            p[e] = slb_softmax::fast_exp2((bits >> (i + e) & 1u ? x : -INFINITY) - row_ref - m_low);
                            sum += p[e];
                            if (CODES) p[e] = bits >> (i + e) & 1u ? p[e] * vs[e] : 0.f;      // (NaN counts where it is seen)
                        }
                        few[i >> 1] = CODES ? slb_codes::half_pair(p[0], p[1]) : slb_softmax::pack2(p[0], p[1]);
                        few[(i >> 1) + 1] = CODES ? slb_codes::half_pair(p[2], p[3]) : slb_softmax::pack2(p[2], p[3]);
                    }
                    tmem_st16(s_col + 16 * half, few);
                }
            }
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
                float factors[4];
                rows_to_fragments(alpha, factors);
                l *= alpha;
#pragma unroll
                for (int i = 0; i < 4; ++i) l_frag[i] *= factors[i];
            }
            l += sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) l_frag[i] += sums[i];
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                // the accumulator is rescaled (rarely): P.V of the previous tile must be done
                if (!mbar_wait(&pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1)) { gave_up(0x302); ok = false; break; }
                fence_after();
#pragma unroll
                for (int c0 = 0; c0 < D; c0 += 32) {
                    uint32_t ov[32];
                    tmem_ld32(tmem + lane_base + O_COL + c0, ov);
                    wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
                    tmem_st32(tmem + lane_base + O_COL + c0, ov);
                }
            }
            wait_st();
            fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&p_full[j & 1]);
                mbar_arrive(&vacated[j % AHEAD]);           // (its scales have been read)
            }
        }
        if (ok && ntiles > 0 && !mbar_wait(&pv_done[(ntiles - 1) & 1], ((ntiles - 1) >> 1) & 1)) { gave_up(0x303); ok = false; }
        fence_after();
        pdl_launch_dependents();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            l_frag[i] += __shfl_xor_sync(0xffffffffu, l_frag[i], 1);
            l_frag[i] += __shfl_xor_sync(0xffffffffu, l_frag[i], 2);
        }
        l += fragments_to_rows(l_frag);
        if (CODES && parts > 1) l *= exp2f(m_low);
        const int h = kvh * g + rho - local * g;
        const float unscale = (parts > 1 ? exp2f(m_low) : l != 0.f ? 1.f / l : 0.f) * (CODES ? 1.f / slb_codes::VALUE_FACTOR : 1.f);
        // A partial result is a tile's, columns in fours: [unit][part][D / 4][BM], and [unit][part][BM] (reference, sum).  A
        // block that gave up leaves NaN there.
        const size_t piece = (size_t)(tile * a.Hkv + kvh) * (a.parts + (a.more > 0 ? 1 : 0)) + part;
        float4* part_o = reinterpret_cast<float4*>(a.part_o) + piece * (D / 4 * BM) + r;
        if (parts > 1) reinterpret_cast<float2*>(a.part_ml)[piece * BM + r] = make_float2(ok ? m_ref : 0.f, ok ? l : NAN);
        bf16* dst = reinterpret_cast<bf16*>(a.out) + (size_t)(q0 + local) * a.ldo + (size_t)h * D;
#pragma unroll
        for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t ov[32];
            if (ntiles > 0) {
                tmem_ld32(tmem + lane_base + O_COL + c0, ov);       // warp-wide: every lane takes part
                wait_ld();
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i) ov[i] = 0u;
            }
            float o[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {                  // (columns 0, 2, 1, 3 of four with int8)
                const int at = slb_codes::swaps<KIND>() ? (i & ~3) | (i & 1) << 1 | (i & 2) >> 1 : i;
                o[i] = __uint_as_float(ov[at]) * unscale;
            }
            if (parts > 1) {
#pragma unroll
                for (int i = 0; i < 32; i += 4) part_o[((c0 + i) >> 2) * BM] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            } else if (ok && r < nrows) {
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    using slb_softmax::pack2;
                    *reinterpret_cast<uint4*>(dst + c0 + i) = make_uint4(pack2(o[i], o[i + 1]), pack2(o[i + 2], o[i + 3]),
                                                                        pack2(o[i + 4], o[i + 5]), pack2(o[i + 6], o[i + 7]));
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    if (warp == MMA_WARP) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// The parts of a tile added up in their order, each at its reference: grid (D / 16, units), a thread per row and eight
// columns; rows of neighbouring threads lie side by side in the parts.
__global__ void __launch_bounds__(2 * BM) cache_attention_tc_join_kernel(const CacheAttnArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int g = a.H / a.Hkv, tile = blockIdx.y / a.Hkv, kvh = blockIdx.y - tile * a.Hkv;
    const Tile t = find_tile(a, g, tile);
    const int r = threadIdx.x % BM, c8 = 2 * blockIdx.x + threadIdx.x / BM;
    const int parts = a.parts + ((a.tiles - 1 - tile) * a.Hkv + kvh >= a.tiles * a.Hkv - a.more ? 1 : 0);
    if (t.s < 0 || r >= t.q_len * g - t.row0 || parts == 1) return;
    const size_t unit = (size_t)blockIdx.y * (a.parts + (a.more > 0 ? 1 : 0));
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + unit * BM + r;
    const float4* po = reinterpret_cast<const float4*>(a.part_o) + unit * (D / 4 * BM) + 2 * c8 * BM + r;
    float m = -INFINITY, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < parts; p0 += 4) {                 // four parts are on their way at once
        float2 x[4];
        float4 u[4], v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = min(p0 + i, parts - 1);
            x[i] = ml[(size_t)p * BM];
            u[i] = po[(size_t)p * (D / 4 * BM)];
            v[i] = po[(size_t)p * (D / 4 * BM) + BM];
            if (p0 + i >= parts) x[i] = make_float2(-INFINITY, 0.f);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, x[i].x);
        const float ref = top == -INFINITY ? 0.f : top, old = exp2f(m - ref);
        m = top;
        l *= old;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] *= old;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p0 + i >= parts) continue;
            const float w = exp2f(x[i].x - ref);
            l += w * x[i].y;
            o[0] += w * u[i].x; o[1] += w * u[i].y; o[2] += w * u[i].z; o[3] += w * u[i].w;
            o[4] += w * v[i].x; o[5] += w * v[i].y; o[6] += w * v[i].z; o[7] += w * v[i].w;
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    const int rho = t.row0 + r, local = rho / g;
    bf16* dst = reinterpret_cast<bf16*>(a.out) + (size_t)(t.q0 + local) * a.ldo + (size_t)(kvh * g + rho - local * g) * D + 8 * c8;
    using slb_softmax::pack2;
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv),
                                                pack2(o[4] * inv, o[5] * inv), pack2(o[6] * inv, o[7] * inv));
}

template <int KIND>
int launch_tc(const CacheAttnArgs& a, int units, cudaStream_t st) {
    static unsigned long long configured = 0;              // a bit per device
    int rc = slb_configure(&configured, cache_attention_tc_kernel<KIND>, SMEM);
    if (rc != 0) return rc;
    rc = slb_launch(cache_attention_tc_kernel<KIND>, dim3((unsigned)(units * a.parts + a.more)), dim3(THREADS), SMEM, st, a);
    if (rc != 0 || (a.parts == 1 && a.more == 0)) return rc;
    return slb_launch(cache_attention_tc_join_kernel, dim3(D / 16, (unsigned)units), dim3(2 * BM), 0, st, a);
}

}  // namespace

int slb_check_cache_attention(const CacheAttnArgs& a);     // attention_cache.cu

extern "C" {

int slb_cache_attention_tc_rows(void) { return BM; }

// a->tiles: tiles of 128 rows that the step has at most.  Parts: float32 [tiles][Hkv][parts, with a->more one more][128] x
// (head size, then 2).
int slb_cache_attention_tc_bf16(const CacheAttnArgs* a, cudaStream_t st) {
    const int rc = slb_check_cache_attention(*a);
    if (rc != 0) return rc;
    const long long units = (long long)a->tiles * a->Hkv;
    if (a->more < 0 || a->more > units || (a->more > 0 && (a->part_o == nullptr || a->part_ml == nullptr))) return SLB_ERR_BAD_ARG;
    if (((a->parts > 1 || a->more > 0) && units > 65535) || units * (a->parts + 1ll) > 0x7fffffffll) return SLB_ERR_TOO_LARGE;
    return a->kind == CACHE_INT8 ? launch_tc<CACHE_INT8>(*a, (int)units, st)
           : a->kind == CACHE_E4M3 ? launch_tc<CACHE_E4M3>(*a, (int)units, st) : launch_tc<CACHE_PLAIN>(*a, (int)units, st);
}
}
