// Attention over a paged cache in bfloat16 or 8 bits for steps of few query rows a kv head (single tokens, small trees of
// drafted tokens), bfloat16 queries, specialised at compile time for one head size (SLB_HEAD_DIM, 64 or 128).
//
// Work unit: (share of the keys, kv head x tile of 8 or 16 query rows, request).  A warp takes 16 keys at a time, which it
// fetches two slices ahead into a ring of its own, and computes the transposed problem on mma.sync.m16n8k16:
//
//     S^T[key, row] = K[key, :] . Q^T[:, row]        O^T[d, row] += V^T[d, key] . P^T[key, row]
//
// so that keys and head elements are the long sides and the few rows the short one.  Codes become float16 exactly
// (cache_codes.cuh); a key's scale multiplies its scores, a value's scale the probabilities, in float32.  The order of a
// head's elements along K is free as long as both operands agree, and the order of the rows of O^T is free altogether: a
// lane therefore takes the 16-byte pieces of a cached row as they lie.
//
// Over a bfloat16 cache probabilities are rounded to bfloat16, the type that a product then takes on both sides: at most
// 2^-8 of a weight, as in the package's other tensor-core attention.
//
// What bounds it: memory where there are many requests (64 tokens over 4,100 keys in e4m3, 28 heads over 4 of 128: 48.4 us, 0.83 of
// the rate of a copy), start, conversion of codes and the cluster's exchange where there are few (8 tokens over 2,049 keys in int8
// 11.6 us, one over 301 keys of 14 heads over 2 of 64 6.0).
#include <cuda.h>

#include "cache_codes.cuh"
#include "cluster_util.cuh"
#include "mma_util.cuh"

#ifndef SLB_HEAD_DIM
#error "compile with -DSLB_HEAD_DIM=<head size>"
#endif

SLB_DEFINE_PDL_SWITCH
SLB_DEFINE_STATUS_WORD(cache_attn_status, slb_cache_attention_status)

namespace {

using slb_mma::mma_bf16;
using slb_mma::pack_bf16;
using namespace slb_cluster;

constexpr int D = SLB_HEAD_DIM;
static_assert(D == 64 || D == 128, "head sizes 64 and 128");
constexpr int FEW_WARPS = 8;
constexpr int KEYS = 16;                       // of a warp's slice
constexpr int MAX_CLUSTER = 8;
constexpr float LAZY_LOG2 = 8.f;               // a row's reference moves when a score exceeds it by 2^8
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ unsigned movmatrix_trans(unsigned a) {
    unsigned d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async4(void* smem, const void* from, bool valid) {
    const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
    const int bytes = valid ? 4 : 0;                   // 0: zeros
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(s), "l"(from), "r"(bytes));
}

template <int KIND> struct Few {
    static constexpr int ROW_BYTES = D * (KIND == CACHE_PLAIN ? 2 : 1);
    static constexpr int KQ = ROW_BYTES / 64;          // 16-byte pieces of a key's row that a lane holds (of four lanes)
    static constexpr int VW = ROW_BYTES / 32;          // words of a value's row that a lane holds (of eight lanes)
    static constexpr int KSTEPS = D / 16, MT = D / 16;
    static constexpr int PIECES = ROW_BYTES / 16;      // 16-byte pieces of a row
    // A warp's ring: a slice is 16 rows of K, 16 of V, their scales (keys', values').
    static constexpr int SLICE = 32 * ROW_BYTES + (KIND == CACHE_PLAIN ? 0 : 128);
    static constexpr int STAGES = 3;
    // Pieces of a row are exchanged so that lanes which read at once (four pieces of rows r, r + 1 of K; piece g and g + 1
    // of rows 0, 2, 4, 6 of V) meet different banks.
    static __device__ __forceinline__ int key_piece(int row, int c) { return PIECES == 4 ? c : c ^ ((row & 1) << 2); }
    static __device__ __forceinline__ int value_piece(int row, int c) { return PIECES == 4 ? c ^ (row >> 1 & 3) : c ^ (row & 7); }
    // head element of row r (0..7; `half`: 8 + r) of tile mm of O^T
    static __device__ __forceinline__ int element(int mm, int r, int half) {
        if constexpr (KIND == CACHE_PLAIN) return 64 * (mm >> 2) + 8 * r + 2 * (mm & 3) + half;
        else return (D / 8) * r + 2 * mm + half;
    }
};

// shared memory of the rings and of the merge that follows in their place
template <int KIND, int NT> __host__ __device__ constexpr int few_ring_bytes() {
    const int rings = FEW_WARPS * Few<KIND>::STAGES * Few<KIND>::SLICE, merge = FEW_WARPS * 8 * NT * D * 4;
    return rings > merge ? rings : merge;
}

// grid (parts * cluster, Hkv * tiles, S).  NT: tiles of 8 query rows.
template <int KIND, int NT>
__global__ void __launch_bounds__(32 * FEW_WARPS, NT == 1 ? 2 : 1) few_rows_kernel(const CacheAttnArgs a) {
    using F = Few<KIND>;
    constexpr int NR = 8 * NT;
    extern __shared__ __align__(128) float smem[];     // the warps' rings, and behind the keys' loop:
    float4* red_o = reinterpret_cast<float4*>(smem);   // [warps][accumulators of a warp]
    float4* from_o = reinterpret_cast<float4*>(reinterpret_cast<unsigned char*>(smem) + few_ring_bytes<KIND, NT>());   // [blocks][share]
    uint2* q_frag = reinterpret_cast<uint2*>(from_o + NR * D / 4);   // [NT][KSTEPS][32], NT > 1
    __shared__ float2 red_ml[FEW_WARPS][NR], from_ml[MAX_CLUSTER][NR];     // (reference, sum) of each row
    __shared__ float lows[FEW_WARPS][NR];              // the second numbers of references (cache_codes.cuh), with `coarse`
    if (a.cluster > 1) cluster_arrive();               // (blocks send to one another: all must have begun)
    bool begun = a.cluster == 1;
    pdl_wait();
    const int tid = threadIdx.x, warp = slb_warp(), lane = tid & 31, lg = lane >> 2, lt = lane & 3;
    const int cs = a.cluster, splits = a.parts * cs;
    const int split = blockIdx.x, part = split / cs, rank = split - part * cs;
    const int kvh = blockIdx.y % a.Hkv, s = blockIdx.z, g = a.H / a.Hkv;
    int q0 = a.cu_q[s], q1 = a.cu_q[s + 1];
    clamp_span(a.T, q0, q1);
    const int q_len = q1 - q0, ctx = a.ctx_len[s], base = ctx - q_len;
    const int* table = a.table + (size_t)s * a.max_pages;
    const int shift = page_shift(a.ps);
    const float scale = a.scale * LOG2E;
    const bf16* q = reinterpret_cast<const bf16*>(a.q);

    for (int tile = blockIdx.y / a.Hkv; (long long)tile * NR < (long long)q_len * g; tile += a.tiles) {
        const int row0 = tile * NR, nrows = min(NR, q_len * g - row0);
        // ---- what the rows of this lane's score columns (2 lt, 2 lt + 1 of each tile) see
        RowView view[NT][2];
        int lo_all = 0x7fffffff, lo_most = 0;          // slots before base: the first that some row, that every row sees
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int local = (row0 + min(8 * nt + 2 * lt + c, nrows - 1)) / g;
                view[nt][c] = row_view(a, base, q0 + local, local);
                lo_all = min(lo_all, view[nt][c].lo);
                lo_most = max(lo_most, view[nt][c].lo);
            }
        lo_all = __reduce_min_sync(0xffffffffu, lo_all);
        if (a.mask != nullptr) lo_all = min(lo_all, base);     // (drafted tokens go by their positions)
        lo_all = max(0, lo_all);
        lo_most = __reduce_max_sync(0xffffffffu, lo_most);
        const int last = a.mask != nullptr ? ctx : min(ctx, base + (row0 + nrows - 1) / g + 1);
        const int kbeg = lo_all / KEYS * KEYS;
        const int slices = (max(0, last - kbeg) + KEYS - 1) / KEYS;
        const int step = splits * FEW_WARPS;

        // lane l (and l + 16): the page, then the cache row, of key l of a slice
        auto page_of = [&](int slice) {
            const int key = kbeg + slice * KEYS + (lane & 15);
            return table_entry(table, a.max_pages, key, a.ps, shift, slice < slices && key < last && key >= lo_all);
        };
        auto row_of = [&](int page, int slice) {
            return cache_row(page, kbeg + slice * KEYS + (lane & 15), a.ps, shift, a.num_pages, a.Hkv, kvh, &cache_attn_status);
        };
        // The rows of a slice into a stage of the warp's ring, piece by piece as they lie (zeros where there is no row).
        unsigned char* ring = reinterpret_cast<unsigned char*>(smem) + warp * (F::STAGES * F::SLICE);
        auto fill = [&](int stage, int row) {
            unsigned char* to = ring + stage * F::SLICE;
            constexpr int PER = 32 / F::PIECES;        // rows that the lanes take at once
#pragma unroll
            for (int i = 0; i < KEYS / PER; ++i) {
                const int r = i * PER + lane / F::PIECES, c = lane % F::PIECES;
                const int from = __shfl_sync(0xffffffffu, row, r);
                const size_t at = (size_t)max(from, 0) * F::ROW_BYTES + 16 * c;
                slb_mma::cp_async16(to + r * F::ROW_BYTES + 16 * F::key_piece(r, c), reinterpret_cast<const char*>(a.k) + at, from >= 0);
                slb_mma::cp_async16(to + (KEYS + r) * F::ROW_BYTES + 16 * F::value_piece(r, c), reinterpret_cast<const char*>(a.v) + at,
                                    from >= 0);
            }
            if constexpr (KIND != CACHE_PLAIN)
                cp_async4(to + 2 * KEYS * F::ROW_BYTES + 4 * lane, (lane < 16 ? a.ks : a.vs) + max(row, 0), row >= 0);
            slb_mma::cp_async_commit();
        };

        int slice = split * FEW_WARPS + warp;
        int pages[F::STAGES];
#pragma unroll
        for (int i = 0; i < F::STAGES; ++i) pages[i] = page_of(slice + i * step);
        uint2 qx[NT][F::KSTEPS];                       // (the queries are on their way while the first slices are asked for)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = 8 * nt + lg, rho = row0 + (r < nrows ? r : 0);
            const bf16* src = q + (size_t)(q0 + rho / g) * a.ldq + (size_t)(kvh * g + rho % g) * D;
#pragma unroll
            for (int k = 0; k < F::KSTEPS; ++k) {
                const int at = KIND == CACHE_PLAIN ? 8 * (lt + 4 * (k >> 1)) + 4 * (k & 1) : 16 * (lt + 4 * (k >> 2)) + 4 * (k & 3);
                qx[nt][k] = *reinterpret_cast<const uint2*>(src + at);      // (a row of padding is the tile's first)
            }
        }
#pragma unroll
        for (int i = 0; i < F::STAGES - 1; ++i) fill(i, row_of(pages[i], slice + i * step));
        int page = pages[F::STAGES - 1], stage = 0;
        // ---- queries: the B operand of S^T, whose lane (lg, lt) holds query row lg
        uint2 qf[NT == 1 ? F::KSTEPS : 1];
        float row_factor[NT][2];                       // of the rows of this lane's score columns
        if (NT > 1) __syncthreads();                   // (the tile before may still be read)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float factor = 1.f;                        // of the row's scores
            if constexpr (KIND != CACHE_PLAIN) {
                float top = 0.f;
#pragma unroll
                for (int k = 0; k < F::KSTEPS; ++k)
                    top = fmaxf(top, fmaxf(fmaxf(fabsf(__uint_as_float(qx[nt][k].x << 16)), fabsf(__uint_as_float(qx[nt][k].x & 0xffff0000u))),
                                           fmaxf(fabsf(__uint_as_float(qx[nt][k].y << 16)), fabsf(__uint_as_float(qx[nt][k].y & 0xffff0000u)))));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int field = slb_codes::query_field(top);
#pragma unroll
                for (int k = 0; k < F::KSTEPS; ++k) {
                    uint2 x = qx[nt][k];
                    if (slb_codes::swaps<KIND>()) x = make_uint2(__byte_perm(x.x, x.y, 0x5410), __byte_perm(x.x, x.y, 0x7632));
                    qx[nt][k] = make_uint2(slb_codes::half_pair(x.x, slb_codes::power(field)), slb_codes::half_pair(x.y, slb_codes::power(field)));
                }
                factor = slb_codes::power(254 - field);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) row_factor[nt][c] = __shfl_sync(0xffffffffu, factor, 4 * (2 * lt + c)) * scale;
#pragma unroll
            for (int k = 0; k < F::KSTEPS; ++k) {
                if constexpr (NT == 1) qf[k] = qx[nt][k];
                else if (warp == nt) q_frag[(nt * F::KSTEPS + k) * 32 + lane] = qx[nt][k];
            }
        }
        if (NT > 1) __syncthreads();
        bool coarse = false;                           // some row of the warp has a reference of two numbers
        float m[NT][2], l[NT][2], acc[NT][F::MT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int i = 0; i < F::MT; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
        }
        for (; slice < slices; slice += step) {
            const int k0 = kbeg + slice * KEYS;
            slb_mma::cp_async_wait<F::STAGES - 2>();   // this slice has landed
            __syncwarp();                              // ... for all lanes, and all are done with the one before
            fill(stage == 0 ? F::STAGES - 1 : stage - 1, row_of(page, slice + (F::STAGES - 1) * step));
            page = page_of(slice + F::STAGES * step);
            const unsigned char* ks_at = ring + stage * F::SLICE;
            const unsigned char* vs_at = ks_at + KEYS * F::ROW_BYTES;
            stage = stage == F::STAGES - 1 ? 0 : stage + 1;
            float ksc[2] = {1.f, 1.f}, vsc[2] = {1.f, 1.f}, lv[2] = {0.f, 0.f};      // of keys lg and lg + 8; log2 of the values'
            if constexpr (KIND != CACHE_PLAIN) {
                const float* sc_at = reinterpret_cast<const float*>(vs_at + KEYS * F::ROW_BYTES);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    ksc[i] = sc_at[lg + 8 * i];
                    vsc[i] = sc_at[16 + lg + 8 * i];
                    lv[i] = (float)slb_codes::scale_log2(vsc[i]);
                    vsc[i] *= slb_codes::VALUE_FACTOR;
                }
            }
            // ---- scores of 16 keys
            float sc[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
            for (int c = 0; c < F::KQ; ++c) {
                const uint4 k0x = *reinterpret_cast<const uint4*>(ks_at + lg * F::ROW_BYTES + 16 * F::key_piece(lg, lt + 4 * c));
                const uint4 k1x = *reinterpret_cast<const uint4*>(ks_at + (lg + 8) * F::ROW_BYTES + 16 * F::key_piece(lg, lt + 4 * c));
                const unsigned x0[4] = {k0x.x, k0x.y, k0x.z, k0x.w}, x1[4] = {k1x.x, k1x.y, k1x.z, k1x.w};
                constexpr int STEPS = KIND == CACHE_PLAIN ? 2 : 4;
#pragma unroll
                for (int j = 0; j < STEPS; ++j) {
                    unsigned fr[4];
                    if constexpr (KIND == CACHE_PLAIN) {
                        fr[0] = x0[2 * j]; fr[1] = x1[2 * j]; fr[2] = x0[2 * j + 1]; fr[3] = x1[2 * j + 1];
                    } else {
                        slb_codes::four<KIND>(x0[j], fr[0], fr[2]);
                        slb_codes::four<KIND>(x1[j], fr[1], fr[3]);
                    }
                    const int k = c * STEPS + j;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        uint2 b;
                        if constexpr (NT == 1) b = qf[k];
                        else b = q_frag[(nt * F::KSTEPS + k) * 32 + lane];
                        if constexpr (KIND == CACHE_PLAIN) mma_bf16(sc[nt], fr, b.x, b.y);
                        else slb_codes::mma_f16(sc[nt], fr, b.x, b.y);
                    }
                }
            }
            // ---- scale, mask
            const bool open = k0 >= lo_most && k0 + KEYS <= min(base, last);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e)            // (rounded here: the maximum and the exponents go by the same number)
                    sc[nt][e] = __fmul_rn(sc[nt][e], ksc[e >> 1] * row_factor[nt][e & 1]);
            if (!open) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k0 + lg + 8 * (e >> 1);
                        if (key >= last || !row_sees(a, view[nt][e & 1], key, base, q0)) sc[nt][e] = -INFINITY;
                    }
            }
            // ---- the rows' references move rarely (cache_codes.cuh)
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float top = fmaxf(sc[nt][c] + lv[0], sc[nt][c + 2] + lv[1]);
                    over |= top > m[nt][c] + LAZY_LOG2;
                }
            if (__any_sync(0xffffffffu, over) || (KIND != CACHE_PLAIN && coarse)) {
                auto rescale = [&](int nt, int c, float alpha) {
                    l[nt][c] *= alpha;
#pragma unroll
                    for (int i = 0; i < F::MT; ++i) { acc[nt][i][c] *= alpha; acc[nt][i][c + 2] *= alpha; }
                };
                if constexpr (KIND != CACHE_PLAIN) {
                    bool big = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) big |= slb_codes::coarse_score(sc[nt][e]);
                    if (__any_sync(0xffffffffu, big) && !coarse) {
                        coarse = true;
                        if (lane < NR) lows[warp][lane] = 0.f;
                        __syncwarp();
                    }
                }
                if (KIND == CACHE_PLAIN || !coarse) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float top = fmaxf(sc[nt][c] + lv[0], sc[nt][c + 2] + lv[1]);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            top = fmaxf(top, m[nt][c]);
                            rescale(nt, c, top == -INFINITY ? 1.f : fast_exp2(m[nt][c] - top));
                            m[nt][c] = top;
                        }
                } else {                               // (from then on with every slice: the scores become relative here)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float hi = fmaxf(sc[nt][c], sc[nt][c + 2]);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                            hi = fmaxf(hi, m[nt][c]);
                            const float from = hi == -INFINITY ? 0.f : hi;
                            float& low_of = lows[warp][8 * nt + 2 * lt + c];
                            const float old = m[nt][c] - from + low_of;
                            float low = fmaxf(old, fmaxf(sc[nt][c] - from + lv[0], sc[nt][c + 2] - from + lv[1]));
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) low = fmaxf(low, __shfl_xor_sync(0xffffffffu, low, o));
                            if (low != -INFINITY) {
                                rescale(nt, c, fast_exp2(old - low));
                                sc[nt][c] = sc[nt][c] - from - low;
                                sc[nt][c + 2] = sc[nt][c + 2] - from - low;
                                const bool two = slb_codes::coarse_score(from);
                                m[nt][c] = two ? from : from + low;
                                if (lg == 0) low_of = two ? low : 0.f;
                            }
                        }
                    __syncwarp();
                }
            }
            // ---- probabilities, times the values' scales, as the B operand of O^T
            unsigned pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float ref = m[nt][e & 1];
                    p[e] = fast_exp2(sc[nt][e] - (ref == -INFINITY || (KIND != CACHE_PLAIN && coarse) ? 0.f : ref));
                    l[nt][e & 1] += p[e];
                    if constexpr (KIND != CACHE_PLAIN) p[e] = sc[nt][e] != -INFINITY ? p[e] * vsc[e >> 1] : 0.f;   // (NaN counts where it is seen)
                }
                pb[nt][0] = movmatrix_trans(KIND == CACHE_PLAIN ? pack_bf16(p[0], p[1]) : slb_codes::half_pair(p[0], p[1]));
                pb[nt][1] = movmatrix_trans(KIND == CACHE_PLAIN ? pack_bf16(p[2], p[3]) : slb_codes::half_pair(p[2], p[3]));
            }
            unsigned vx[4][F::VW];                     // keys 2 lt, 2 lt + 1, 2 lt + 8, 2 lt + 9
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 2 * lt + (i & 1) + 8 * (i >> 1);
                const unsigned char* at = vs_at + r * F::ROW_BYTES;
                if constexpr (F::VW == 2) {
                    const uint2 x = *reinterpret_cast<const uint2*>(at + 16 * F::value_piece(r, lg >> 1) + 8 * (lg & 1));
                    vx[i][0] = x.x; vx[i][1] = x.y;
                } else {
#pragma unroll
                    for (int c = 0; c < F::VW / 4; ++c) {
                        const uint4 x = *reinterpret_cast<const uint4*>(at + 16 * F::value_piece(r, lg + 8 * c));
                        vx[i][4 * c] = x.x; vx[i][4 * c + 1] = x.y; vx[i][4 * c + 2] = x.z; vx[i][4 * c + 3] = x.w;
                    }
                }
            }
#pragma unroll
            for (int w = 0; w < F::VW; ++w) {
                unsigned fr[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {          // keys 2 lt, 2 lt + 1, then 8 further
                    const unsigned x = vx[2 * i][w], y = vx[2 * i + 1][w];
                    if constexpr (KIND == CACHE_PLAIN) {
                        fr[0][2 * i] = __byte_perm(x, y, 0x5410);
                        fr[0][2 * i + 1] = __byte_perm(x, y, 0x7632);
                    } else {
                        slb_codes::beside<KIND, false>(x, y, fr[0][2 * i], fr[0][2 * i + 1]);
                        slb_codes::beside<KIND, true>(x, y, fr[1][2 * i], fr[1][2 * i + 1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (KIND == CACHE_PLAIN) {
                        mma_bf16(acc[nt][w], fr[0], pb[nt][0], pb[nt][1]);
                    } else {
                        slb_codes::mma_f16(acc[nt][2 * w], fr[0], pb[nt][0], pb[nt][1]);
                        slb_codes::mma_f16(acc[nt][2 * w + 1], fr[1], pb[nt][0], pb[nt][1]);
                    }
                }
            }
        }

        slb_mma::cp_async_wait<0>();
        // ---- the warps' results become the block's, four accumulators (rows 2 lt, 2 lt + 1 of two head elements) at a time
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
                if (KIND != CACHE_PLAIN && coarse) l[nt][c] *= fast_exp2(lows[warp][8 * nt + 2 * lt + c]);
                if (lg == 0) red_ml[warp][8 * nt + 2 * lt + c] = make_float2(m[nt][c], l[nt][c]);
            }
        __syncthreads();
        constexpr float BACK = KIND == CACHE_PLAIN ? 1.f : 1.f / slb_codes::VALUE_FACTOR;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float f[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, red_ml[w][8 * nt + 2 * lt + c].x);
                // (a row without a reference has seen nothing, sum 0, or nothing but NaN)
                f[c] = (m[nt][c] == -INFINITY ? l[nt][c] * 0.f : fast_exp2(m[nt][c] - top)) * BACK;
                if (KIND != CACHE_PLAIN && coarse) f[c] *= fast_exp2(lows[warp][8 * nt + 2 * lt + c]);
            }
#pragma unroll
            for (int i = 0; i < F::MT; ++i)
                red_o[(warp * NT * F::MT + nt * F::MT + i) * 32 + lane] =
                    make_float4(acc[nt][i][0] * f[0], acc[nt][i][1] * f[1], acc[nt][i][2] * f[0], acc[nt][i][3] * f[1]);
        }
        __syncthreads();
        // ---- and the blocks' the cluster's: a block finishes a share of the accumulators, which the others send to it (their
        // order in `from` is the order of the sum)
        if (!begun) cluster_wait();
        begun = true;
        constexpr int FOURS = NT * F::MT * 32;
        const int share = FOURS / cs;
        for (int i = tid; i < FOURS; i += 32 * FEW_WARPS) {
            float4 x = red_o[i];
#pragma unroll
            for (int w = 1; w < FEW_WARPS; ++w) {
                const float4 y = red_o[w * FOURS + i];
                x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
            }
            const int owner = i / share;
            store_float4(in_block(from_o + rank * share + (i - owner * share), owner), x);
        }
        for (int i = tid; i < NR * cs; i += 32 * FEW_WARPS) {
            const int r = i % NR;
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; ++w) top = fmaxf(top, red_ml[w][r].x);
#pragma unroll
            for (int w = 0; w < FEW_WARPS; ++w) {
                const float2 ml = red_ml[w][r];
                sum += ml.y * (ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top));
            }
            store_float2(in_block(&from_ml[rank][r], i / NR), make_float2(top, sum));
        }
        if (cs > 1) cluster_sync();                    // (nothing is sent behind it: a block may leave)
        else __syncthreads();
        for (int i = tid; i < share; i += 32 * FEW_WARPS) {
            const int at = rank * share + i, ln = at & 31, mm = (at >> 5) % F::MT, nt = (at >> 5) / F::MT;
            float4 x[MAX_CLUSTER];
#pragma unroll
            for (int k = 0; k < MAX_CLUSTER; ++k) x[k] = k < cs ? from_o[k * share + i] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = 8 * nt + 2 * (ln & 3) + c;
                float top = -INFINITY, sum = 0.f, o[2] = {0.f, 0.f};
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) top = fmaxf(top, k < cs ? from_ml[k][r].x : -INFINITY);
#pragma unroll
                for (int k = 0; k < MAX_CLUSTER; ++k) {
                    if (k >= cs) continue;
                    const float2 ml = from_ml[k][r];
                    const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
                    sum += w * ml.y;
                    o[0] += w * (c ? x[k].y : x[k].x);
                    o[1] += w * (c ? x[k].w : x[k].z);
                }
                if (r >= nrows) continue;
                const int tok = q0 + (row0 + r) / g, h = kvh * g + (row0 + r) % g;
                const size_t slot = ((size_t)tok * a.H + h) * a.parts + part;
                if (a.parts > 1 && ln < 4 && mm == 0) { a.part_ml[2 * slot] = top; a.part_ml[2 * slot + 1] = sum; }
                const float inv = sum != 0.f ? 1.f / sum : 0.f;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int d = F::element(mm, ln >> 2, half);
                    if (a.parts > 1) a.part_o[slot * D + d] = o[half];
                    else reinterpret_cast<bf16*>(a.out)[(size_t)tok * a.ldo + (size_t)h * D + d] = __float2bfloat16_rn(o[half] * inv);
                }
            }
        }
        // (the next tile: what is sent then must not meet this one's reads)
        if (tile + a.tiles < (q_len * g + NR - 1) / NR) {
            if (cs > 1) cluster_sync();
            else __syncthreads();
        }
    }
    if (!begun) cluster_wait();
    pdl_launch_dependents();
}

template <int KIND, int NT>
int few_setup(size_t& smem) {
    constexpr int NR = 8 * NT;
    smem = (size_t)few_ring_bytes<KIND, NT>() + NR * D * 4 + (NT > 1 ? NT * Few<KIND>::KSTEPS * 32 * 8 : 0);
    static unsigned long long configured = 0;          // a bit per device
    return slb_configure(&configured, few_rows_kernel<KIND, NT>, smem);
}
template <int KIND, int NT>
int launch_few(const CacheAttnArgs& in, cudaStream_t st) {
    CacheAttnArgs a = in;
    size_t smem = 0;
    const int rc = few_setup<KIND, NT>(smem);
    if (rc != 0) return rc;
    if ((long long)a.Hkv * a.tiles > 65535) a.tiles = 65535 / a.Hkv;
    if (a.tiles < 1) return SLB_ERR_TOO_LARGE;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.parts * a.cluster), (unsigned)(a.Hkv * a.tiles), (unsigned)a.S);
    cfg.blockDim = dim3(32 * FEW_WARPS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)a.cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = slb_pdl_enabled ? attr : attr + 1;
    cfg.numAttrs = (slb_pdl_enabled ? 1 : 0) + (a.cluster > 1 ? 1 : 0);
    return (int)cudaLaunchKernelEx(&cfg, few_rows_kernel<KIND, NT>, a);
}
// Clusters that the device holds at once, or a negative number.
template <int KIND, int NT>
int few_resident(int cluster) {
    size_t smem = 0;
    if (few_setup<KIND, NT>(smem) != 0) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)cluster, 1024, 1);
    cfg.blockDim = dim3(32 * FEW_WARPS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    return cudaOccupancyMaxActiveClusters(&n, few_rows_kernel<KIND, NT>, &cfg) == cudaSuccess ? n : -1;
}

}  // namespace

int slb_check_cache_attention(const CacheAttnArgs& a) {
    if (a.T <= 0 || a.S <= 0 || a.H <= 0 || a.Hkv <= 0 || a.H % a.Hkv || a.D != D || a.ps <= 0 || a.num_pages <= 0 ||
        a.max_pages <= 0 || a.parts <= 0 || a.tiles <= 0 || !(a.scale > 0.f) || a.kind < 0 || a.kind > 2)
        return SLB_ERR_BAD_ARG;
    if (a.cluster != 1 && a.cluster != 2 && a.cluster != 4 && a.cluster != 8) return SLB_ERR_BAD_ARG;
    if (a.kind != CACHE_PLAIN && (a.ks == nullptr || a.vs == nullptr)) return SLB_ERR_BAD_ARG;
    if (a.mask != nullptr && (a.mask_words <= 0 || (a.window > 0 && a.pos == nullptr))) return SLB_ERR_BAD_ARG;
    if (a.parts > 1 && (a.part_o == nullptr || a.part_ml == nullptr)) return SLB_ERR_BAD_ARG;
    if (a.ldq % 8 || a.ldo % 8 || ((uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)a.k | (uintptr_t)a.v) % 16) return SLB_ERR_BAD_ARG;
    if ((long long)a.num_pages * a.Hkv * a.ps > 0x7fffffffll || a.S > 65535 || (long long)a.parts * a.cluster > 1024)
        return SLB_ERR_TOO_LARGE;
    return 0;
}

extern "C" {

int slb_cache_attention_head_dim(void) { return SLB_HEAD_DIM; }

// Clusters of the kernel for few rows (8 or 16 a block) that the device holds at once; negative: no such kernel.
int slb_cache_attention_few_resident(int kind, int rows, int cluster) {
    if ((rows != 8 && rows != 16) || kind < 0 || kind > 2 || (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8)) return -1;
    if (rows == 8)
        return kind == CACHE_INT8 ? few_resident<CACHE_INT8, 1>(cluster)
               : kind == CACHE_E4M3 ? few_resident<CACHE_E4M3, 1>(cluster) : few_resident<CACHE_PLAIN, 1>(cluster);
    return kind == CACHE_INT8 ? few_resident<CACHE_INT8, 2>(cluster)
           : kind == CACHE_E4M3 ? few_resident<CACHE_E4M3, 2>(cluster) : few_resident<CACHE_PLAIN, 2>(cluster);
}

// rows: query rows a block takes, 8 or 16
int slb_cache_attention_few_bf16(const CacheAttnArgs* a, int rows, cudaStream_t st) {
    const int rc = slb_check_cache_attention(*a);
    if (rc != 0) return rc;
    if (rows == 8)
        return a->kind == CACHE_INT8 ? launch_few<CACHE_INT8, 1>(*a, st)
               : a->kind == CACHE_E4M3 ? launch_few<CACHE_E4M3, 1>(*a, st) : launch_few<CACHE_PLAIN, 1>(*a, st);
    if (rows == 16)
        return a->kind == CACHE_INT8 ? launch_few<CACHE_INT8, 2>(*a, st)
               : a->kind == CACHE_E4M3 ? launch_few<CACHE_E4M3, 2>(*a, st) : launch_few<CACHE_PLAIN, 2>(*a, st);
    return SLB_ERR_BAD_ARG;
}
}
