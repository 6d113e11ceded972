// A key/value cache in 8 bits: written by the step, read back, and attended to by the plain kernel.
//
//   cache_write     a step's q|k|v rows: bias, rotation, queries out, keys and values into the pages as codes with a
//                   scale per (token, kv head).  A token's slot (where it is written) and its position (what it is
//                   rotated by) are two arrays: drafted tokens of one depth share a position.
//   cache_read      rows of requests from the pages, times their scales, in the compute type
//   plain attention (CUDA cores, float32 throughout, any head size up to 256, any kind of cache) and the kernel that
//                   adds up the partial results of key ranges that blocks have shared
//
// The reference's quantisers (servelab/kv_cache/quant.py:54-93) are symmetric per (row, head) too.
#include "cache_codes.cuh"

SLB_DEFINE_STATUS_WORD(cache8_status_word, slb_cache8_status)

namespace {

// ------------------------------------------------------------------------------------------------ writing
template <int KIND> __device__ __forceinline__ float largest_code() { return KIND == CACHE_INT8 ? 127.f : 448.f; }

// Scale of a row and the factor that turns its elements into codes.  A row with an infinity or NaN: scale NaN, factor 0
// (`amax` is NaN or infinite then).
template <int KIND> __device__ __forceinline__ void row_scale(float amax, float& scale, float& inv) {
    scale = fmaxf(amax / largest_code<KIND>(), 1.17549435e-38f);
    inv = 1.f / scale;
    if (!(amax <= 3.402823466e38f)) {
        scale = __int_as_float(0x7fffffff);
        inv = 0.f;
    }
}
// the code of x = element * inv; of NaN (an element of a row whose scale is NaN): 0
template <int KIND> __device__ __forceinline__ unsigned char code_of(float x) {
    if constexpr (KIND == CACHE_INT8) return (unsigned char)(signed char)max(-127, min(127, __float2int_rn(x)));
    else return x == x ? __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : 0;
}
// Four codes of elements times inv, packed (inv 0: a row without codes, zeros).  int8: behind the addition of 1.5 x 2^23 a
// float32's low byte is the integer, rounded to even.
template <int KIND> __device__ __forceinline__ unsigned four_codes(float a, float b, float c, float d, float inv) {
    unsigned r;
    if constexpr (KIND == CACHE_INT8) {
        const float magic = 12582912.f;
        const unsigned lo = __byte_perm(__float_as_uint(fmaf(a, inv, magic)), __float_as_uint(fmaf(b, inv, magic)), 0x0040);
        const unsigned hi = __byte_perm(__float_as_uint(fmaf(c, inv, magic)), __float_as_uint(fmaf(d, inv, magic)), 0x0040);
        r = __byte_perm(lo, hi, 0x5410);
    } else {
        asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
            : "=r"(r) : "f"(a * inv), "f"(b * inv), "f"(c * inv), "f"(d * inv));
    }
    return inv == 0.f ? 0u : r;
}
// larger of two magnitudes, NaN if one is
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// Angle pos * f, reduced to [-pi, pi]: the product is exact in 64 bits, so that far positions turn as exactly as near
// ones (in 32 bits an angle of 1e5 is off by up to 4e-3).  Not EXACT: the product rounded to float32, the angle of the
// models' definition and of the kernels that decode and prompt steps write their keys with (rope_cache.cu).
template <bool EXACT> __device__ __forceinline__ void turn_of(int pos, float f, float& cs, float& sn) {
    if constexpr (!EXACT) {
        sincosf((float)pos * f, &sn, &cs);
        return;
    }
    const double a = (double)pos * (double)f;
    const double r = a - rint(a * 0.15915494309189535) * 6.283185307179586;
    sincosf((float)r, &sn, &cs);
}

// A rotation pair turned.  (Which of the products are rounded is said here, so that pairs come out as rope_cache.cu's do: in its
// kernel for 16-byte accesses, `pieces`, and in the other one.)
__device__ __forceinline__ void turn_pair(float& a, float& b, float cs, float sn, bool pieces) {
    const float x = fmaf(a, cs, -__fmul_rn(b, sn));
    b = pieces ? fmaf(b, cs, __fmul_rn(a, sn)) : fmaf(a, sn, __fmul_rn(b, cs));
    a = x;
}

// First element of the cache rows that token t is written to, and whether it is written at all.
__device__ __forceinline__ bool token_page(const CacheWriteArgs& a, int t, int& page, int& at) {
    const int slot = a.slots != nullptr ? a.slots[t] : a.pos[t];
    const int s = a.seq[t];
    page = -1;
    at = 0;
    if (slot < 0 || slot / a.ps >= a.max_pages || s < 0 || s >= a.num_seqs) {
        atomicCAS(&cache8_status_word, 0, 2);
        return false;
    }
    page = a.table[(size_t)s * a.max_pages + slot / a.ps];
    at = slot % a.ps;
    if (page >= a.num_pages) { atomicCAS(&cache8_status_word, 0, 1); return false; }
    return page >= 0;
}

// 16-byte accesses.  A head is D / (2 VEC) units of 2 VEC elements (VEC = 16 bytes of T): VEC rotation pairs, or 2 VEC
// neighbours that pass through; neighbouring lanes hold a head, so that its largest magnitude is a few shuffles (the units of
// a head are a power of two up to 32).  A thread has one unit, whose bias it keeps, and walks tokens, the next one's elements
// and page on their way while it works; grid (tokens at once, passes over the units).
template <typename T, int KIND, bool EXACT>
__global__ void __launch_bounds__(512, 2) cache_write_vec_kernel(const CacheWriteArgs a, int units_per_head) {
    constexpr int VEC = 16 / (int)sizeof(T);
    extern __shared__ __align__(16) float trig[];          // cos[half], sin[half], of this token and the next
    pdl_launch_dependents();
    pdl_wait();
    const int D = a.D, H = a.H, Hkv = a.Hkv, units = (H + 2 * Hkv) * units_per_head;
    const int half = a.inv_freq != nullptr ? a.rot >> 1 : 0, rot_units = half / VEC;
    const int w0 = blockIdx.y * blockDim.x + threadIdx.x, w = min(w0, units - 1);
    const int j = w / units_per_head, u = w - j * units_per_head;
    const bool is_v = j >= H + Hkv, rot = !is_v && u < rot_units;
    const int ea = rot ? u * VEC : (is_v ? 2 * VEC * u : 2 * half + 2 * VEC * (u - rot_units));
    const int eb = rot ? ea + half : ea + VEC;
    const size_t off = (size_t)j * D;
    const T* x = reinterpret_cast<const T*>(a.qkv) + off;
    int t = blockIdx.x;
    uint4 va = *reinterpret_cast<const uint4*>(x + (size_t)t * a.ld + ea), vb = *reinterpret_cast<const uint4*>(x + (size_t)t * a.ld + eb);
    float ba[VEC], bb[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) ba[e] = bb[e] = 0.f;
    if (a.bias) {
#pragma unroll
        for (int e = 0; e < VEC; e += 4) {
            *reinterpret_cast<float4*>(ba + e) = *reinterpret_cast<const float4*>(a.bias + off + ea + e);
            *reinterpret_cast<float4*>(bb + e) = *reinterpret_cast<const float4*>(a.bias + off + eb + e);
        }
    }
    float freq = (int)threadIdx.x < half ? a.inv_freq[threadIdx.x] : 0.f;
    int pos = a.pos[t], page, at;
    bool have_page = token_page(a, t, page, at);
    for (int turn = 0; t < a.T; turn ^= 1) {
        float* cs = trig + turn * 2 * half;
        float* sn = cs + half;
        if ((int)threadIdx.x < half) turn_of<EXACT>(pos, freq, cs[threadIdx.x], sn[threadIdx.x]);
        for (int i = threadIdx.x + blockDim.x; i < half; i += blockDim.x) turn_of<EXACT>(pos, a.inv_freq[i], cs[i], sn[i]);
        float fa[VEC], fb[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            fa[e] = to_float(reinterpret_cast<const T*>(&va)[e]) + ba[e];
            fb[e] = to_float(reinterpret_cast<const T*>(&vb)[e]) + bb[e];
        }
        const int now = t, now_page = page, now_at = at;
        const bool now_there = have_page;
        t += gridDim.x;
        if (t < a.T) {
            va = *reinterpret_cast<const uint4*>(x + (size_t)t * a.ld + ea);
            vb = *reinterpret_cast<const uint4*>(x + (size_t)t * a.ld + eb);
            pos = a.pos[t];
            have_page = token_page(a, t, page, at);
        }
        __syncthreads();                                   // (one a token: the other half of `trig` is read meanwhile)
        if (rot) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                const float4 c4 = *reinterpret_cast<const float4*>(cs + ea + e);
                const float4 s4 = *reinterpret_cast<const float4*>(sn + ea + e);
                const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) turn_pair(fa[e + k], fb[e + k], c[k], s[k], true);
            }
        }
        float scale = 1.f, inv = 1.f;
        if constexpr (KIND != CACHE_PLAIN) {
            float amax = 0.f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) amax = max_nan(amax, max_nan(fabsf(fa[e]), fabsf(fb[e])));
            for (int o = units_per_head >> 1; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            row_scale<KIND>(amax, scale, inv);
        }
        if (w0 >= units) continue;
        if (j < H || KIND == CACHE_PLAIN) {
            if (j >= H && !now_there) continue;
            const int g = is_v ? j - H - Hkv : j - H;
            T* dst = j < H ? reinterpret_cast<T*>(a.q_out) + (size_t)now * a.ldq + off
                           : reinterpret_cast<T*>(is_v ? a.v : a.k) + (((size_t)now_page * Hkv + g) * a.ps + now_at) * D;
            __align__(16) T oa[VEC], ob[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) { oa[e] = from_float<T>(fa[e]); ob[e] = from_float<T>(fb[e]); }
            *reinterpret_cast<uint4*>(dst + ea) = *reinterpret_cast<const uint4*>(oa);
            *reinterpret_cast<uint4*>(dst + eb) = *reinterpret_cast<const uint4*>(ob);
        } else if (now_there) {
            const int g = is_v ? j - H - Hkv : j - H;
            const size_t row = ((size_t)now_page * Hkv + g) * a.ps + now_at;
            unsigned char* dst = reinterpret_cast<unsigned char*>(is_v ? a.v : a.k) + row * D;
            unsigned ca[VEC / 4], cb[VEC / 4];
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
                ca[e / 4] = four_codes<KIND>(fa[e], fa[e + 1], fa[e + 2], fa[e + 3], inv);
                cb[e / 4] = four_codes<KIND>(fb[e], fb[e + 1], fb[e + 2], fb[e + 3], inv);
            }
            if constexpr (VEC == 8) {
                *reinterpret_cast<uint2*>(dst + ea) = make_uint2(ca[0], ca[1]);
                *reinterpret_cast<uint2*>(dst + eb) = make_uint2(cb[0], cb[1]);
            } else {
                *reinterpret_cast<unsigned*>(dst + ea) = ca[0];
                *reinterpret_cast<unsigned*>(dst + eb) = cb[0];
            }
            if (u == 0) (is_v ? a.vs : a.ks)[row] = scale;
        }
    }
}

// The same for any even head size up to 1,024: a warp per head, element pairs over its lanes.
template <typename T, int KIND, bool EXACT>
__global__ void cache_write_kernel(const CacheWriteArgs a, bool pieces) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int MOST = 16;                               // pairs a lane holds
    const int t = blockIdx.x, lane = threadIdx.x & 31, D = a.D, H = a.H, Hkv = a.Hkv;
    const int half = a.inv_freq != nullptr ? a.rot >> 1 : 0;
    const int pos = a.pos[t];
    int page, at;
    const bool have_page = token_page(a, t, page, at);
    const T* x = reinterpret_cast<const T*>(a.qkv) + (size_t)t * a.ld;
    for (int j = threadIdx.x >> 5; j < H + 2 * Hkv; j += blockDim.x >> 5) {
        const bool is_v = j >= H + Hkv;
        const size_t off = (size_t)j * D;
        float fa[MOST], fb[MOST];
        float amax = 0.f;
#pragma unroll
        for (int n = 0; n < MOST; ++n) {
            const int i = lane + 32 * n;
            fa[n] = fb[n] = 0.f;
            if (i >= D / 2) continue;
            const bool rot = !is_v && i < half;
            const int ea = rot ? i : is_v ? 2 * i : 2 * half + 2 * (i - half), eb = rot ? i + half : ea + 1;
            fa[n] = to_float(x[off + ea]);
            fb[n] = to_float(x[off + eb]);
            if (a.bias) { fa[n] += a.bias[off + ea]; fb[n] += a.bias[off + eb]; }
            if (rot) {
                float cs, sn;
                turn_of<EXACT>(pos, a.inv_freq[i], cs, sn);
                turn_pair(fa[n], fb[n], cs, sn, pieces);
            }
            amax = max_nan(amax, max_nan(fabsf(fa[n]), fabsf(fb[n])));
        }
        float scale = 1.f, inv = 1.f;
        if constexpr (KIND != CACHE_PLAIN) {
            for (int o = 16; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            row_scale<KIND>(amax, scale, inv);
        }
        const int g = is_v ? j - H - Hkv : j - H;
        const size_t row = ((size_t)(have_page ? page : 0) * Hkv + (j < H ? 0 : g)) * a.ps + at;
        if (j >= H && !have_page) continue;
#pragma unroll
        for (int n = 0; n < MOST; ++n) {
            const int i = lane + 32 * n;
            if (i >= D / 2) continue;
            const bool rot = !is_v && i < half;
            const int ea = rot ? i : is_v ? 2 * i : 2 * half + 2 * (i - half), eb = rot ? i + half : ea + 1;
            if (j < H || KIND == CACHE_PLAIN) {
                T* dst = j < H ? reinterpret_cast<T*>(a.q_out) + (size_t)t * a.ldq + off
                               : reinterpret_cast<T*>(is_v ? a.v : a.k) + row * D;
                dst[ea] = from_float<T>(fa[n]);
                dst[eb] = from_float<T>(fb[n]);
            } else {
                unsigned char* dst = reinterpret_cast<unsigned char*>(is_v ? a.v : a.k) + row * D;
                dst[ea] = code_of<KIND>(fa[n] * inv);
                dst[eb] = code_of<KIND>(fb[n] * inv);
            }
        }
        if (KIND != CACHE_PLAIN && j >= H && lane == 0) (is_v ? a.vs : a.ks)[row] = scale;
    }
}

template <typename T, int KIND, bool EXACT>
int launch_cache_write_turned(const CacheWriteArgs& a, cudaStream_t st) {
    constexpr int VEC = 16 / (int)sizeof(T);
    const int rot = a.inv_freq != nullptr ? a.rot : 0;
    const int per_head = a.D / (2 * VEC);
    const bool pieces = a.D % (2 * VEC) == 0 && rot % (2 * VEC) == 0 && a.ld % VEC == 0 && a.ldq % VEC == 0 &&
                        ((uintptr_t)a.qkv | (uintptr_t)a.q_out | (uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0;
    const bool vec_ok = pieces && per_head <= 32 && (per_head & (per_head - 1)) == 0 && (uintptr_t)a.bias % 16 == 0;
    const int heads = a.H + 2 * a.Hkv;
    if (!vec_ok) return slb_launch(cache_write_kernel<T, KIND, EXACT>, dim3(a.T), dim3(32 * (heads < 8 ? heads : 8)), 0, st, a, pieces);
    const int units = heads * per_head;
    const int passes = (units + 511) / 512;
    const int threads = ((units + passes - 1) / passes + 31) / 32 * 32;      // (whole heads: 32 is a multiple of per_head)
    // as many blocks as the SMs hold (64 registers a thread): every block has a token at least
    const int at_once = slb_num_sms() * (1024 / threads);
    return slb_launch(cache_write_vec_kernel<T, KIND, EXACT>, dim3(a.T < at_once ? a.T : at_once, passes), dim3(threads),
                      (size_t)rot * 2 * sizeof(float), st, a, per_head);
}
template <typename T, int KIND> int launch_cache_write(const CacheWriteArgs& a, cudaStream_t st) {
    return a.exact ? launch_cache_write_turned<T, KIND, true>(a, st) : launch_cache_write_turned<T, KIND, false>(a, st);
}

// ------------------------------------------------------------------------------------------------ reading back
// Slots and pages of output rows n0 .. n0 + 31, looked up by a warp, lane r for row n0 + r, into `where`: x the slot (-1: the row
// belongs to no request), y the page (-1: none, or one outside the cache).  A row's request is the number of those that end at or
// before it, counted from the lanes that hold their ends.
constexpr int READ_ROWS = 32;
__device__ __forceinline__ void look_rows_up(const CacheReadArgs& a, int n0, int2* where) {
    const int lane = threadIdx.x & 31, n = n0 + lane;
    int s = 0, from = a.cu[0];
    for (int s0 = 0; s0 < a.num_seqs; s0 += 32) {
        const int end = s0 + lane < a.num_seqs ? a.cu[s0 + lane + 1] : 0x7fffffff;
#pragma unroll 8
        for (int i = 0; i < 32; ++i) {
            const int e = __shfl_sync(0xffffffffu, end, i);
            s += e <= n ? 1 : 0;
            from = e <= n ? e : from;
        }
    }
    int slot = -1, page = -1;
    if (s < a.num_seqs && n < a.rows && n >= from) {
        slot = a.first[s] + (n - from);
        if (slot >= 0 && slot / a.ps < a.max_pages) page = a.table[(size_t)s * a.max_pages + slot / a.ps];
        if (page >= a.num_pages) {
            atomicCAS(&cache8_status_word, 0, 1);
            page = -1;
        }
        slot = max(slot, 0);
    }
    where[lane] = make_int2(slot, page);
}

// 16 bytes of T: the codes of that many elements times their scale.  (By way of float16, which holds them exactly: the conversion
// of bytes to float32 runs at an eighth of the rate.)
template <typename T, int KIND> __device__ __forceinline__ uint4 scaled_codes(uint2 codes, float scale) {
    float2 v[4];
#pragma unroll
    for (int i = 0; i < (sizeof(T) == 2 ? 2 : 1); ++i) {
        unsigned lo, hi;
        slb_codes::four<KIND == CACHE_PLAIN ? CACHE_INT8 : KIND>(i ? codes.y : codes.x, lo, hi);
        float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        if (slb_codes::swaps<KIND>()) { const float x = a.y; a.y = b.x; b.x = x; }
        v[2 * i] = make_float2(a.x * scale, a.y * scale);
        v[2 * i + 1] = make_float2(b.x * scale, b.y * scale);
    }
    if constexpr (sizeof(T) == 4) {
        return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
    } else {
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(v[i].x, v[i].y);
            w[i] = *reinterpret_cast<const unsigned*>(&x);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// A block copies 32 rows that its first warp has looked up; a thread 16 bytes of output of K and of V at a time (neighbouring
// threads: pieces of a row, then the kv heads), AT_ONCE of them on their way.  Pieces go by the output: with 16 bytes of codes
// a thread, 32 or 64 bytes apart in the output, 28,000 rows took 25 to 39 us.
template <typename T, int KIND>
__global__ void __launch_bounds__(256, 4) cache_read_kernel(const CacheReadArgs a, int pieces, int piece_shift, int row_shift) {
    constexpr int N = 16 / (int)sizeof(T);                 // elements of a piece
    constexpr int AT_ONCE = 4;
    __shared__ int2 where[READ_ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const int per_row = a.Hkv * pieces, n0 = blockIdx.x * READ_ROWS, shift = page_shift(a.ps);
    if (threadIdx.x < 32) look_rows_up(a, n0, where);
    __syncthreads();
    for (int e0 = threadIdx.x; e0 < READ_ROWS * per_row; e0 += 256 * AT_ONCE) {
        uint4 ck[AT_ONCE], cv[AT_ONCE];                    // (of codes the first 8 or 4 bytes)
        float sk[AT_ONCE], sv[AT_ONCE];
        int n[AT_ONCE], to[AT_ONCE];                       // output row (-1: none), first element within it
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int e = min(e0 + 256 * i, READ_ROWS * per_row - 1);
            const int r = row_shift >= 0 ? e >> row_shift : e / per_row, in = e - r * per_row;
            const int h = piece_shift >= 0 ? in >> piece_shift : in / pieces, first = (in - h * pieces) * N;
            const int2 at = where[r];
            n[i] = at.x >= 0 && e0 + 256 * i < READ_ROWS * per_row ? n0 + r : -1;
            to[i] = h * a.D + first;
            ck[i] = cv[i] = make_uint4(0, 0, 0, 0);
            sk[i] = sv[i] = 0.f;
            if (n[i] >= 0 && at.y >= 0) {
                const size_t row = ((size_t)at.y * a.Hkv + h) * a.ps + (shift >= 0 ? at.x & (a.ps - 1) : at.x % a.ps);
                const size_t el = row * a.D + first;
                if constexpr (KIND == CACHE_PLAIN) {
                    ck[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.k) + el);
                    cv[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.v) + el);
                } else {
                    const unsigned char *k = reinterpret_cast<const unsigned char*>(a.k) + el, *v = reinterpret_cast<const unsigned char*>(a.v) + el;
                    if constexpr (N == 8) {
                        const uint2 x = *reinterpret_cast<const uint2*>(k), y = *reinterpret_cast<const uint2*>(v);
                        ck[i].x = x.x; ck[i].y = x.y; cv[i].x = y.x; cv[i].y = y.y;
                    } else {
                        ck[i].x = *reinterpret_cast<const unsigned*>(k);
                        cv[i].x = *reinterpret_cast<const unsigned*>(v);
                    }
                    sk[i] = a.ks[row];
                    sv[i] = a.vs[row];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (n[i] < 0) continue;
            T* dk = reinterpret_cast<T*>(a.k_out) + (size_t)n[i] * a.ldk + to[i];
            T* dv = reinterpret_cast<T*>(a.v_out) + (size_t)n[i] * a.ldv + to[i];
            *reinterpret_cast<uint4*>(dk) = KIND == CACHE_PLAIN ? ck[i] : scaled_codes<T, KIND>(make_uint2(ck[i].x, ck[i].y), sk[i]);
            *reinterpret_cast<uint4*>(dv) = KIND == CACHE_PLAIN ? cv[i] : scaled_codes<T, KIND>(make_uint2(cv[i].x, cv[i].y), sv[i]);
        }
    }
}

// any head size and alignment: an element a thread
template <typename T, int KIND>
__global__ void __launch_bounds__(256) cache_read_any_kernel(const CacheReadArgs a) {
    __shared__ int2 where[READ_ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const int per_row = a.Hkv * a.D, n0 = blockIdx.x * READ_ROWS;
    if (threadIdx.x < 32) look_rows_up(a, n0, where);
    __syncthreads();
    for (int r = 0; r < READ_ROWS; ++r) {
        const int2 at = where[r];
        if (at.x < 0) continue;
        for (int in = threadIdx.x; in < per_row; in += blockDim.x) {
            const int h = in / a.D, d = in - h * a.D;
            float ok = 0.f, ov = 0.f;
            if (at.y >= 0) {
                const size_t row = ((size_t)at.y * a.Hkv + h) * a.ps + at.x % a.ps;
                ok = cache_code<T, KIND>(a.k, row * a.D + d);
                ov = cache_code<T, KIND>(a.v, row * a.D + d);
                if constexpr (KIND != CACHE_PLAIN) { ok *= a.ks[row]; ov *= a.vs[row]; }
            }
            reinterpret_cast<T*>(a.k_out)[(size_t)(n0 + r) * a.ldk + in] = from_float<T>(ok);
            reinterpret_cast<T*>(a.v_out)[(size_t)(n0 + r) * a.ldv + in] = from_float<T>(ov);
        }
    }
}

template <typename T, int KIND>
int launch_cache_read(const CacheReadArgs& a, cudaStream_t st) {
    constexpr int N = 16 / (int)sizeof(T);
    const bool vec_ok = a.D % N == 0 && a.ldk % N == 0 && a.ldv % N == 0 &&
                        ((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.k_out | (uintptr_t)a.v_out) % 16 == 0;
    if ((long long)a.Hkv * a.D > (1 << 24)) return SLB_ERR_TOO_LARGE;
    const dim3 grid((unsigned)(((long long)a.rows + READ_ROWS - 1) / READ_ROWS));
    if (!vec_ok) return slb_launch(cache_read_any_kernel<T, KIND>, grid, dim3(256), 0, st, a);
    auto shift_of = [](int x) { return (x & (x - 1)) == 0 ? 31 - __builtin_clz((unsigned)x) : -1; };
    const int pieces = a.D / N;
    return slb_launch(cache_read_kernel<T, KIND>, grid, dim3(256), 0, st, a, pieces, shift_of(pieces), shift_of(a.Hkv * pieces));
}

// ------------------------------------------------------------------------------------------------ plain attention
constexpr int PA_ROWS = 8, PA_WARPS = 4;

// Elements e .. e + 3 (e a multiple of 4) of 16 bytes of a cached row, as floats without their scale.
template <typename T, int KIND> __device__ __forceinline__ float4 four_of(const uint4& x, int e) {
    const unsigned w[4] = {x.x, x.y, x.z, x.w};
    if constexpr (KIND != CACHE_PLAIN) {
        unsigned lo, hi;
        slb_codes::four<KIND>(w[e >> 2], lo, hi);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        return slb_codes::swaps<KIND>() ? make_float4(a.x, b.x, a.y, b.y) : make_float4(a.x, a.y, b.x, b.y);
    } else if constexpr (sizeof(T) == 4) {
        return make_float4(__uint_as_float(w[0]), __uint_as_float(w[1]), __uint_as_float(w[2]), __uint_as_float(w[3]));
    } else {
        const unsigned a = w[e >> 1], b = w[(e >> 1) + 1];
        return make_float4(__uint_as_float(a << 16), __uint_as_float(a & 0xffff0000u), __uint_as_float(b << 16), __uint_as_float(b & 0xffff0000u));
    }
}

// An element of a cached row as it lies in memory, in a register of its own, and its value.
template <typename T, int KIND> __device__ __forceinline__ int raw_element(const void* base, size_t i) {
    if constexpr (KIND == CACHE_INT8) return reinterpret_cast<const signed char*>(base)[i];
    else if constexpr (KIND == CACHE_E4M3) return reinterpret_cast<const unsigned char*>(base)[i];
    else if constexpr (sizeof(T) == 4) return reinterpret_cast<const int*>(base)[i];
    else return reinterpret_cast<const unsigned short*>(base)[i];
}
template <typename T, int KIND> __device__ __forceinline__ float raw_value(int x) {
    if constexpr (KIND == CACHE_INT8) return __int_as_float(x + 0x4B400000) - 12582912.f;     // (exact: 1.5 x 2^23 + x)
    else if constexpr (KIND == CACHE_E4M3) return e4m3_float((unsigned char)x);
    else if constexpr (sizeof(T) == 4) return __int_as_float(x);
    else return __uint_as_float((unsigned)x << 16);
}

// Block (range of keys, kv head, tiles of rows of a request): eight query rows share the keys.  A warp takes 32 keys at a
// time: a lane computes the eight scores of its key (the queries are read from shared memory by all lanes at once),
// then the lanes hold the head's elements and every key's values are read once for the eight rows.  Loads are what it waits
// for: 16 bytes each and several of them on their way, the values' before their weights are known (8 drafts over 700 keys in
// float32, 14 heads of 64: 17.0 us with the parts' sum; an element at a time 25.2).
template <typename T, int KIND, int DL>                    // DL: elements of a head a lane holds, D <= 32 DL
__global__ void __launch_bounds__(32 * PA_WARPS, 2) plain_cache_attention_kernel(const CacheAttnArgs a) {
    __shared__ __align__(16) float qs[PA_ROWS][32 * DL];
    __shared__ __align__(16) float ps[PA_WARPS][PA_ROWS][32];
    constexpr int PIECE = KIND == CACHE_PLAIN ? 16 / (int)sizeof(T) : 16;      // elements in 16 bytes
    constexpr int GROUP = DL <= 2 ? (KIND == CACHE_PLAIN ? 8 : 4) : DL <= 4 ? 4 : 2;
    constexpr int AHEAD = KIND == CACHE_PLAIN && sizeof(T) == 4 ? 8 : 4;
    __shared__ float red_m[PA_WARPS][PA_ROWS], red_l[PA_WARPS][PA_ROWS];
    __shared__ float red_o[PA_WARPS][32 * DL];
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = a.D;
    const int part = blockIdx.x, s = blockIdx.z;
    const int kvh = blockIdx.y % a.Hkv, g = a.H / a.Hkv;
    int q0 = a.cu_q[s], q1 = a.cu_q[s + 1];
    clamp_span(a.T, q0, q1);
    const int q_len = q1 - q0, ctx = a.ctx_len[s], base = ctx - q_len;
    const int* table = a.table + (size_t)s * a.max_pages;
    const int shift = page_shift(a.ps);
    const char* kbase = reinterpret_cast<const char*>(a.k);
    const bool vec = D % PIECE == 0 && (uintptr_t)kbase % 16 == 0;
    for (int tile = blockIdx.y / a.Hkv; (long long)tile * PA_ROWS < (long long)q_len * g; tile += a.tiles) {
        const int row0 = tile * PA_ROWS, nrows = min(PA_ROWS, q_len * g - row0);
        bool far = false;                                  // an element is so large that sums with codes may overflow
        __syncthreads();
        for (int i = threadIdx.x; i < PA_ROWS * 32 * DL; i += blockDim.x) {
            const int r = i / (32 * DL), d = i - r * (32 * DL);
            float x = 0.f;
            if (r < nrows && d < D) {
                const int tok = q0 + (row0 + r) / g, h = kvh * g + (row0 + r) % g;
                x = to_float(reinterpret_cast<const T*>(a.q)[(size_t)tok * a.ldq + (size_t)h * D + d]);
            }
            qs[r][d] = x;
            far |= fabsf(x) > 1.2379400392853803e27f;      // 2^90
        }
        float moved = 1.f;
        if (KIND == CACHE_PLAIN) {
            __syncthreads();
        } else if (__syncthreads_or(far)) {                // (their keys' scales are as small: 2^40 moves there)
            for (int i = threadIdx.x; i < PA_ROWS * 32 * DL; i += blockDim.x) qs[i / (32 * DL)][i % (32 * DL)] *= 9.094947017729282e-13f;
            moved = 1099511627776.f;
            __syncthreads();
        }
        RowView view[PA_ROWS];
        int least = ctx;                                   // first slot that a row of the tile sees
#pragma unroll
        for (int r = 0; r < PA_ROWS; ++r) {
            const int local = (row0 + min(r, nrows - 1)) / g;
            view[r] = row_view(a, base, q0 + local, local);
            least = min(least, max(0, min(view[r].lo, base)));
        }
        const int last = a.mask != nullptr ? ctx : min(ctx, base + (row0 + nrows - 1) / g + 1);
        const int per = ((last - least + a.parts - 1) / a.parts + 31) / 32 * 32;
        const int kbeg = least + min(part * per, max(0, last - least)), kend = min(last, kbeg + per);
        float m[PA_ROWS], l[PA_ROWS], acc[PA_ROWS][DL];
#pragma unroll
        for (int r = 0; r < PA_ROWS; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.f;
#pragma unroll
            for (int e = 0; e < DL; ++e) acc[r][e] = 0.f;
        }
        int ahead[GROUP][DL];                              // (turned into floats where they are used: that would wait for them)
        auto bring_values = [&](int row, int i0) {         // of the warp's keys i0 .. i0 + GROUP - 1 (row -1: none)
#pragma unroll
            for (int i = 0; i < GROUP; ++i) {
                const int vrow = __shfl_sync(0xffffffffu, row, i0 + i);
#pragma unroll
                for (int e = 0; e < DL; ++e) {
                    const int d = lane + 32 * e;
                    ahead[i][e] = vrow >= 0 && d < D ? raw_element<T, KIND>(a.v, (size_t)vrow * D + d) : 0;
                }
            }
        };
        for (int k0 = kbeg + warp * 32; k0 < kend; k0 += PA_WARPS * 32) {
            const int key = k0 + lane;
            const int row = cache_row(table_entry(table, a.max_pages, key, a.ps, shift, key < kend), key, a.ps, shift, a.num_pages,
                                      a.Hkv, kvh, &cache8_status_word);
            float sc[PA_ROWS];
#pragma unroll
            for (int r = 0; r < PA_ROWS; ++r) sc[r] = 0.f;
            float vscale = 1.f;
            bring_values(row, 0);
            if (row >= 0) {
                const size_t at = (size_t)row * D;
                if (vec) {
                    for (int d0 = 0; d0 < D; d0 += PIECE * AHEAD) {
                        uint4 x[AHEAD];
#pragma unroll
                        for (int c = 0; c < AHEAD; ++c)
                            if (d0 + PIECE * c < D) x[c] = *reinterpret_cast<const uint4*>(kbase + (at + d0 + PIECE * c) * (16 / PIECE));
#pragma unroll
                        for (int c = 0; c < AHEAD; ++c) {
                            if (d0 + PIECE * c >= D) continue;
#pragma unroll
                            for (int e = 0; e < PIECE; e += 4) {
                                const float4 y = four_of<T, KIND>(x[c], e);
#pragma unroll
                                for (int r = 0; r < PA_ROWS; ++r) {
                                    const float4 q = *reinterpret_cast<const float4*>(&qs[r][d0 + PIECE * c + e]);
                                    sc[r] = fmaf(q.w, y.w, fmaf(q.z, y.z, fmaf(q.y, y.y, fmaf(q.x, y.x, sc[r]))));
                                }
                            }
                        }
                    }
                } else {
                    for (int d = 0; d < D; ++d) {
                        const float x = cache_code<T, KIND>(a.k, at + d);
#pragma unroll
                        for (int r = 0; r < PA_ROWS; ++r) sc[r] = fmaf(qs[r][d], x, sc[r]);
                    }
                }
                float kscale = a.scale * 1.4426950408889634f;
                if constexpr (KIND != CACHE_PLAIN) { kscale = kscale * moved * a.ks[row]; vscale = a.vs[row]; }
#pragma unroll
                for (int r = 0; r < PA_ROWS; ++r) sc[r] = __fmul_rn(sc[r], kscale);   // (the maximum and the exponents go by this number)
            }
#pragma unroll
            for (int r = 0; r < PA_ROWS; ++r) {
                // (a slot without a page holds zeros: score 0, value 0)
                const bool seen = r < nrows && key < kend && row_sees(a, view[r], key, base, q0);
                const float x = seen ? sc[r] : -INFINITY;
                const float top = fmaxf(m[r], warp_max(x));
                const float ref = top == -INFINITY ? 0.f : top;
                const float alpha = exp2f(m[r] - ref);
                const float p = seen ? exp2f(x - ref) : 0.f;
                m[r] = top;
                l[r] = l[r] * alpha + p;                   // (a lane's keys; added up at the end)
                ps[warp][r][lane] = seen ? p * vscale : 0.f;
#pragma unroll
                for (int e = 0; e < DL; ++e) acc[r][e] *= alpha;
            }
            __syncwarp();
            const int n = min(32, kend - k0);
            for (int i0 = 0; i0 < n; i0 += GROUP) {        // the next keys' values are on their way meanwhile
                float x[GROUP][DL];
#pragma unroll
                for (int i = 0; i < GROUP; ++i)
#pragma unroll
                    for (int e = 0; e < DL; ++e) x[i][e] = raw_value<T, KIND>(ahead[i][e]);
                if (i0 + GROUP < n) bring_values(row, i0 + GROUP);
#pragma unroll
                for (int r = 0; r < PA_ROWS; ++r) {
#pragma unroll
                    for (int i = 0; i < GROUP; ++i) {
                        const float p = ps[warp][r][i0 + i];
#pragma unroll
                        for (int e = 0; e < DL; ++e) acc[r][e] = p != 0.f ? fmaf(p, x[i][e], acc[r][e]) : acc[r][e];  // (0 x NaN: a key that is not seen)
                    }
                }
            }
            __syncwarp();
        }
#pragma unroll
        for (int r = 0; r < PA_ROWS; ++r) {
            l[r] = warp_sum(l[r]);
            if (lane == 0) { red_m[warp][r] = m[r]; red_l[warp][r] = l[r]; }
        }
        for (int r = 0; r < nrows; ++r) {
            __syncthreads();
            float top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < PA_WARPS; ++w) top = fmaxf(top, red_m[w][r]);
            const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < PA_WARPS; ++w) sum += red_l[w][r] * exp2f(red_m[w][r] - ref);
            const float mine = exp2f(red_m[warp][r] - ref);
#pragma unroll
            for (int e = 0; e < DL; ++e) {
                float x = 0.f;
#pragma unroll
                for (int q = 0; q < PA_ROWS; ++q) x = q == r ? acc[q][e] : x;
                red_o[warp][lane + 32 * e] = x * mine;
            }
            __syncthreads();
            const int tok = q0 + (row0 + r) / g, h = kvh * g + (row0 + r) % g;
            for (int d = threadIdx.x; d < D; d += blockDim.x) {
                float x = 0.f;
#pragma unroll
                for (int w = 0; w < PA_WARPS; ++w) x += red_o[w][d];
                if (a.parts > 1) {
                    const size_t slot = ((size_t)tok * a.H + h) * a.parts + part;
                    a.part_o[slot * D + d] = x;
                    if (d == 0) { a.part_ml[2 * slot] = top; a.part_ml[2 * slot + 1] = sum; }
                } else {
                    reinterpret_cast<T*>(a.out)[(size_t)tok * a.ldo + (size_t)h * D + d] = from_float<T>(sum != 0.f ? x / sum : 0.f);
                }
            }
        }
    }
}

// out = the parts of a row added up, each at its reference; a row behind the last request's is left as it is.  A warp per row.
template <typename T>
__global__ void __launch_bounds__(256) cache_attention_join_kernel(const CacheAttnArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= (long long)a.T * a.H) return;
    const int tok = (int)(row / a.H), h = (int)(row - (long long)tok * a.H);
    if (tok >= a.cu_q[a.S]) return;
    const float* ml = a.part_ml + (size_t)row * a.parts * 2;
    const float* o = a.part_o + (size_t)row * a.parts * a.D;
    float top = -INFINITY;
    for (int p = lane; p < a.parts; p += 32) top = fmaxf(top, ml[2 * p]);
    top = warp_max(top);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f, weight[2] = {0.f, 0.f};               // a lane's: of parts lane and lane + 32
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int p = lane + 32 * i;
        if (p < a.parts) {
            weight[i] = exp2f(ml[2 * p] - ref);
            sum += ml[2 * p + 1] * weight[i];
        }
    }
    sum = warp_sum(sum);
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    T* out = reinterpret_cast<T*>(a.out) + (size_t)tok * a.ldo + (size_t)h * a.D;
    for (int d0 = 0; d0 < a.D; d0 += 32) {
        const int d = d0 + lane;
        float x = 0.f;
        for (int p0 = 0; p0 < a.parts; p0 += 8) {          // eight parts are on their way at once
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = p0 + i < a.parts && d < a.D ? o[(size_t)(p0 + i) * a.D + d] : 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = __shfl_sync(0xffffffffu, p0 < 32 ? weight[0] : weight[1], (p0 + i) & 31);
                if (p0 + i < a.parts) x += w * y[i];
            }
        }
        if (d < a.D) out[d] = from_float<T>(x * inv);
    }
}

int check_attn(const CacheAttnArgs& a) {
    if (a.T <= 0 || a.S <= 0 || a.H <= 0 || a.Hkv <= 0 || a.H % a.Hkv || a.D <= 0 || a.ps <= 0 || a.num_pages <= 0 ||
        a.max_pages <= 0 || a.parts <= 0 || a.tiles <= 0 || !(a.scale > 0.f) || a.kind < 0 || a.kind > 2)
        return SLB_ERR_BAD_ARG;
    if (a.kind != CACHE_PLAIN && (a.ks == nullptr || a.vs == nullptr)) return SLB_ERR_BAD_ARG;
    if (a.mask != nullptr && (a.mask_words <= 0 || (a.window > 0 && a.pos == nullptr))) return SLB_ERR_BAD_ARG;
    if (a.parts > 1 && (a.part_o == nullptr || a.part_ml == nullptr)) return SLB_ERR_BAD_ARG;
    if (a.parts > 64) return SLB_ERR_BAD_ARG;              // (the joining kernel has two weights a lane)
    if (a.D > 256 || (long long)a.num_pages * a.Hkv * a.ps > 0x7fffffffll || a.S > 65535) return SLB_ERR_TOO_LARGE;
    return 0;
}

template <typename T, int KIND>
int launch_plain_attention(const CacheAttnArgs& in, cudaStream_t st) {
    CacheAttnArgs a = in;
    if ((long long)a.Hkv * a.tiles > 65535) a.tiles = 65535 / a.Hkv;
    if (a.tiles < 1) return SLB_ERR_TOO_LARGE;
    const dim3 grid(a.parts, a.Hkv * a.tiles, a.S), block(32 * PA_WARPS);
    if (a.D <= 64) return slb_launch_after(plain_cache_attention_kernel<T, KIND, 2>, grid, block, 0, st, a);
    if (a.D <= 128) return slb_launch_after(plain_cache_attention_kernel<T, KIND, 4>, grid, block, 0, st, a);
    return slb_launch_after(plain_cache_attention_kernel<T, KIND, 8>, grid, block, 0, st, a);
}

}  // namespace

extern "C" {

static int check_write(const CacheWriteArgs& a) {
    if (a.H <= 0 || a.Hkv <= 0 || a.D <= 0 || (a.D & 1) || a.ps <= 0 || a.max_pages <= 0 || a.num_pages <= 0 ||
        a.num_seqs <= 0 || a.rot < 0 || a.rot > a.D || (a.rot & 1) || a.kind < 0 || a.kind > 2)
        return SLB_ERR_BAD_ARG;
    if (a.kind != CACHE_PLAIN && (a.ks == nullptr || a.vs == nullptr)) return SLB_ERR_BAD_ARG;
    if (a.D > 1024) return SLB_ERR_TOO_LARGE;
    return 0;
}
int slb_cache_write_f32(const CacheWriteArgs* a, cudaStream_t st) {
    if (a->T <= 0) return 0;
    const int rc = check_write(*a);
    if (rc != 0) return rc;
    return a->kind == CACHE_INT8 ? launch_cache_write<float, CACHE_INT8>(*a, st)
           : a->kind == CACHE_E4M3 ? launch_cache_write<float, CACHE_E4M3>(*a, st) : launch_cache_write<float, CACHE_PLAIN>(*a, st);
}
int slb_cache_write_bf16(const CacheWriteArgs* a, cudaStream_t st) {
    if (a->T <= 0) return 0;
    const int rc = check_write(*a);
    if (rc != 0) return rc;
    return a->kind == CACHE_INT8 ? launch_cache_write<bf16, CACHE_INT8>(*a, st)
           : a->kind == CACHE_E4M3 ? launch_cache_write<bf16, CACHE_E4M3>(*a, st) : launch_cache_write<bf16, CACHE_PLAIN>(*a, st);
}

static int check_read(const CacheReadArgs& a) {
    if (a.Hkv <= 0 || a.D <= 0 || a.ps <= 0 || a.max_pages <= 0 || a.num_pages <= 0 || a.num_seqs <= 0 || a.kind < 0 || a.kind > 2)
        return SLB_ERR_BAD_ARG;
    if (a.kind != CACHE_PLAIN && (a.ks == nullptr || a.vs == nullptr)) return SLB_ERR_BAD_ARG;
    return 0;
}
int slb_cache_read_f32(const CacheReadArgs* a, cudaStream_t st) {
    if (a->rows <= 0) return 0;
    const int rc = check_read(*a);
    if (rc != 0) return rc;
    return a->kind == CACHE_INT8 ? launch_cache_read<float, CACHE_INT8>(*a, st)
           : a->kind == CACHE_E4M3 ? launch_cache_read<float, CACHE_E4M3>(*a, st) : launch_cache_read<float, CACHE_PLAIN>(*a, st);
}
int slb_cache_read_bf16(const CacheReadArgs* a, cudaStream_t st) {
    if (a->rows <= 0) return 0;
    const int rc = check_read(*a);
    if (rc != 0) return rc;
    return a->kind == CACHE_INT8 ? launch_cache_read<bf16, CACHE_INT8>(*a, st)
           : a->kind == CACHE_E4M3 ? launch_cache_read<bf16, CACHE_E4M3>(*a, st) : launch_cache_read<bf16, CACHE_PLAIN>(*a, st);
}

// query rows that a block of the plain attention takes
int slb_cache_attention_plain_rows(void) { return PA_ROWS; }

int slb_cache_attention_plain_f32(const CacheAttnArgs* a, cudaStream_t st) {
    const int rc = check_attn(*a);
    if (rc != 0) return rc;
    return a->kind == CACHE_INT8 ? launch_plain_attention<float, CACHE_INT8>(*a, st)
           : a->kind == CACHE_E4M3 ? launch_plain_attention<float, CACHE_E4M3>(*a, st)
                                   : launch_plain_attention<float, CACHE_PLAIN>(*a, st);
}
int slb_cache_attention_plain_bf16(const CacheAttnArgs* a, cudaStream_t st) {
    const int rc = check_attn(*a);
    if (rc != 0) return rc;
    return a->kind == CACHE_INT8 ? launch_plain_attention<bf16, CACHE_INT8>(*a, st)
           : a->kind == CACHE_E4M3 ? launch_plain_attention<bf16, CACHE_E4M3>(*a, st)
                                   : launch_plain_attention<bf16, CACHE_PLAIN>(*a, st);
}
int slb_cache_attention_join_f32(const CacheAttnArgs* a, cudaStream_t st) {
    const long long blocks = ((long long)a->T * a->H + 7) / 8;
    if (blocks <= 0 || a->parts <= 1 || a->parts > 64) return SLB_ERR_BAD_ARG;
    if (blocks > 0x7fffffffll) return SLB_ERR_TOO_LARGE;
    return slb_launch(cache_attention_join_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, st, *a);
}
int slb_cache_attention_join_bf16(const CacheAttnArgs* a, cudaStream_t st) {
    const long long blocks = ((long long)a->T * a->H + 7) / 8;
    if (blocks <= 0 || a->parts <= 1 || a->parts > 64) return SLB_ERR_BAD_ARG;
    if (blocks > 0x7fffffffll) return SLB_ERR_TOO_LARGE;
    return slb_launch(cache_attention_join_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, st, *a);
}
}
