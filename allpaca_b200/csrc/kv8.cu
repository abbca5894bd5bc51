// Writing the 8-bit cache of keys and values (kv8.cuh: its layout and numbers), and reading it back.
//
//   store   rows of the stacked Q, K, V projection: Q and K rotated, Q out in the activation type, K and V rounded to 8 bits
//           into the pages, one scale to a row of a head
//   read    cached rows back as values
//
// Reference counterparts: rope_qk_kernel (cuda/src/kernels.cu:1244) and the page-slot copies of
// crates/allpaca-core/src/kv_tier.rs:1101-1203 and :1317-1417; the reference's CUDA path keeps 32-bit pages only.
#include "kv8.cuh"

#define KV8_THREADS 256

// sums of S slices of eight neighbouring numbers, in the slices' order
template <typename TI> __device__ __forceinline__ void kv8_load8(float (&x)[8], const TI* p, int S, size_t stride);
template <> __device__ __forceinline__ void kv8_load8<float>(float (&x)[8], const float* p, int S, size_t stride) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    for (int s = 1; s < S; ++s) {
        p += stride;
        const float4 c = *reinterpret_cast<const float4*>(p), d = *reinterpret_cast<const float4*>(p + 4);
        x[0] += c.x; x[1] += c.y; x[2] += c.z; x[3] += c.w; x[4] += d.x; x[5] += d.y; x[6] += d.z; x[7] += d.w;
    }
}
template <> __device__ __forceinline__ void kv8_load8<bf16>(float (&x)[8], const bf16* p, int, size_t) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void kv8_store8(float* p, const float* x) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void kv8_store8(bf16* p, const float* x) {
    uint4 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}

// LPH lanes side by side take a head of a row (hd / 16 of them work): a lane holds numbers i .. i + 7 and i + hd/2 .. i + hd/2 + 7,
// i = 8 * lane, which are eight whole pairs of the rotation; the maximum goes round the lanes in registers, so the row is read
// and written once.  The products of the rotation are rounded one by one (no fused multiply-add), so that the same inputs give the
// same bytes as the formula computed step by step.
template <typename TI, typename TO, int LPH>
__global__ void __launch_bounds__(KV8_THREADS)
rope_kv8_store_kernel(const TI* __restrict__ in, int S, size_t in_stride, TO* __restrict__ q_out, uint8_t* __restrict__ cache,
                      const int* __restrict__ positions, const int* __restrict__ token_seq, const int* __restrict__ block_table,
                      int max_blocks, int nseq, const float2* __restrict__ cos_sin, int pairing, int nh, int nkv, int hd, int P,
                      size_t page_bytes, int num_pages, int chunks, int heads) {
    const int t = blockIdx.x / chunks;
    const int head = (blockIdx.x - t * chunks) * (KV8_THREADS / LPH) + threadIdx.x / LPH;
    const int lane = threadIdx.x & (LPH - 1), half = hd >> 1, i = lane * 8;
    ap_pdl_trigger();
    ap_pdl_wait();
    const bool works = head < heads && i < half;
    float a[8], b[8];
    if (works) {
        const TI* src = in + ((size_t)t * (nh + 2 * nkv) + head) * hd;
        const bool pairs_side_by_side = pairing != 0 && head < nh + nkv;
        const int ia = pairs_side_by_side ? 2 * i : i, ib = pairs_side_by_side ? 2 * i + 8 : i + half;
        kv8_load8<TI>(a, src + ia, S, in_stride);
        kv8_load8<TI>(b, src + ib, S, in_stride);
        if (pairs_side_by_side) {
            float x[8], y[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[k] = a[2 * k];     y[k] = a[2 * k + 1];
                x[k + 4] = b[2 * k]; y[k + 4] = b[2 * k + 1];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) a[k] = x[k], b[k] = y[k];
        }
        if (cos_sin && head < nh + nkv) {
            const float4* cs = reinterpret_cast<const float4*>(cos_sin + (size_t)t * half + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 c = cs[k];                       // (cos, sin) of pairs 2k and 2k + 1
                const float a0 = a[2 * k], b0 = b[2 * k], a1 = a[2 * k + 1], b1 = b[2 * k + 1];
                a[2 * k] = __fsub_rn(__fmul_rn(a0, c.x), __fmul_rn(b0, c.y));
                b[2 * k] = __fadd_rn(__fmul_rn(a0, c.y), __fmul_rn(b0, c.x));
                a[2 * k + 1] = __fsub_rn(__fmul_rn(a1, c.z), __fmul_rn(b1, c.w));
                b[2 * k + 1] = __fadd_rn(__fmul_rn(a1, c.w), __fmul_rn(b1, c.z));
            }
        }
        if (pairing == 1 && head < nh + nkv) {                // the results are neighbours as well: a: 2i .. 2i + 7, b: 2i + 8 ..
            float x[8], y[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[2 * k] = a[k];     x[2 * k + 1] = b[k];
                y[2 * k] = a[k + 4]; y[2 * k + 1] = b[k + 4];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) a[k] = x[k], b[k] = y[k];
        }
        const int oa = pairing == 1 && head < nh + nkv ? 2 * i : i;
        const int ob = pairing == 1 && head < nh + nkv ? 2 * i + 8 : i + half;
        if (head < nh) {
            TO* dst = q_out + ((size_t)t * nh + head) * hd;
            kv8_store8(dst + oa, a);
            kv8_store8(dst + ob, b);
        }
    }
    // (warp-wide from here on, as the lanes of a head exchange their maxima)
    uint32_t amax = 0;
    if (works && head >= nh) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t ua = __float_as_uint(a[k]) & 0x7fffffffu, ub = __float_as_uint(b[k]) & 0x7fffffffu;
            amax = max(amax, ua < 0x7f800000u ? ua : 0u);
            amax = max(amax, ub < 0x7f800000u ? ub : 0u);
        }
    }
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!works || head < nh) return;
    const int pos = positions[t], seq = token_seq[t];
    if (pos < 0 || pos / P >= max_blocks || seq < 0 || seq >= nseq) return;
    const int page = block_table[(size_t)seq * max_blocks + pos / P];
    if (page < 0 || page >= num_pages) return;                // a row without a page is not kept
    const int byte = kv8_scale_byte(amax);
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);     // 2^-e
#pragma unroll
    for (int k = 0; k < 8; ++k) {                             // x - x: 0, or NaN where x is not finite
        a[k] = fmaf(a[k], inv, a[k] - a[k]);
        b[k] = fmaf(b[k], inv, b[k] - b[k]);
    }
    const int which = head >= nh + nkv ? 1 : 0, kvh = head - nh - which * nkv;
    const int oa = pairing == 1 && !which ? 2 * i : i, ob = pairing == 1 && !which ? 2 * i + 8 : i + half;
    const size_t row = (size_t)(which * nkv + kvh) * P + pos % P;
    uint8_t* base = cache + (size_t)page * page_bytes;
    *reinterpret_cast<uint2*>(base + row * hd + oa) = make_uint2(kv8_pack4(a[0], a[1], a[2], a[3]), kv8_pack4(a[4], a[5], a[6], a[7]));
    *reinterpret_cast<uint2*>(base + row * hd + ob) = make_uint2(kv8_pack4(b[0], b[1], b[2], b[3]), kv8_pack4(b[4], b[5], b[6], b[7]));
    if (lane == 0) base[(size_t)2 * nkv * P * hd + row] = (uint8_t)byte;
}

static int kv8_check(const char* what, const void* cache, long long num_pages, long long page_bytes, int nkv, int hd, int P,
                     int max_blocks, int nseq) {
    AP_REQUIRE(nkv > 0 && hd > 0 && hd % 16 == 0 && hd <= 256 && P > 0, "%s: bad sizes kv_heads=%d head_dim=%d page=%d", what, nkv, hd, P);
    AP_REQUIRE(max_blocks > 0 && nseq > 0, "%s: the block table is empty", what);
    AP_REQUIRE(num_pages >= 0 && num_pages < (1LL << 31), "%s: %lld pages", what, num_pages);
    AP_REQUIRE(page_bytes == kv8_page_bytes(nkv, P, hd), "%s: a page of %d KV heads x %d rows x %d has %lld bytes, not %lld", what, nkv,
               P, hd, kv8_page_bytes(nkv, P, hd), page_bytes);
    AP_REQUIRE(((uintptr_t)cache & 15) == 0, "%s: the cache must be 16-byte aligned", what);
    return AP_OK;
}

AP_EXPORT int ap_rope_kv8_store(const void* in, int in_dtype, int S, long long in_stride, void* q_out, int act_dtype, void* cache,
                                long long num_pages, long long page_bytes, const int* positions, const int* token_seq,
                                const int* block_table, int max_blocks, int nseq, const float* cos_sin, int pairing, int T, int nh,
                                int nkv, int hd, int P, cudaStream_t stream) {
    AP_REQUIRE(T >= 0 && nh > 0 && S >= 1, "rope_kv8_store: bad sizes T=%d heads=%d S=%d", T, nh, S);
    AP_REQUIRE(pairing >= 0 && pairing <= 2, "rope_kv8_store: unknown pairing %d", pairing);
    int rc = kv8_check("rope_kv8_store", cache, num_pages, page_bytes, nkv, hd, P, max_blocks, nseq);
    if (rc != AP_OK) return rc;
    AP_REQUIRE(((uintptr_t)in & 15) == 0 && ((uintptr_t)q_out & 15) == 0 && ((uintptr_t)cos_sin & 15) == 0,
               "rope_kv8_store: operands must be 16-byte aligned");
    AP_REQUIRE(in_dtype == AP_F32 || S == 1, "rope_kv8_store: partial sums must be 32-bit");
    if (T == 0) return AP_OK;
    const int heads = nh + 2 * nkv, lanes = hd / 16;
    const int lph = lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
    const int per = KV8_THREADS / lph, chunks = (heads + per - 1) / per;
    AP_REQUIRE((long long)T * chunks < (1LL << 31), "rope_kv8_store: %d rows exceed the grid", T);
    const dim3 grid((unsigned)((long long)T * chunks));
#define KV8_STORE(TI, TO, L)                                                                                                     \
    AP_CHECK_PDL_LAUNCH("rope_kv8_store", ap_launch_pdl(rope_kv8_store_kernel<TI, TO, L>, grid, dim3(KV8_THREADS), 0, stream,     \
                        (const TI*)in, S, (size_t)in_stride, (TO*)q_out, (uint8_t*)cache, positions, token_seq, block_table, max_blocks, \
                        nseq, (const float2*)cos_sin, pairing, nh, nkv, hd, P, (size_t)page_bytes, (int)num_pages, chunks, heads))
#define KV8_STORE_BY_LANES(TI, TO)                  \
    do {                                            \
        if (lph == 1) KV8_STORE(TI, TO, 1);         \
        else if (lph == 2) KV8_STORE(TI, TO, 2);    \
        else if (lph == 4) KV8_STORE(TI, TO, 4);    \
        else if (lph == 8) KV8_STORE(TI, TO, 8);    \
        else KV8_STORE(TI, TO, 16);                 \
    } while (0)
    if (in_dtype == AP_F32 && act_dtype == AP_F32) KV8_STORE_BY_LANES(float, float);
    else if (in_dtype == AP_F32 && act_dtype == AP_BF16) KV8_STORE_BY_LANES(float, bf16);
    else if (in_dtype == AP_BF16 && act_dtype == AP_BF16) KV8_STORE_BY_LANES(bf16, bf16);
    else AP_REQUIRE(false, "rope_kv8_store: unsupported dtypes in=%d act=%d", in_dtype, act_dtype);
#undef KV8_STORE_BY_LANES
#undef KV8_STORE
    return AP_OK;
}

// Reading back: a thread takes 16 numbers of a row of a head (one 16-byte load, one scale); neighbouring threads write
// neighbouring runs of the output.
template <typename TO>
__global__ void __launch_bounds__(KV8_THREADS)
kv8_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ positions, const int* __restrict__ token_seq,
                const int* __restrict__ block_table, int max_blocks, int nseq, TO* __restrict__ k_out, TO* __restrict__ v_out, int T,
                int nkv, int hd, int P, size_t page_bytes, int num_pages) {
    const int runs = hd / 16, per_row = 2 * nkv * runs;
    ap_pdl_trigger();
    ap_pdl_wait();
    const long long id = (long long)blockIdx.x * KV8_THREADS + threadIdx.x;
    const long long t = id / per_row;
    if (t >= T) return;
    const int item = (int)(id - t * per_row);
    const int plane = item / runs, run = item - plane * runs;          // plane: which * nkv + head
    TO* out = plane < nkv ? k_out : v_out;
    if (!out) return;
    const int pos = positions[t], seq = token_seq[t];
    int page = -1;
    if (pos >= 0 && pos / P < max_blocks && seq >= 0 && seq < nseq) page = block_table[(size_t)seq * max_blocks + pos / P];
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;                           // a row without a page reads as zeros
    if (page >= 0 && page < num_pages) {
        const uint8_t* base = cache + (size_t)page * page_bytes;
        const size_t row = (size_t)plane * P + pos % P;
        const uint4 u = *reinterpret_cast<const uint4*>(base + row * hd + run * 16);
        const float s = kv8_scale(base[(size_t)2 * nkv * P * hd + row]);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = kv8_unpack(w[i]);
            x[4 * i] = f.x * s; x[4 * i + 1] = f.y * s; x[4 * i + 2] = f.z * s; x[4 * i + 3] = f.w * s;
        }
    }
    TO* dst = out + (size_t)t * nkv * hd + (size_t)(plane < nkv ? plane : plane - nkv) * hd + run * 16;
    kv8_store8(dst, x);
    kv8_store8(dst + 8, x + 8);
}

// k_out, v_out: [T][nkv][hd] of `dtype`; either may be null.
AP_EXPORT int ap_kv8_read(const void* cache, long long num_pages, long long page_bytes, const int* positions, const int* token_seq,
                          const int* block_table, int max_blocks, int nseq, void* k_out, void* v_out, int dtype, int T, int nkv,
                          int hd, int P, cudaStream_t stream) {
    AP_REQUIRE(T >= 0, "kv8_read: bad number of rows %d", T);
    int rc = kv8_check("kv8_read", cache, num_pages, page_bytes, nkv, hd, P, max_blocks, nseq);
    if (rc != AP_OK) return rc;
    AP_REQUIRE(((uintptr_t)k_out & 15) == 0 && ((uintptr_t)v_out & 15) == 0, "kv8_read: outputs must be 16-byte aligned");
    if (T == 0 || (!k_out && !v_out)) return AP_OK;
    const long long threads = (long long)T * 2 * nkv * (hd / 16), ctas = (threads + KV8_THREADS - 1) / KV8_THREADS;
    AP_REQUIRE(ctas < (1LL << 31), "kv8_read: %d rows exceed the grid", T);
#define KV8_READ(TO)                                                                                                       \
    AP_CHECK_PDL_LAUNCH("kv8_read", ap_launch_pdl(kv8_read_kernel<TO>, dim3((unsigned)ctas), dim3(KV8_THREADS), 0, stream,  \
                        (const uint8_t*)cache, positions, token_seq, block_table, max_blocks, nseq, (TO*)k_out, (TO*)v_out, T, nkv, hd, P, \
                        (size_t)page_bytes, (int)num_pages))
    if (dtype == AP_F32) KV8_READ(float);
    else if (dtype == AP_BF16) KV8_READ(bf16);
    else AP_REQUIRE(false, "kv8_read: unknown dtype %d", dtype);
#undef KV8_READ
    return AP_OK;
}
