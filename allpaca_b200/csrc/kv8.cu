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

// sums of S slices of four neighbouring numbers, in the slices' order
template <typename TI> __device__ __forceinline__ float4 kv8_load4(const TI* p, int S, size_t stride);
template <> __device__ __forceinline__ float4 kv8_load4<float>(const float* p, int S, size_t stride) {
    float4 x = *reinterpret_cast<const float4*>(p);
    for (int s = 1; s < S; ++s) {
        p += stride;
        const float4 c = *reinterpret_cast<const float4*>(p);
        x.x += c.x; x.y += c.y; x.z += c.z; x.w += c.w;
    }
    return x;
}
template <> __device__ __forceinline__ float4 kv8_load4<bf16>(const bf16* p, int, size_t) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void kv8_store4(float* p, const float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void kv8_store4(bf16* p, const float4 x) {
    uint2 u;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
    h[0] = __floats2bfloat162_rn(x.x, x.y);
    h[1] = __floats2bfloat162_rn(x.z, x.w);
    *reinterpret_cast<uint2*>(p) = u;
}
// the largest magnitude among the finite ones
__device__ __forceinline__ uint32_t kv8_largest(uint32_t m, const float4 x) {
    const uint32_t u[4] = {__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu, __float_as_uint(x.z) & 0x7fffffffu,
                           __float_as_uint(x.w) & 0x7fffffffu};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, u[i] < 0x7f800000u ? u[i] : 0u);
    return m;
}
// x * f as four numbers of 8 bits (x - x: 0, or NaN where x is not finite)
__device__ __forceinline__ uint32_t kv8_round4(const float4 x, float f) {
    return kv8_pack4(fmaf(x.x, f, x.x - x.x), fmaf(x.y, f, x.y - x.y), fmaf(x.z, f, x.z - x.z), fmaf(x.w, f, x.w - x.w));
}

// A CTA takes 256 lanes' worth of a row's heads, 2^side_bits lanes side by side a head, hd / 8 of which work: a lane holds numbers
// i .. i + 3 and i + hd/2 .. i + hd/2 + 3, i four times its place, which are four whole pairs of the rotation; the maximum goes round
// the lanes in registers, so the row is read and written once.  The products of the rotation are rounded one by one (no fused
// multiply-add), so that the same inputs give the same bytes as the formula computed step by step.
//
// Few rows are bound by their launch and three loads that wait for one another (position, page, store): 1 row of a small model 2.5 us,
// 64 rows 2.0 in a stream of such launches.  Many rows are bound by instructions (2.9 of 4 issued a cycle with a division for the
// row and the pairing decided in the kernel; without them 2048 rows of 32 + 16 heads of 128, 47 MB, floor 7.3 us, take 12.7 us instead of
// 14.3, 8192 rows 45.8 instead of 50.2).  Eight numbers to a half and lane, rows of a prompt in turns of CTAs of 128
// threads, were 13.3 and 42.6, but 64 rows 3.1; several heads to a thread with all loads ahead were slower everywhere (two 19.4 for 2048
// rows, four 29.9), and so was looking the page up ahead of the rotation (16.1).
template <typename TI, typename TO, int PAIRING>
__global__ void __launch_bounds__(KV8_THREADS, 6)
rope_kv8_store_kernel(const TI* __restrict__ in, int S, size_t in_stride, TO* __restrict__ q_out, uint8_t* __restrict__ cache,
                      const int* __restrict__ positions, const int* __restrict__ token_seq, const int* __restrict__ block_table,
                      int max_blocks, int nseq, const float2* __restrict__ cos_sin, int nh, int nkv, int hd, int P, int side_bits,
                      size_t page_bytes, int num_pages) {
    const int heads = nh + 2 * nkv, t = blockIdx.x, half = hd >> 1;
    const int head = (blockIdx.y * KV8_THREADS + threadIdx.x) >> side_bits, i = (threadIdx.x & ((1 << side_bits) - 1)) * 4;
    ap_pdl_trigger();
    ap_pdl_wait();
    const bool works = head < heads && i < half, turns = head < nh + nkv;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    int at_a = i, at_b = i + half;                            // where the results go
    if (works) {
        const TI* src = in + (size_t)t * heads * hd + head * hd;
        const bool pairs = PAIRING != 0 && turns;
        a = kv8_load4<TI>(src + (pairs ? 2 * i : i), S, in_stride);
        b = kv8_load4<TI>(src + (pairs ? 2 * i + 4 : i + half), S, in_stride);
        if (pairs) {
            const float4 x = a;
            a = make_float4(x.x, x.z, b.x, b.z);
            b = make_float4(x.y, x.w, b.y, b.w);
        }
        if (cos_sin && turns) {
            const float4* cs = reinterpret_cast<const float4*>(cos_sin + (size_t)t * half + i);
            const float4 c = cs[0], d = cs[1], x = a;         // (cos, sin) of two pairs each
            a = make_float4(__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(b.x, c.y)), __fsub_rn(__fmul_rn(x.y, c.z), __fmul_rn(b.y, c.w)),
                            __fsub_rn(__fmul_rn(x.z, d.x), __fmul_rn(b.z, d.y)), __fsub_rn(__fmul_rn(x.w, d.z), __fmul_rn(b.w, d.w)));
            b = make_float4(__fadd_rn(__fmul_rn(x.x, c.y), __fmul_rn(b.x, c.x)), __fadd_rn(__fmul_rn(x.y, c.w), __fmul_rn(b.y, c.z)),
                            __fadd_rn(__fmul_rn(x.z, d.y), __fmul_rn(b.z, d.x)), __fadd_rn(__fmul_rn(x.w, d.w), __fmul_rn(b.w, d.z)));
        }
        if (PAIRING == 1 && turns) {                          // the results are neighbours as well
            const float4 x = a;
            a = make_float4(x.x, b.x, x.y, b.y);
            b = make_float4(x.z, b.z, x.w, b.w);
            at_a = 2 * i;
            at_b = 2 * i + 4;
        }
        if (head < nh) {
            TO* dst = q_out + (size_t)t * nh * hd + head * hd;
            kv8_store4(dst + at_a, a);
            kv8_store4(dst + at_b, b);
        }
    }
    // (warp-wide from here on, as the lanes of a head exchange their maxima)
    const bool kept = works && head >= nh;
    if (!__any_sync(0xffffffffu, kept)) return;
    uint32_t amax = kv8_largest(kv8_largest(0u, a), b);
    for (int o = (1 << side_bits) >> 1; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (!kept) return;
    const int pos = positions[t], seq = token_seq[t];
    if (pos < 0 || seq < 0 || seq >= nseq) return;
    const int block = pos / P;
    if (block >= max_blocks) return;
    const int page = block_table[(size_t)seq * max_blocks + block];
    if (page < 0 || page >= num_pages) return;                // a row without a page is not kept
    const int byte = kv8_scale_byte(amax);
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);     // 2^-e
    const size_t row = (size_t)(head - nh) * P + (pos - block * P);
    uint8_t* base = cache + (size_t)page * page_bytes;
    *reinterpret_cast<uint32_t*>(base + row * hd + at_a) = kv8_round4(a, inv);
    *reinterpret_cast<uint32_t*>(base + row * hd + at_b) = kv8_round4(b, inv);
    if (i == 0) base[(size_t)2 * nkv * P * hd + row] = (uint8_t)byte;
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
    const int heads = nh + 2 * nkv, lanes = hd / 8;
    const int bits = lanes <= 2 ? 1 : lanes <= 4 ? 2 : lanes <= 8 ? 3 : lanes <= 16 ? 4 : 5;
    AP_REQUIRE(heads <= (65535 * KV8_THREADS >> bits), "rope_kv8_store: %d heads exceed the grid", heads);
    const dim3 grid((unsigned)T, (unsigned)(((heads << bits) + KV8_THREADS - 1) / KV8_THREADS));
#define KV8_STORE(TI, TO, PAIRING)                                                                                                 \
    AP_CHECK_PDL_LAUNCH("rope_kv8_store", ap_launch_pdl(rope_kv8_store_kernel<TI, TO, PAIRING>, grid, dim3(KV8_THREADS), 0, stream,  \
                        (const TI*)in, S, (size_t)in_stride, (TO*)q_out, (uint8_t*)cache, positions, token_seq, block_table, max_blocks, \
                        nseq, (const float2*)cos_sin, nh, nkv, hd, P, bits, (size_t)page_bytes, (int)num_pages))
#define KV8_STORE_BY_PAIRING(TI, TO)                \
    do {                                            \
        if (pairing == 0) KV8_STORE(TI, TO, 0);     \
        else if (pairing == 1) KV8_STORE(TI, TO, 1); \
        else KV8_STORE(TI, TO, 2);                  \
    } while (0)
    if (in_dtype == AP_F32 && act_dtype == AP_F32) KV8_STORE_BY_PAIRING(float, float);
    else if (in_dtype == AP_F32 && act_dtype == AP_BF16) KV8_STORE_BY_PAIRING(float, bf16);
    else if (in_dtype == AP_BF16 && act_dtype == AP_BF16) KV8_STORE_BY_PAIRING(bf16, bf16);
    else AP_REQUIRE(false, "rope_kv8_store: unsupported dtypes in=%d act=%d", in_dtype, act_dtype);
#undef KV8_STORE_BY_PAIRING
#undef KV8_STORE
    return AP_OK;
}

// Reading back: a CTA takes `tile` rows of one head's keys or values.  Its first threads look up where the rows lie and their scales; then
// runs = hd / 8 threads side by side take a row, eight numbers (one 8-byte load, two stores) to each, eight rows to a thread
// with all eight loads under way.
//
// Bound by memory: 42,300 rows of 16 sequences, 8 KV heads of 128, to bfloat16 (260 MB, floor 40.4 us at the copy rate) take 44.2 us,
// 5.9 TB/s, pages scattered.  What counts is loads in flight: 51.3 us with four rows to a thread, 67.4 with two, 46.6 with
// sixteen; 62.4 with sixteen numbers of one row to a thread and its place looked up by every thread.  CTAs of 256 threads: 45.3.
#define KV8_READ_THREADS 128
#define KV8_READ_ROWS 8
template <typename TO>
__global__ void __launch_bounds__(KV8_READ_THREADS)
kv8_read_kernel(const uint8_t* __restrict__ cache, const int* __restrict__ positions, const int* __restrict__ token_seq,
                const int* __restrict__ block_table, int max_blocks, int nseq, TO* __restrict__ k_out, TO* __restrict__ v_out, int T,
                int nkv, int hd, int P, size_t page_bytes, int num_pages) {
    __shared__ long long at_s[KV8_READ_ROWS * KV8_READ_THREADS / 2];        // where a row's numbers lie (-1: nowhere)
    __shared__ float scale_s[KV8_READ_ROWS * KV8_READ_THREADS / 2];
    const int runs = hd / 8, side = KV8_READ_THREADS / runs, tile = side * KV8_READ_ROWS;
    const int planes = k_out && v_out ? 2 * nkv : nkv;                 // which * nkv + head
    const int plane = (int)(blockIdx.x % planes) + (k_out ? 0 : nkv);
    const long long t0 = (long long)(blockIdx.x / planes) * tile;
    ap_pdl_trigger();
    ap_pdl_wait();
    for (int i = threadIdx.x; i < tile; i += KV8_READ_THREADS) {
        long long at = -1;
        float s = 0.f;
        if (t0 + i < T) {
            const int pos = positions[t0 + i], seq = token_seq[t0 + i];
            int page = -1;
            if (pos >= 0 && pos / P < max_blocks && seq >= 0 && seq < nseq) page = block_table[(size_t)seq * max_blocks + pos / P];
            if (page >= 0 && page < num_pages) {
                const size_t row = (size_t)plane * P + pos % P;
                at = (long long)((size_t)page * page_bytes + row * hd);
                s = kv8_scale(cache[(size_t)page * page_bytes + (size_t)2 * nkv * P * hd + row]);
            }
        }
        at_s[i] = at;
        scale_s[i] = s;
    }
    __syncthreads();
    const int first = threadIdx.x / runs, col = (threadIdx.x - first * runs) * 8;
    if (first >= side) return;                                         // (where the runs do not divide the threads)
    uint2 u[KV8_READ_ROWS];
#pragma unroll
    for (int i = 0; i < KV8_READ_ROWS; ++i) {
        const long long at = at_s[first + i * side];                   // a row without a page reads as zeros
        u[i] = at >= 0 ? *reinterpret_cast<const uint2*>(cache + at + col) : make_uint2(0u, 0u);
    }
    TO* out = (plane < nkv ? k_out : v_out) + (size_t)(plane < nkv ? plane : plane - nkv) * hd + col;
#pragma unroll
    for (int i = 0; i < KV8_READ_ROWS; ++i) {
        const long long t = t0 + first + i * side;
        if (t >= T) break;
        const float s = scale_s[first + i * side];
        const float4 a = kv8_unpack(u[i].x), b = kv8_unpack(u[i].y);
        TO* to = out + (size_t)t * nkv * hd;
        kv8_store4(to, make_float4(a.x * s, a.y * s, a.z * s, a.w * s));
        kv8_store4(to + 4, make_float4(b.x * s, b.y * s, b.z * s, b.w * s));
    }
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
    const int tile = KV8_READ_THREADS / (hd / 8) * KV8_READ_ROWS;
    const long long ctas = ((long long)T + tile - 1) / tile * (k_out && v_out ? 2 * nkv : nkv);
    AP_REQUIRE(ctas < (1LL << 31), "kv8_read: %d rows exceed the grid", T);
#define KV8_READ(TO)                                                                                                       \
    AP_CHECK_PDL_LAUNCH("kv8_read", ap_launch_pdl(kv8_read_kernel<TO>, dim3((unsigned)ctas), dim3(KV8_READ_THREADS), 0, stream,  \
                        (const uint8_t*)cache, positions, token_seq, block_table, max_blocks, nseq, (TO*)k_out, (TO*)v_out, T, nkv, hd, P, \
                        (size_t)page_bytes, (int)num_pages))
    if (dtype == AP_F32) KV8_READ(float);
    else if (dtype == AP_BF16) KV8_READ(bf16);
    else AP_REQUIRE(false, "kv8_read: unknown dtype %d", dtype);
#undef KV8_READ
    return AP_OK;
}
