// Causal grouped-query attention over the 8-bit paged cache (kv8.cuh), for one head size fixed at compile time
// (-DAP_HEAD_DIM=...): the kernel that takes any batch, in either activation type, all in 32 bits.
//
//   q, out : [T, nh, HD];  row r attends to keys at positions <= positions[r] of sequence token_seq[r] (and > positions[r] - window
//   when window > 0).  Keys whose page was given back (id < 0) do not count; a row that sees no key gets zeros.
//
// With key j kept as codes c_j and scale 2^a_j, value j as d_j and 2^b_j:
//   s_j = scale * 2^a_j * (q . c_j),   out = sum_j exp(s_j - m) 2^b_j d_j / sum_j exp(s_j - m).
//
// A CTA takes a row of one query head and walks its keys K8_CHUNK at a time, a key to a thread for the scores, a column of four to
// a thread for the values, with the running maximum and sum of a softmax.  It is here for float32 activations, whose products no
// tensor core takes in full, and for what the kernels of bfloat16 rows and portions refuse (pages of other sizes, caches of 64 GB and more):
// it reads a KV head's keys once for every query head and row, so arithmetic and L2 bound it, not the 8-bit keys' bytes (4 float32 rows of
// 32 heads of 64 with 20 to 700 keys: 10.0 us, floor 0.5; 64 rows of 2000 keys, heads of 128: 250, floor 42).  The chunks of a row wait for
// one another, hence many keys to a chunk: with 128 threads the two take 15.9 and 309 us, with 512 9.5 and 319; a prompt of 499
// rows takes 131 us, 117 with 128 threads, 182 with 512.
//
// Reference counterparts: attention_qtile_kernel and attention_split_gqa_kernel (cuda/src/kernels.cu:1801, :1874), the causal
// rule :1583-1585; the reference's keys and values are 32-bit.
#include "kv8.cuh"
#include <float.h>
#include <math.h>

#ifndef AP_HEAD_DIM
#error "compile with -DAP_HEAD_DIM=<head size>"
#endif

#define HD AP_HEAD_DIM
#define K8_THREADS 256
#define K8_CHUNK K8_THREADS                               // keys at a time: one to a thread
#define K8_LANES (HD / 4 < K8_THREADS ? HD / 4 : K8_THREADS)     // threads side by side on a value row, four numbers each
#define K8_GROUPS (K8_THREADS / K8_LANES)

template <typename T>
__global__ void __launch_bounds__(K8_THREADS)
attention_kv8_rows_kernel(const T* __restrict__ q, T* __restrict__ out, const uint8_t* __restrict__ cache, size_t page_bytes,
                          int num_pages, const int* __restrict__ block_table, int max_blocks, int nseq,
                          const int* __restrict__ token_seq, const int* __restrict__ positions, int nh, int nkv, int P, float scale,
                          int window) {
    __shared__ float q_s[HD];
    __shared__ float p_s[K8_CHUNK];
    __shared__ long long at_s[K8_CHUNK];                   // where a key of the chunk lies (-1: nowhere)
    __shared__ float red[32];
    __shared__ float part_s[K8_GROUPS * HD];
    const int t = blockIdx.x, h = blockIdx.y, kvh = h / (nh / nkv);
    ap_pdl_trigger();
    ap_pdl_wait();
    const int seq = token_seq[t];
    const int qpos = seq >= 0 && seq < nseq ? min(positions[t], max_blocks * P - 1) : -1;
    const int* table = block_table + (size_t)max(seq, 0) * max_blocks;
    const T* qr = q + ((size_t)t * nh + h) * HD;
    for (int d = threadIdx.x; d < HD; d += K8_THREADS) q_s[d] = ap_to_float(qr[d]);
    __syncthreads();
    const size_t rows = (size_t)2 * nkv * P;               // of a page
    const int lane = threadIdx.x % K8_LANES, group = threadIdx.x / K8_LANES;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = -INFINITY, l = 0.f;
    const int kfirst = (window > 0 && qpos - window + 1 > 0) ? qpos - window + 1 : 0;
    for (int c0 = kfirst; c0 <= qpos; c0 += K8_CHUNK) {
        const int kpos = c0 + threadIdx.x;
        float s = -INFINITY, vscale = 0.f;
        long long at = -1;
        if (kpos <= qpos) {
            const int page = table[kpos / P];
            if (page >= 0 && page < num_pages) {
                const uint8_t* base = cache + (size_t)page * page_bytes;
                const size_t row = (size_t)kvh * P + kpos % P;
                const uint4* k = reinterpret_cast<const uint4*>(base + row * HD);
                float dot = 0.f;
#pragma unroll 4
                for (int i = 0; i < HD / 16; ++i) {
                    const uint4 u = k[i];
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float4 f = kv8_unpack(w[e]);
                        const float* qq = q_s + i * 16 + e * 4;
                        dot = fmaf(qq[0], f.x, dot); dot = fmaf(qq[1], f.y, dot);
                        dot = fmaf(qq[2], f.z, dot); dot = fmaf(qq[3], f.w, dot);
                    }
                }
                const uint8_t* scales = base + rows * HD;
                s = dot * (scale * kv8_scale(scales[row]));
                vscale = kv8_scale(scales[row + (size_t)nkv * P]);
                at = (long long)((size_t)page * page_bytes + (row + (size_t)nkv * P) * HD);
            }
        }
        at_s[threadIdx.x] = at;
        const float cmax = ap_block_max(s, red);
        const float m_new = fmaxf(m, cmax), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float p = expf(s - m_use);                   // 0 where nothing is seen
        const float csum = ap_block_sum(p, red);
        p_s[threadIdx.x] = p * vscale;
        __syncthreads();
        const float alpha = expf(m - m_use);
        l = l * alpha + csum;
        m = m_new;
        acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
        const int nk = min(K8_CHUNK, qpos - c0 + 1);
        if (group < K8_GROUPS) {
#pragma unroll 4
            for (int j = group; j < nk; j += K8_GROUPS) {
                const long long a = at_s[j];
                if (a < 0) continue;
                const float4 v = kv8_unpack(*reinterpret_cast<const uint32_t*>(cache + a + lane * 4));
                const float pj = p_s[j];
                acc.x = fmaf(pj, v.x, acc.x); acc.y = fmaf(pj, v.y, acc.y);
                acc.z = fmaf(pj, v.z, acc.z); acc.w = fmaf(pj, v.w, acc.w);
            }
        }
        __syncthreads();
    }
    if (group < K8_GROUPS) *reinterpret_cast<float4*>(part_s + group * HD + lane * 4) = acc;
    __syncthreads();
    T* o = out + ((size_t)t * nh + h) * HD;
    const float inv = l > 0.f ? 1.0f / l : 0.f;
    for (int d = threadIdx.x; d < HD; d += K8_THREADS) {
        float a = part_s[d];
#pragma unroll
        for (int g = 1; g < K8_GROUPS; ++g) a += part_s[g * HD + d];
        o[d] = ap_from_float<T>(qpos < 0 ? 0.f : l != l ? l : a * inv);
    }
}

AP_EXPORT int ap_attention_kv8_rows(const void* q, void* out, int dtype, const void* cache, long long num_pages, long long page_bytes,
                                    const int* block_table, int max_blocks, int nseq, const int* token_seq, const int* positions,
                                    int T, int nh, int nkv, int hd, int P, float scale, int window, cudaStream_t stream) {
    AP_REQUIRE(hd == HD, "attention_kv8: this library was compiled for head size %d, not %d", HD, hd);
    AP_REQUIRE(T >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0 && P > 0 && max_blocks > 0 && nseq > 0,
               "attention_kv8: bad sizes T=%d heads=%d kv_heads=%d page=%d", T, nh, nkv, P);
    AP_REQUIRE(nh <= 65535, "attention_kv8: %d heads exceed the grid", nh);
    AP_REQUIRE(num_pages >= 0 && num_pages < (1LL << 31) && page_bytes == kv8_page_bytes(nkv, P, HD),
               "attention_kv8: the pages do not match the heads");
    AP_REQUIRE(((uintptr_t)cache & 15) == 0, "attention_kv8: the cache must be 16-byte aligned");
    // (a chunk's last key may lie K8_CHUNK past a row's)
    AP_REQUIRE((long long)max_blocks * P < (1LL << 31) - 2 * K8_CHUNK, "attention_kv8: the block table names some 2^31 keys or more");
    if (T == 0) return AP_OK;
    const dim3 grid(T, nh);
#define K8_ROWS(TT)                                                                                                          \
    AP_CHECK_PDL_LAUNCH("attention_kv8_rows", ap_launch_pdl(attention_kv8_rows_kernel<TT>, grid, dim3(K8_THREADS), 0, stream, \
                        (const TT*)q, (TT*)out, (const uint8_t*)cache, (size_t)page_bytes, (int)num_pages, block_table, max_blocks, nseq, \
                        token_seq, positions, nh, nkv, P, scale, window))
    if (dtype == AP_F32) K8_ROWS(float);
    else if (dtype == AP_BF16) K8_ROWS(bf16);
    else AP_REQUIRE(false, "attention_kv8: unknown dtype %d", dtype);
#undef K8_ROWS
    return AP_OK;
}
