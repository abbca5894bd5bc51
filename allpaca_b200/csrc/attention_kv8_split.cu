// bfloat16 causal grouped-query attention over the 8-bit paged cache (kv8.cuh) for few rows: single rows of many sequences, and
// portions that the tcgen05 kernel does not take.  Head sizes 32, 64, 96 and 128 (-DAP_HEAD_DIM).
//
// Such a step streams the cache, so the kernel is built around the loads.  A warp owns 32 keys at a time and nothing is staged in
// shared memory: lanes load the 8-bit numbers straight into the registers from which mma.sync takes them (m16n8k32, e4m3 x e4m3, the
// order of the summed index being free as long as both operands agree on it), the next keys' numbers while this step's are worked on:
// 8 KB in flight to a warp at head size 128.  A key's numbers are its B operand as loaded.  A value's are not, as the summed index of the second product
// is the key: 4 x 4 byte transposes in registers (two byte permutes to a register) put four keys' numbers of one column side by side.
//
// The numbers are never widened: it is the queries and the weights that are split into two e4m3 numbers each, x = hi + lo / 16, which
// keeps the eight significant bits of bfloat16 (hi is off by half of its last of four bits, and so much needs four bits again).  A tile
// of 16 rows holds eight query rows twice, hi above lo, so the split costs no instruction.  Queries are scaled by a power of two to a
// row (numbers down to 2^-15 of a row's largest keep all eight bits), weights lie between 0 and 256.
//
//   t_j = log2(e) scale 2^a_j (q . c_j),   m = max_j (t_j + b_j),   l = sum_j 2^(t_j - m),   out = sum_j 2^(t_j + b_j - m) d_j / l
//
// with scales 2^a_j of keys and 2^b_j of values: taking the maximum over what meets the 8-bit numbers keeps the largest products exact
// however values differ in size, and with b_j between -60 and 40 neither sum leaves the range of 32-bit numbers.
//
// A CTA takes 8 rows (tokens x heads of one KV head) and a slice of the keys, its warps take turns over batches of 32 keys and are
// merged through shared memory at the end; the slices of one tile form a cluster of up to 16 CTAs and are merged through
// distributed shared memory by its first: one launch, no scratch, sums in a fixed order.
//
// Reference counterparts (cuda/src/kernels.cu): attention_split_gqa_kernel :1874 and attention_merge_kernel :1997, the causal rule
// :1583-1585.
#include "kv8.cuh"
#include "tcgen05.cuh"
#include <math.h>

#ifndef AP_HEAD_DIM
#error "compile with -DAP_HEAD_DIM=<head size>"
#endif

#if (AP_HEAD_DIM % 32 == 0 && AP_HEAD_DIM <= 128)

#define HD AP_HEAD_DIM
#define K8S_ROWS 8                             // query rows of a tile
#define K8S_KEYS 32                            // keys of a batch, one to a lane
#define KVEC (HD % 64 == 0 ? 16 : 8)           // bytes of a key that a lane loads at once
#define KLOADS (HD / (4 * KVEC))
#define KWORDS (HD / 16)                       // words of a key to a lane
#define VWORDS (HD / 32)                       // words of a value to a lane
#define NTILES (HD / 8)
#define XROW (HD + 2)                          // a row's result: HD sums, maximum, sum of weights

struct K8sParams {
    const bf16* q;
    bf16* out;
    const uint8_t* cache;
    const int* block_table;
    const int* seq_start;                      // null: row r is sequence r's only one
    const int* positions;
    size_t page_bytes;
    int num_pages, max_blocks, nseq, nh, nkv, P, window;
    int heads, n_chunks, tokens, nsplit;       // heads and tokens of a tile, tiles of heads to a KV head, key slices
    float scale_log2;
};

template <int BYTES> struct K8Run { uint32_t w[BYTES / 4]; };
template <int BYTES> __device__ __forceinline__ K8Run<BYTES> k8_load(const uint8_t* p) {
    K8Run<BYTES> r;
    if constexpr (BYTES == 16)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "l"(p));
    else if constexpr (BYTES == 8)
        asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
    else
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) asm volatile("ld.global.L1::no_allocate.u32 %0, [%1];" : "=r"(r.w[i]) : "l"(p + 4 * i));
    return r;
}
__device__ __forceinline__ float k8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void k8_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// four numbers as hi + lo / 16
__device__ __forceinline__ void k8_split(float a, float b, float c, float d, uint32_t& hi, uint32_t& lo) {
    hi = kv8_pack4(a, b, c, d);
    const float4 h = kv8_unpack(hi);
    lo = kv8_pack4((a - h.x) * 16.f, (b - h.y) * 16.f, (c - h.z) * 16.f, (d - h.w) * 16.f);
}

template <int NW, bool CLUSTER>
__global__ void __launch_bounds__(NW * 32, NW == 4 ? 3 : 1)
attention_kv8_split_kernel(const K8sParams p) {
    extern __shared__ float sh[];                          // the warps' results, then (cluster) the slices'
    __shared__ uint32_t off_s[NW][2][K8S_KEYS];            // where a key lies in the cache, in units of 16 bytes
    __shared__ uint32_t meta_s[NW][2][K8S_KEYS];           // scale bytes of key and value; bit 16: the key is there
    __shared__ int s_seq, s_tile;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (CLUSTER) tc::cluster_arrive();
    ap_pdl_trigger();
    ap_pdl_wait();
    int seq = blockIdx.x, row0 = blockIdx.x, ntok = 1;
    if (p.seq_start) {
        if (threadIdx.x == 0) {
            // late tiles of a sequence have the most keys to walk: hand them out first
            int t = gridDim.x - 1 - blockIdx.x, found = -1;
            for (int s = 0; s < p.nseq; ++s) {
                const int n = p.seq_start[s + 1] - p.seq_start[s], nt = (n + p.tokens - 1) / p.tokens;
                if (t < nt) { found = s; break; }
                t -= nt;
            }
            s_seq = found;
            s_tile = t;
        }
        __syncthreads();
        seq = s_seq;
        if (seq >= 0) {
            row0 = p.seq_start[seq] + s_tile * p.tokens;
            ntok = min(p.tokens, p.seq_start[seq + 1] - row0);
        } else {
            ntok = 0;
        }
    }
    const int kvh = blockIdx.y / p.n_chunks, chunk = blockIdx.y - kvh * p.n_chunks;
    const int head0 = kvh * (p.nh / p.nkv) + chunk * p.heads;
    const int nheads = min(p.heads, p.nh / p.nkv - chunk * p.heads);
    const int rows = ntok * p.heads;                       // rows of the tile (those of heads past the last are not written)
    const int* table = p.block_table + (size_t)max(seq, 0) * p.max_blocks;

    // this lane's query row g
    const int tok = g / p.heads, hq = g - tok * p.heads;
    const bool rvalid = g < rows && hq < nheads;
    const int last_key = p.max_blocks * p.P - 1;
    int qpos = -1;
    if (ntok > 0) qpos = rvalid ? min(p.positions[row0 + tok], last_key) : -1;
    uint32_t qh[KWORDS], ql[KWORDS];
    float rowfac;
    {
        float x[KWORDS][4];
        uint32_t amax = 0;
        const bf16* qr = p.q + ((size_t)(rvalid ? row0 + tok : 0) * p.nh + head0 + (rvalid ? hq : 0)) * HD;
#pragma unroll
        for (int i = 0; i < KLOADS; ++i)
#pragma unroll
            for (int w = 0; w < KVEC / 4; ++w) {
                uint2 u = make_uint2(0, 0);
                if (rvalid) u = *reinterpret_cast<const uint2*>(qr + i * 4 * KVEC + c * KVEC + w * 4);
                float* y = x[i * (KVEC / 4) + w];
                y[0] = __uint_as_float(u.x << 16); y[1] = __uint_as_float(u.x & 0xffff0000u);
                y[2] = __uint_as_float(u.y << 16); y[3] = __uint_as_float(u.y & 0xffff0000u);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t m = __float_as_uint(y[e]) & 0x7fffffffu;
                    amax = max(amax, m < 0x7f800000u ? m : 0u);
                }
            }
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // 2^-e with e the smallest exponent under which no number exceeds 448 (kept where both 2^e and 2^-e are normal numbers)
        const int e = min(max((int)(amax >> 23) - 135 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0), -120), 120);
        const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
        rowfac = p.scale_log2 * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < KWORDS; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) x[i][k] = fmaf(x[i][k], inv, x[i][k] - x[i][k]);      // NaN where not finite
            k8_split(x[i][0], x[i][1], x[i][2], x[i][3], qh[i], ql[i]);
        }
    }
    // keys any row of the tile sees, and those that all rows of this warp see
    int kmax = -1, kmin = 0;
    if (ntok > 0) {
        kmax = min(p.positions[row0 + ntok - 1], last_key);
        const int first = p.positions[row0];
        kmin = (p.window > 0 && first - p.window + 1 > 0) ? first - p.window + 1 : 0;
    }
    int all_to = rvalid ? qpos : 0x7fffffff, all_from = rvalid && p.window > 0 ? qpos - p.window + 1 : -0x7fffffff;
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
        all_to = min(all_to, __shfl_xor_sync(0xffffffffu, all_to, o));
        all_from = max(all_from, __shfl_xor_sync(0xffffffffu, all_from, o));
    }
    const int b_first = kmin / K8S_KEYS, b_last = kmax >= kmin ? kmax / K8S_KEYS : b_first - 1;
    const int per = (b_last - b_first + 1 + p.nsplit - 1) / p.nsplit;
    const int lo = b_first + blockIdx.z * per, hi = min(b_last + 1, lo + per);

    const size_t rows_of_page = (size_t)2 * p.nkv * p.P;
    const uint32_t v_units = (uint32_t)((size_t)p.nkv * p.P * HD / 16);
    uint32_t* off_w = off_s[warp][0];
    uint32_t* meta_w = meta_s[warp][0];
    // the page of this lane's key of batch b (-1: nowhere), and where the key lies
    auto page_of = [&](int b) {
        const int kpos = b * K8S_KEYS + lane;
        return b < hi && kpos >= kmin && kpos <= kmax ? table[kpos / p.P] : -1;
    };
    auto place = [&](int b, int page, uint32_t& off, uint32_t& ks, uint32_t& vs) {
        const int kpos = b * K8S_KEYS + lane, slot = kpos - kpos / p.P * p.P;
        const bool there = page >= 0 && page < p.num_pages;
        const uint8_t* base = p.cache + (size_t)(there ? page : 0) * p.page_bytes;
        const size_t row = (size_t)kvh * p.P + (there ? slot : 0);
        off = (uint32_t)(((size_t)(base - p.cache) + row * HD) >> 4);
        const uint8_t* sc = base + rows_of_page * HD + row;
        ks = there ? (uint32_t)sc[0] | 0x10000u : 0u;                // (a key that is not there reads row 0 and does not count)
        vs = there ? (uint32_t)sc[(size_t)p.nkv * p.P] << 8 : 0u;
    };
    K8Run<KVEC> kr[4][KLOADS];
    K8Run<VWORDS * 4> vr[4][2];
    auto load_keys = [&](const uint32_t* off) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint8_t* k = p.cache + ((size_t)off[j * 8 + g] << 4) + c * KVEC;
#pragma unroll
            for (int i = 0; i < KLOADS; ++i) kr[j][i] = k8_load<KVEC>(k + i * 4 * KVEC);
        }
    };
    auto load_values = [&](const uint32_t* off) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint2 o = *reinterpret_cast<const uint2*>(off + j * 8 + c * 2);
            vr[j][0] = k8_load<VWORDS * 4>(p.cache + ((size_t)(o.x + v_units) << 4) + g * (VWORDS * 4));
            vr[j][1] = k8_load<VWORDS * 4>(p.cache + ((size_t)(o.y + v_units) << 4) + g * (VWORDS * 4));
        }
    };

    float o[NTILES][4];
#pragma unroll
    for (int j = 0; j < NTILES; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m = -INFINITY, l = 0.f;
    int b = lo + warp;
    int page1 = -1;
    if (b < hi) {
        uint32_t off, ks, vs;
        place(b, page_of(b), off, ks, vs);
        page1 = page_of(b + NW);
        off_w[lane] = off;
        __syncwarp();
        load_keys(off_w);
        load_values(off_w);
        meta_w[lane] = ks | vs;
        __syncwarp();
    }
    for (int at = 0; b < hi; b += NW, at ^= K8S_KEYS) {
        const bool more = b + NW < hi;
        const uint32_t *meta = meta_w + at;
        uint32_t off = 0, ks = 0, vs = 0;
        if (more) {
            place(b + NW, page1, off, ks, vs);
            page1 = page_of(b + 2 * NW);
        }
        float s[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
            for (int w = 0; w < KWORDS; w += 2) {
                const K8Run<KVEC>& r = kr[j][w / (KVEC / 4)];
                k8_mma(s[j], qh[w], ql[w], qh[w + 1], ql[w + 1], r.w[w % (KVEC / 4)], r.w[w % (KVEC / 4) + 1]);
            }
        }
        if (more) {
            off_w[(at ^ K8S_KEYS) + lane] = off;
            __syncwarp();
            load_keys(off_w + (at ^ K8S_KEYS));
        }
        // scores of keys 8 j + 2 c and the one after it, for query row g, in units of log2
        float t[4][2];
        uint32_t md[4][2];
        const int k0 = b * K8S_KEYS;
        bool every = k0 >= all_from && k0 + K8S_KEYS - 1 <= all_to;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint2 u = *reinterpret_cast<const uint2*>(meta + j * 8 + c * 2);
            md[j][0] = u.x; md[j][1] = u.y;
            every = every && (u.x & u.y & 0x10000u);
        }
        every = __all_sync(0xffffffffu, every);
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                t[j][i] = fmaf(s[j][2 + i], 0.0625f, s[j][i]) * (rowfac * kv8_scale(md[j][i] & 0xffu));
                if (!every) {
                    const int kpos = k0 + j * 8 + c * 2 + i;
                    const bool seen = (md[j][i] & 0x10000u) && kpos <= qpos && (p.window <= 0 || qpos - kpos < p.window);
                    t[j][i] = seen ? t[j][i] : -INFINITY;
                }
                mx = fmaxf(mx, t[j][i] + (float)((int)(md[j][i] >> 8 & 0xffu) - 127));
            }
        if (!every) {
            // what lies where no key is must not meet a weight of zero: it may be NaN
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (!(md[j][i] & 0x10000u))
#pragma unroll
                        for (int w = 0; w < VWORDS; ++w) vr[j][i].w[w] = 0u;
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = k8_exp2(m - m_use);
        if (__any_sync(0xffffffffu, m_new != m)) {
            l *= alpha;
#pragma unroll
            for (int j = 0; j < NTILES; ++j) {
                o[j][0] *= alpha; o[j][1] *= alpha; o[j][2] *= alpha; o[j][3] *= alpha;
            }
        }
        m = m_new;
        uint32_t ph[2], pl[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int j = 2 * h + (k >> 1), i = k & 1;
                const float e = k8_exp2(t[j][i] - m_use);
                l += e;
                w[k] = e * kv8_scale((md[j][i] >> 8 & 0xffu) + 8u);       // 2^8 times the weight: between 0 and 256
            }
            k8_split(w[0], w[1], w[2], w[3], ph[h], pl[h]);
        }
        // the four keys' numbers of a column side by side, as their weights are
#pragma unroll
        for (int w = 0; w < VWORDS; ++w) {
            uint32_t col[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t a0 = vr[2 * h][0].w[w], a1 = vr[2 * h][1].w[w], a2 = vr[2 * h + 1][0].w[w], a3 = vr[2 * h + 1][1].w[w];
                const uint32_t x0 = __byte_perm(a0, a1, 0x5140), x1 = __byte_perm(a0, a1, 0x7362);
                const uint32_t y0 = __byte_perm(a2, a3, 0x5140), y1 = __byte_perm(a2, a3, 0x7362);
                col[h][0] = __byte_perm(x0, y0, 0x5410); col[h][1] = __byte_perm(x0, y0, 0x7632);
                col[h][2] = __byte_perm(x1, y1, 0x5410); col[h][3] = __byte_perm(x1, y1, 0x7632);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) k8_mma(o[w * 4 + e], ph[0], pl[0], ph[1], pl[1], col[0][e], col[1][e]);
        }
        if (more) {
            load_values(off_w + (at ^ K8S_KEYS));
            meta_w[(at ^ K8S_KEYS) + lane] = ks | vs;
        }
        __syncwarp();
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);

    // merge the warps: row r of warp w at sh[(w * 8 + r) * XROW].  A lane's column n of tile 4 w + e is column 8 words of its lane: the
    // accumulator holds columns 2c and 2c + 1 (as lanes g' of the values), i.e. numbers (2c + i) * 4 VWORDS + 4 w + e of the head
    {
        float* mine = sh + (size_t)(warp * K8S_ROWS + g) * XROW;
#pragma unroll
        for (int j = 0; j < NTILES; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) mine[(2 * c + i) * (VWORDS * 4) + j] = fmaf(o[j][2 + i], 0.0625f, o[j][i]) * 0x1p-8f;
        if (c == 0) {
            mine[HD] = m;
            mine[HD + 1] = l;
        }
    }
    __syncthreads();
    float* xch = sh + NW * K8S_ROWS * XROW;                // cluster: [slice][row][XROW] in the first CTA
    uint32_t xch0 = 0;
    if (CLUSTER) {
        tc::cluster_wait();                                // every CTA of the cluster has started
        xch0 = tc::map_to_rank(tc::smem_addr(xch), 0u);
    }
    for (int idx = threadIdx.x; idx < rows * HD; idx += NW * 32) {
        const int r = idx / HD, d = idx - r * HD, rt = r / p.heads, rh = r - rt * p.heads;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sh[(w * K8S_ROWS + r) * XROW + HD]);
        const float use = M == -INFINITY ? 0.f : M;
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float* x = sh + (w * K8S_ROWS + r) * XROW;
            const float f = k8_exp2(x[HD] - use);
            L += x[HD + 1] * f;
            O += x[d] * f;
        }
        if (CLUSTER) {
            const uint32_t to = xch0 + (uint32_t)((blockIdx.z * rows + r) * XROW) * 4u;
            tc::st_cluster_f32(to + (uint32_t)d * 4u, O);
            if (d == 0) {
                tc::st_cluster_f32(to + (uint32_t)HD * 4u, M);
                tc::st_cluster_f32(to + (uint32_t)(HD + 1) * 4u, L);
            }
        } else if (rh < nheads) {
            p.out[((size_t)(row0 + rt) * p.nh + head0 + rh) * HD + d] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
        }
    }
    if (CLUSTER) {
        tc::cluster_sync();                                // every slice has delivered
        if (blockIdx.z != 0) return;
        for (int idx = threadIdx.x; idx < rows * HD; idx += NW * 32) {
            const int r = idx / HD, d = idx - r * HD, rt = r / p.heads, rh = r - rt * p.heads;
            if (rh >= nheads) continue;
            float M = -INFINITY;
            for (int z = 0; z < p.nsplit; ++z) M = fmaxf(M, xch[(z * rows + r) * XROW + HD]);
            const float use = M == -INFINITY ? 0.f : M;
            float L = 0.f, O = 0.f;
            for (int z = 0; z < p.nsplit; ++z) {           // slices in order
                const float* x = xch + (z * rows + r) * XROW;
                const float f = k8_exp2(x[HD] - use);
                L += x[HD + 1] * f;
                O += x[d] * f;
            }
            p.out[((size_t)(row0 + rt) * p.nh + head0 + rh) * HD + d] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
        }
    }
}

static int k8s_smem(int nw, int rows, int nsplit) {
    return (nw * K8S_ROWS + (nsplit > 1 ? nsplit * rows : 0)) * XROW * (int)sizeof(float);
}

// 1 where ap_attention_kv8_split takes the head size
AP_EXPORT int ap_attention_kv8_split_supports(int hd) { return hd == HD; }

// Tokens of one sequence in a tile: as many as fill its eight rows
AP_EXPORT int ap_attention_kv8_split_tokens(int nh, int nkv) {
    const int group = nh / nkv;
    return group >= K8S_ROWS ? 1 : K8S_ROWS / group;
}

// seq_start null: row r is sequence r's only one (tiles = rows); else `tiles` = the sum over the sequences of ceil(rows / tokens of a
// tile).  nsplit: 1, 2, 4, 8 or 16 key slices; warps: 4 or 8 to a CTA.
AP_EXPORT int ap_attention_kv8_split(const void* q, void* out, const void* cache, long long num_pages, long long page_bytes,
                                     const int* block_table, int max_blocks, const int* seq_start, const int* positions, int nseq,
                                     int tiles, int nh, int nkv, int hd, int P, float scale, int window, int nsplit, int warps,
                                     cudaStream_t stream) {
    AP_REQUIRE(hd == HD, "attention_kv8: this library was compiled for head size %d, not %d", HD, hd);
    AP_REQUIRE(tiles >= 0 && nseq > 0 && nh > 0 && nkv > 0 && nh % nkv == 0 && P > 0 && max_blocks > 0,
               "attention_kv8: bad sizes tiles=%d heads=%d kv_heads=%d page=%d", tiles, nh, nkv, P);
    AP_REQUIRE(num_pages > 0 && num_pages < (1LL << 31) && page_bytes == kv8_page_bytes(nkv, P, HD) && num_pages * page_bytes < (1LL << 36),
               "attention_kv8: the pages do not match the heads, or hold 64 GB and more");
    AP_REQUIRE(((uintptr_t)cache & 15) == 0 && ((uintptr_t)q & 15) == 0, "attention_kv8: operands must be 16-byte aligned");
    AP_REQUIRE((long long)max_blocks * P < (1LL << 31) - 64, "attention_kv8: the block table names more than 2^31 keys");
    AP_REQUIRE(nsplit >= 1 && nsplit <= 16 && (nsplit & (nsplit - 1)) == 0, "attention_kv8: bad number of key slices %d", nsplit);
    AP_REQUIRE(warps == 4 || warps == 8, "attention_kv8: %d warps", warps);
    if (tiles == 0) return AP_OK;
    K8sParams p;
    p.q = (const bf16*)q; p.out = (bf16*)out; p.cache = (const uint8_t*)cache; p.block_table = block_table;
    p.seq_start = seq_start; p.positions = positions; p.page_bytes = (size_t)page_bytes; p.num_pages = (int)num_pages;
    p.max_blocks = max_blocks; p.nseq = nseq; p.nh = nh; p.nkv = nkv; p.P = P; p.window = window; p.nsplit = nsplit;
    p.scale_log2 = scale * 1.4426950408889634f;
    const int group = nh / nkv;
    p.heads = group < K8S_ROWS ? group : K8S_ROWS;
    p.n_chunks = (group + p.heads - 1) / p.heads;
    p.tokens = seq_start ? K8S_ROWS / p.heads : 1;
    AP_REQUIRE(nkv * p.n_chunks <= 65535, "attention_kv8: too many KV heads for the grid");
    static bool configured[64];
    int dev = 0;
    AP_REQUIRE(cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64, "attention_kv8: cannot tell the current device");
    if (!configured[dev]) {
        const void* kernels[4] = {(const void*)attention_kv8_split_kernel<4, false>, (const void*)attention_kv8_split_kernel<8, false>,
                                  (const void*)attention_kv8_split_kernel<4, true>, (const void*)attention_kv8_split_kernel<8, true>};
        for (int i = 0; i < 4; ++i) {
            cudaError_t e = cudaFuncSetAttribute(kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize, k8s_smem(8, K8S_ROWS, i < 2 ? 1 : 16));
            if (e == cudaSuccess && i >= 2) e = cudaFuncSetAttribute(kernels[i], cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            AP_REQUIRE(e == cudaSuccess, "attention_kv8: cannot configure the kernel: %s", cudaGetErrorString(e));
        }
        configured[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles, nkv * p.n_chunks, nsplit);
    cfg.blockDim = dim3(warps * 32);
    cfg.dynamicSmemBytes = k8s_smem(warps, p.tokens * p.heads, nsplit);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = ap_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = nsplit;
    cfg.attrs = attr;
    cfg.numAttrs = nsplit > 1 ? 2 : 1;
    AP_CHECK_PDL_LAUNCH("attention_kv8_split",
                        nsplit > 1 ? (warps == 4 ? cudaLaunchKernelEx(&cfg, attention_kv8_split_kernel<4, true>, p)
                                                 : cudaLaunchKernelEx(&cfg, attention_kv8_split_kernel<8, true>, p))
                                   : (warps == 4 ? cudaLaunchKernelEx(&cfg, attention_kv8_split_kernel<4, false>, p)
                                                 : cudaLaunchKernelEx(&cfg, attention_kv8_split_kernel<8, false>, p)));
    return AP_OK;
}

#else   // head sizes this kernel is not built for

AP_EXPORT int ap_attention_kv8_split_supports(int) { return 0; }

#endif
