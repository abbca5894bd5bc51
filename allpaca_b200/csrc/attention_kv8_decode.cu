// bfloat16 grouped-query attention of single rows over the 8-bit paged cache (kv8.cuh), any head size up to 256 (-DAP_HEAD_DIM), pages
// of 8, 16 or 32 rows or of whole tiles of 64: every row by itself, with its own sequence and position, so a batch of any kind may come.
//
// Such rows stream the cache; the rest has to stay out of the way.  One CTA to an SM lives through the whole launch: two warps
// bring tiles of 64 keys (a TMA box to a page, the scale bytes by cp.async) into a ring in shared memory, eight warps work on
// them, 32 keys at a time each.  The work, all tiles of all (row, KV head) pairs end to end, is cut into runs of equal cost, one
// to a CTA, so no SM waits for another whatever the lengths; the loads never pause, as the ring runs on from one pair into the next,
// and two more warps prepare the next pair's queries and add up the last one's sums meanwhile.  (Loading with cp.async, any page size
// and no swizzle, took four warps 1500 to 2500 cycles of dependent instructions to a tile: 2.5 TB/s.)  A pair that a cut falls
// into is put together by the CTA that finishes its part last: parts go to scratch, nobody waits, and they are added in an order of
// their own.  Few pairs get a cluster of CTAs each instead, whose parts meet in distributed shared memory.
//
// Bound by memory while it streams, at 5.8 to 6.4 TB/s with pages scattered: 64 rows of 2048 keys (8 KV heads of 128: 270 MB, floor 41.9 us at
// the copy rate) take 57.5 us, of which 5.5 pass before the first tile is there (positions, block table and tile are read one after
// the other) and 3 after the last.  One row of 32768 keys (floor 10.5) takes 24.3: 5.5, 10.5 of streaming, the rest until parts are written,
// seen and added up.  Ragged rows (64 of 150 to 4096 keys, floor 24.7) take 47.4: each pair costs four tiles' time beside its own.  Heads of
// 64 (64 rows of 4096 keys: 75.5, floor 42.2) are bound by what the working warps do per tile, which does not shrink with the head.
//
// The numbers are never widened: the products are e4m3 x e4m3 (mma.sync m16n8k32) with the keys, and the columns of the values, as
// the 16 rows, and it is the queries and the weights that are split into two e4m3 numbers, x = hi + lo / 16, side by side in the
// eight columns: four query rows to a product.  That keeps the eight significant bits of bfloat16 (hi is off by half of the last of
// four bits, and so much needs four bits again).  Queries are scaled by a power of two to a row (numbers down to 2^-15 of the largest keep all
// eight bits).  Weights, with their values' scales, lie between 0 and 256, off by 2^-8 of themselves or by 2^-14: so they are taken relative to
// a reference that follows the largest of each 32 keys, up at once, down when those lie 2^4 below it (rescaling the sums then, 1 to 1.5 % of
// the time).  Against one maximum for all keys, weights of less than 2^-22 of it were lost, and of 70000 keys behind one that took nearly
// all of the softmax a tenth of their sum.
//
//   t_j = log2(e) scale 2^a_j (q . c_j),   m >= t_j + b_j,   l = sum_j 2^(t_j - m),   out = sum_j 2^(t_j + b_j - m) d_j / l
//
// with scales 2^a_j of keys and 2^b_j of values: a maximum over what meets the 8-bit numbers keeps the largest products exact
// however values differ in size, and with b_j between -60 and 40, and the reference no more than 2^30 below the maximum, neither sum leaves the
// range of 32-bit numbers.
//
// The key is the summed index of the second product, so four keys' numbers of a column have to lie side by side in a register: a
// transposing ldmatrix brings two columns of two keys, two byte permutes sort two such registers.  Which key is which row of a tile
// is free; it is chosen so that the weights a lane has computed are the four summed indices of one lane of the second product (two
// shuffles), and so that the eight rows of every ldmatrix lie in different banks.
//
// Reference counterparts (cuda/src/kernels.cu): attention_split_gqa_kernel :1874 and attention_merge_kernel :1997.
#include "kv8.cuh"
#include "tcgen05.cuh"
#include <cuda.h>
#include <math.h>

#ifndef AP_HEAD_DIM
#error "compile with -DAP_HEAD_DIM=<head size>"
#endif

#define HD AP_HEAD_DIM
#define CHUNKS (HD / 16)                       // 16-byte chunks of a row
#define TILE 64                                // keys of a tile
#define PWARPS 2
#define CWARPS 8
#define LANES (CWARPS / 2)                     // tiles at work at a time: a pair of warps to each
#define QUERY_WARP (CWARPS + PWARPS)
#define MERGE_WARP (QUERY_WARP + 1)
#define K8D_THREADS ((CWARPS + PWARPS + 2) * 32)
#define MAX_STAGES 24
#define K8D_PAIR_COST 4                        // tiles
#define K8D_FEW_PARTS 4                        // of a pair, up to which one warp adds them up
#define K8D_MAX_ROWS 512                       // of a launch
#define K8D_NEAR 4.f                           // powers of two that a tile's largest weight may lie below what its weights are relative to,
#define K8D_FALL 30.f                          // and that this may lie below the largest of all
// Rows lie in shared memory as TMA leaves them: `BOX` bytes to a row, the 16-byte chunks of 8 (4, 2) rows swizzled where a box is 128 (64,
// 32) bytes wide, so that eight rows of one ldmatrix lie in different banks; other head sizes take what conflicts they have.
#define BOX (HD % 128 == 0 ? 128 : HD)
#define NBOX (HD / BOX)
#define STAGE_BYTES (2 * TILE * HD)            // [box][page][keys, values][row]: a box brings a page's keys and values
#define SCALE_BYTES (2 * TILE)
#define XROW (HD + 8)                          // a partial result: HD sums, maximum, sum of weights (and rows in different banks)
#define K8D_ERR_WAIT 8

static __device__ int g_k8d_status;

struct K8dParams {
    const bf16* q;
    bf16* out;
    const uint8_t* cache;
    const int *block_table, *token_seq, *positions;
    float* parts;                              // [CTA][2][heads][XROW]
    unsigned long long* arrivals;              // [CTA][2]: a part is there when this holds the call's number
    unsigned long long nonce;                  // the call's number: tells its arrivals from whatever the scratch held before
    size_t page_bytes;
    int num_pages, max_blocks, nseq, T, nh, nkv, P, P_shift, window;
    int heads, n_chunks, stages;               // query heads of a pair's product, products to a KV head
    float scale_log2;
};

__device__ __forceinline__ float k8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void k8_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void k8_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void k8_ldmatrix_x2(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(addr) : "memory");
    r[2] = r[3] = 0u;
}
__device__ __forceinline__ void k8_ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 4 bytes to shared memory; zeros where `there` is false
__device__ __forceinline__ void k8_copy4(uint32_t dst, const uint8_t* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void k8_arrive_when_copied(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(tc::smem_addr(bar)) : "memory");
}
// four numbers as hi + lo / 16
__device__ __forceinline__ void k8_split(float a, float b, float c, float d, uint32_t& hi, uint32_t& lo) {
    hi = kv8_pack4(a, b, c, d);
    const float4 h = kv8_unpack(hi);
    lo = kv8_pack4((a - h.x) * 16.f, (b - h.y) * 16.f, (c - h.z) * 16.f, (d - h.w) * 16.f);
}

// Where chunk `ch` of row `key` lies in a stage; value: its value's row, one page further on.
__device__ __forceinline__ uint32_t k8_at(int key, int ch, int rows_shift, bool value) {
    const int box = ch / (BOX / 16), c = ch - box * (BOX / 16), page = key >> rows_shift;
    const int x = BOX == 128 ? key & 7 : BOX == 64 ? (key >> 1) & 3 : BOX == 32 ? (key >> 2) & 1 : 0;
    return (uint32_t)(box * 2 * TILE * BOX + ((((page << 1) | (value ? 1 : 0)) << rows_shift) + (key & ((1 << rows_shift) - 1))) * BOX +
                      ((c ^ x) << 4));
}

// A place in the work: tile `tile` of pair (row, j); tiles of a row from first_of(row) on.
struct K8dAt {
    int row, j, tile, end;                     // end: tiles of the row
};

// The cuts are equal in cost: a pair costs its tiles and `pair` tiles more (its queries, its merging); the first `more` CTAs take one unit
// beyond `each`.
struct K8dWork {
    const int* start;                          // [T + 1] tiles before a row (shared memory)
    int T, J, pair, each, more;
    // the row whose tiles, or costs, hold x
    __device__ __forceinline__ int row_of(int x, int cost) const {
        int lo = 0, hi = T;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((start[mid] + mid * cost) * J <= x) lo = mid; else hi = mid;
        }
        return lo;
    }
    // the first tile of a CTA
    __device__ __forceinline__ int from(int cta) const {
        const int x = cta * each + min(cta, more), row = row_of(x, pair);
        const int in = x - (start[row] + row * pair) * J, end = start[row + 1] - start[row];
        const int j = min(in / (end + pair), J), rest = in - j * (end + pair);
        return start[row] * J + j * end + min(rest, end);
    }
    __device__ __forceinline__ int cta_of(int w) const {
        const int row = row_of(w, 0), end = start[row + 1] - start[row], in = w - start[row] * J, j = in / end;
        const int x = (start[row] + row * pair) * J + in + j * pair, cut = more * (each + 1);
        return x < cut ? x / (each + 1) : more + (x - cut) / each;
    }
    __device__ __forceinline__ K8dAt at(int w) const {
        K8dAt a;
        a.row = row_of(w, 0);
        a.end = start[a.row + 1] - start[a.row];
        const int in = w - start[a.row] * J;
        a.j = in / a.end;
        a.tile = in - a.j * a.end;
        return a;
    }
    __device__ __forceinline__ void next(K8dAt& a, int n) const {
        a.tile += n;
        while (a.tile >= a.end && a.row < T) {
            a.tile -= a.end;
            if (++a.j < J) continue;
            a.j = 0;
            if (++a.row < T) a.end = start[a.row + 1] - start[a.row];
        }
    }
};

// the first key that a row sees whose last one is `last`
__device__ __forceinline__ int k8d_first(const K8dParams& p, int last) {
    return p.window > 0 && last - p.window + 1 > 0 ? last - p.window + 1 : 0;
}

// The working warps' sums of a pair (merge: [warp][4 NT][XROW]) added up by one warp: to the pair's rows of the output, or, unfinished, to
// `part`.
template <int NT>
__device__ __noinline__ void k8d_combine(const float* merge, int nheads, bf16* out, float* part) {
    const int lane = threadIdx.x & 31;
    const bool to_out = part == nullptr;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        // lane 8 h + x: head 4 n + h of working warp x
        const float* head = merge + 4 * n * XROW;
        const float* row = head + ((lane & 7) * 4 * NT + (lane >> 3)) * XROW;
        const float2 ml = *reinterpret_cast<const float2*>(row + HD);
        float M = ml.x;
#pragma unroll
        for (int o = 1; o < CWARPS; o <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float f = k8_exp2(ml.x - (M == -INFINITY ? 0.f : M));
        float L = ml.y * f;
#pragma unroll
        for (int o = 1; o < CWARPS; o <<= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (!to_out && (lane & 7) == 0 && 4 * n + (lane >> 3) < nheads)
            *reinterpret_cast<float2*>(part + (4 * n + (lane >> 3)) * XROW + HD) = make_float2(M, L);
        for (int d0 = 0; d0 < HD; d0 += 128) {     // (all lanes take part in the shuffles)
            const int d = d0 + lane * 4;
            float4 O[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) O[h] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int x = 0; x < CWARPS; ++x)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const float fx = __shfl_sync(0xffffffffu, f, 8 * h + x);
                    const float4 v = *reinterpret_cast<const float4*>(head + (x * 4 * NT + h) * XROW + (d < HD ? d : 0));
                    O[h].x += v.x * fx; O[h].y += v.y * fx; O[h].z += v.z * fx; O[h].w += v.w * fx;
                }
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const float ih = __shfl_sync(0xffffffffu, inv, 8 * h);
                if (d >= HD || 4 * n + h >= nheads) continue;
                if (to_out) {
                    uint2 u;
                    __nv_bfloat162* u2 = reinterpret_cast<__nv_bfloat162*>(&u);
                    u2[0] = __floats2bfloat162_rn(O[h].x * ih, O[h].y * ih);
                    u2[1] = __floats2bfloat162_rn(O[h].z * ih, O[h].w * ih);
                    *reinterpret_cast<uint2*>(out + (4 * n + h) * HD + d) = u;
                } else {
                    *reinterpret_cast<float4*>(part + (4 * n + h) * XROW + d) = O[h];
                }
            }
        }
    }
}

// A pair's few parts added up by one warp, in their order.
template <int NT>
__device__ __noinline__ void k8d_add_few(const float* parts, int i0, int nparts, int heads, int nheads, bf16* out) {
    const int lane = threadIdx.x & 31;
    for (int d0 = 0; d0 < HD; d0 += 128) {
        const int d = d0 + lane * 4;
#pragma unroll 1
        for (int n = 0; n < NT; ++n) {
            float M[4], L[4];
            float4 O[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                M[h] = -INFINITY;
                L[h] = 0.f;
                O[h] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll 2
            for (int i = 0; i < nparts; ++i) {         // in their order
                const float* from = parts + ((size_t)(i0 + i) * 2 + (i == 0 ? 1 : 0)) * heads * XROW;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const float* row = from + min(4 * n + h, nheads - 1) * XROW;
                    const float2 ml = __ldcg(reinterpret_cast<const float2*>(row + HD));
                    const float4 po = __ldcg(reinterpret_cast<const float4*>(row + (d < HD ? d : 0)));
                    const float m_new = fmaxf(M[h], ml.x), use = m_new == -INFINITY ? 0.f : m_new;
                    const float f = k8_exp2(M[h] - use), fk = k8_exp2(ml.x - use);
                    M[h] = m_new;
                    L[h] = L[h] * f + ml.y * fk;
                    O[h].x = O[h].x * f + po.x * fk; O[h].y = O[h].y * f + po.y * fk;
                    O[h].z = O[h].z * f + po.z * fk; O[h].w = O[h].w * f + po.w * fk;
                }
            }
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                if (4 * n + h >= nheads || d >= HD) continue;
                const float inv = L[h] == 0.f ? 0.f : 1.f / L[h];
                uint2 v;
                __nv_bfloat162* v2 = reinterpret_cast<__nv_bfloat162*>(&v);
                v2[0] = __floats2bfloat162_rn(O[h].x * inv, O[h].y * inv);
                v2[1] = __floats2bfloat162_rn(O[h].z * inv, O[h].w * inv);
                *reinterpret_cast<uint2*>(out + (4 * n + h) * HD + d) = v;
            }
        }
    }
}

// NT: products of four query heads.  CL: a pair to a cluster, CTA x of it the x-th part of the pair's tiles (blockIdx.y: the pair).
template <int NT, bool CL>
__global__ void __launch_bounds__(K8D_THREADS, 1)
attention_kv8_decode_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ K8dParams p) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_start[K8D_MAX_ROWS + 1];              // tiles before a row
    __shared__ int s_last[K8D_MAX_ROWS], s_seq[K8D_MAX_ROWS];   // the last key a row sees (-1: none) and its sequence
    __shared__ int s_warp[K8D_THREADS / 32];
    __shared__ int s_dead, s_join[2];
    __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], q_full[2], q_empty[2], dumped, taken;
    __shared__ uint64_t join[2];                           // of either late pair: one is decided while a warp may still wait for the other
    __shared__ uint32_t s_query[2][NT][CHUNKS + 1][32];    // a pair's queries as the products take them; last: the rows' factors
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* scales = smem + (size_t)p.stages * STAGE_BYTES;
    float* merge = reinterpret_cast<float*>(scales + p.stages * SCALE_BYTES);           // [warp][4 NT][XROW]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            tc::mbar_init(&full[s], 1 + 32);               // what TMA brings, and every lane's scale bytes
            tc::mbar_init(&empty[s], 2);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&q_full[i], 1);
            tc::mbar_init(&q_empty[i], CWARPS);
            tc::mbar_init(&join[i], 1);
        }
        tc::mbar_init(&dumped, CWARPS);
        tc::mbar_init(&taken, 1);
        tc::fence_barrier_init();
        tc::prefetch_tensormap(&tmap);
        s_dead = *(volatile int*)&g_k8d_status;            // one reading for all, as they meet at barriers
    }
    ap_pdl_trigger();
    ap_pdl_wait();
    const int J = CL ? 1 : p.nkv * p.n_chunks, T = CL ? 1 : p.T;       // pairs of a row, and rows, in this CTA's work
    const int row0 = CL ? blockIdx.y / (p.nkv * p.n_chunks) : 0, j0 = CL ? blockIdx.y - row0 * (p.nkv * p.n_chunks) : 0;
    // tiles before every row
    if (CL) {
        if (threadIdx.x == 0) {
            const int seq = p.token_seq[row0], pos = p.positions[row0];
            const int last = seq >= 0 && seq < p.nseq ? min(pos, p.max_blocks * p.P - 1) : -1, first = k8d_first(p, last);
            s_last[0] = last;
            s_seq[0] = seq;
            s_start[0] = 0;
            s_start[1] = last >= first ? last / TILE - first / TILE + 1 : 1;
        }
        __syncthreads();
    } else {
        const int per = (p.T + K8D_THREADS - 1) / K8D_THREADS, r0 = threadIdx.x * per;
        int n[(K8D_MAX_ROWS + K8D_THREADS - 1) / K8D_THREADS], sum = 0;
#pragma unroll
        for (int i = 0; i < (K8D_MAX_ROWS + K8D_THREADS - 1) / K8D_THREADS; ++i) {
            n[i] = 0;
            if (i < per && r0 + i < p.T) {
                const int seq = p.token_seq[r0 + i], pos = p.positions[r0 + i];
                const int last = seq >= 0 && seq < p.nseq ? min(pos, p.max_blocks * p.P - 1) : -1, first = k8d_first(p, last);
                s_last[r0 + i] = last;
                s_seq[r0 + i] = seq;
                n[i] = last >= first ? last / TILE - first / TILE + 1 : 1;      // (a row that sees nothing: one empty tile)
            }
            sum += n[i];
        }
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, before, o);
            if (lane >= o) before += v;
        }
        if (lane == 31) s_warp[warp] = before;
        __syncthreads();
        before -= sum;
        for (int w = 0; w < warp; ++w) before += s_warp[w];
#pragma unroll
        for (int i = 0; i < (K8D_MAX_ROWS + K8D_THREADS - 1) / K8D_THREADS; ++i) {
            if (i < per && r0 + i < p.T) s_start[r0 + i] = before;
            before += n[i];
            if (i < per && r0 + i == p.T - 1) s_start[p.T] = before;
        }
        __syncthreads();
    }
    const int W = s_start[T] * J;
    const int G = CL ? (int)gridDim.x : min((int)gridDim.x, W);        // (a cut pair's parts lie in CTAs one behind the other)
    if (!CL && (int)blockIdx.x >= G) return;
    const int pair = CL ? 0 : K8D_PAIR_COST, cost = W + T * J * pair;
    const K8dWork work = {s_start, T, J, pair, cost / G, cost % G};
    const int lo = work.from(blockIdx.x), hi = (int)blockIdx.x + 1 < G ? work.from(blockIdx.x + 1) : W;
    if (!CL && lo >= hi) return;
    // The run's order: its last pair's part where the run ends inside that pair, its first pair's part where it starts inside one, then the
    // whole pairs: what has to be put together with other CTAs' parts is done while there is work left to hide it behind.
    int cut1 = CL ? hi : lo, cut2 = hi;                    // [lo, cut1) the first part, [cut1, cut2) whole pairs, [cut2, hi) the last part
    if (!CL) {
        const K8dAt a = work.at(lo), b = work.at(hi - 1);
        if (a.tile) cut1 = min(hi, lo + a.end - a.tile);
        if (b.tile + 1 < b.end && hi > cut1) cut2 = hi - 1 - b.tile;
        if (cut2 < cut1) cut2 = cut1;
    }
    auto run_from = [&](int seg) { return seg == 0 ? cut2 : seg == 1 ? lo : cut1; };
    auto run_to = [&](int seg) { return seg == 0 ? hi : seg == 1 ? cut1 : cut2; };
    auto place = [&](int v) {                              // the run's v-th tile
        v += cut2;
        if (v < hi) return v;
        v += lo - hi;
        return v;                                          // (first part and whole pairs lie side by side)
    };
    const int tiles = hi - lo;
    if (!CL && s_dead != 0) return;
    const bool dead = s_dead != 0;                         // (a cluster's CTA still goes to the barriers)
    const size_t rows_of_page = (size_t)2 * p.nkv * p.P;

    const int group = p.nh / p.nkv;
    auto give_up = [&] { atomicExch(&g_k8d_status, K8D_ERR_WAIT); };
    float* own_part = merge + CWARPS * 4 * NT * XROW;      // cluster: this CTA's part, [4 NT][XROW]
    const int g = lane >> 2, c = lane & 3;
    // A pair's parts brought by the working warps, this one every CWARPS-th of them, for k8d_combine.
    auto gather = [&](int nparts, auto fetch) {
        for (int d0 = 0; d0 < HD; d0 += 128) {
            const int d = d0 + lane * 4 < HD ? d0 + lane * 4 : 0;
            float M[4 * NT], L[4 * NT];
            float4 O[4 * NT];
#pragma unroll
            for (int h = 0; h < 4 * NT; ++h) {
                M[h] = -INFINITY;
                L[h] = 0.f;
                O[h] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll 1
            for (int i = warp; i < nparts; i += CWARPS) {
                float2 ml[4 * NT];
                float4 po[4 * NT];
#pragma unroll
                for (int h = 0; h < 4 * NT; ++h) fetch(i, min(h, p.heads - 1), d, ml[h], po[h]);      // (heads past the last one: the last one again)
#pragma unroll
                for (int h = 0; h < 4 * NT; ++h) {
                    const float m_new = fmaxf(M[h], ml[h].x), use = m_new == -INFINITY ? 0.f : m_new;
                    const float f = k8_exp2(M[h] - use), fk = k8_exp2(ml[h].x - use);
                    M[h] = m_new;
                    L[h] = L[h] * f + ml[h].y * fk;
                    O[h].x = O[h].x * f + po[h].x * fk; O[h].y = O[h].y * f + po[h].y * fk;
                    O[h].z = O[h].z * f + po[h].z * fk; O[h].w = O[h].w * f + po[h].w * fk;
                }
            }
#pragma unroll
            for (int h = 0; h < 4 * NT; ++h) {
                float* to = merge + (warp * 4 * NT + h) * XROW;
                *reinterpret_cast<float4*>(to + d) = O[h];
                if (d == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(M[h], L[h]);
            }
        }
    };
    if (dead) {
        // nothing more
    } else if (warp >= CWARPS && warp < QUERY_WARP) {
        // ---- loading: the warps take turns.  A warp looks up as many of its tiles at once as their pages fill its lanes, a round
        // ahead of their loads; lane l then owns page l % n_pages of the round's tile l / n_pages ----
        const int pw = warp - CWARPS;
        const int n_pages = p.P < TILE ? TILE / p.P : 1, page_rows = TILE / n_pages, in_round = 32 / n_pages;
        const int mine = lane / n_pages, my_page = lane - mine * n_pages;
        const int s_page = (lane & 15) * 4 / page_rows;    // the page of this lane's scale bytes (keys for lanes 0 to 15, values for the others)
        const uint8_t* const scale_bytes = p.cache + rows_of_page * HD + (lane < 16 ? 0 : p.nkv * p.P) + ((lane & 15) * 4 & (page_rows - 1));
        const uint32_t group_mask = n_pages == 8 ? 0xffu : (1u << n_pages) - 1u;
        auto look_up = [&](int v, int& page, int& krow) {
            page = -1;
            krow = 0;
            if (v < tiles) {
                const K8dAt at = work.at(place(v));
                const int last = s_last[at.row], first = k8d_first(p, last), tile = first / TILE + at.tile;
                const int key0 = tile * TILE + my_page * page_rows;                        // of the page's part of the tile
                if (key0 <= last && key0 + page_rows > first)
                    page = p.block_table[(size_t)s_seq[at.row] * p.max_blocks + (p.P_shift >= 0 ? key0 >> p.P_shift : key0 / p.P)];
                krow = (p.n_chunks == 1 ? j0 + at.j : (j0 + at.j) / p.n_chunks) * p.P + (p.P > TILE ? tile * TILE % p.P : 0);
            }
        };
        int page_n, krow_n;
        look_up(pw + mine * PWARPS, page_n, krow_n);
        int s = pw % p.stages;
        uint32_t ph = 1;                                   // the first round of the ring is free
        bool fine = true;
        for (int v0 = pw; v0 < tiles && fine; v0 += in_round * PWARPS) {
            const int page = page_n < p.num_pages ? page_n : -1, krow = krow_n;
            look_up(v0 + (in_round + mine) * PWARPS, page_n, krow_n);
            const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
            for (int i = 0; i < in_round && v0 + i * PWARPS < tiles; ++i) {
                const int from = i * n_pages, n = __popc(there >> from & group_mask);
                const int page_s = __shfl_sync(0xffffffffu, page, from + s_page), krow_s = __shfl_sync(0xffffffffu, krow, from);
                if (!tc::mbar_wait(&empty[s], ph)) {
                    give_up();
                    fine = false;
                    break;
                }
                if (lane == 0) tc::mbar_expect_tx(&full[s], (uint32_t)(n * page_rows * HD * 2));
                __syncwarp();
                if (mine == i && page >= 0) {
                    uint8_t* to = smem + (size_t)s * STAGE_BYTES + my_page * 2 * page_rows * BOX;
#pragma unroll
                    for (int b = 0; b < NBOX; ++b) tc::tma_load_4d(to + b * 2 * TILE * BOX, &tmap, b * BOX, krow, 0, page, &full[s]);
                }
                k8_copy4(tc::smem_addr(scales + s * SCALE_BYTES) + lane * 4,
                         scale_bytes + (size_t)max(page_s, 0) * p.page_bytes + krow_s, page_s >= 0);
                k8_arrive_when_copied(&full[s]);
                s += PWARPS;
                if (s >= p.stages) { s -= p.stages; ph ^= 1; }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == QUERY_WARP) {
        // ---- queries: of every pair ahead of its turn, split and in the order of the products' operands ----
        int k = 0;
        for (int seg = 0; seg < 3; ++seg) {
            K8dAt at = work.at(min(run_from(seg), W - 1));
            for (int w = run_from(seg); w < run_to(seg); ++k) {
                const int kvh = (j0 + at.j) / p.n_chunks, chunk = j0 + at.j - kvh * p.n_chunks;
                const int head0 = kvh * group + chunk * p.heads, nheads = min(p.heads, group - chunk * p.heads);
                // column g of product n is query head 4 n + g / 2, its high half where g is even
                uint32_t words[NT][CHUNKS];
                float factor[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int hq = 4 * n + (g >> 1);
                    const bf16* qr = p.q + ((size_t)(row0 + at.row) * p.nh + head0 + (hq < nheads ? hq : 0)) * HD + c * 4;
                    uint2 raw[CHUNKS];
                    uint32_t amax = 0;
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) raw[i] = hq < nheads ? *reinterpret_cast<const uint2*>(qr + i * 16) : make_uint2(0u, 0u);
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) {
                        const uint32_t x[4] = {raw[i].x << 16, raw[i].x & 0xffff0000u, raw[i].y << 16, raw[i].y & 0xffff0000u};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t m = x[e] & 0x7fffffffu;
                            amax = max(amax, m < 0x7f800000u ? m : 0u);
                        }
                    }
                    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                    // 2^e with e the smallest exponent under which no number exceeds 448 (kept where 2^e and 2^-e are normal numbers)
                    const int e = min(max((int)(amax >> 23) - 135 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0), -120), 120);
                    const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
                    factor[n] = __shfl_sync(0xffffffffu, p.scale_log2 * __uint_as_float((uint32_t)(127 + e) << 23), 8 * c);   // of head 4 n + c
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) {
                        float x[4] = {__uint_as_float(raw[i].x << 16), __uint_as_float(raw[i].x & 0xffff0000u),
                                      __uint_as_float(raw[i].y << 16), __uint_as_float(raw[i].y & 0xffff0000u)};
#pragma unroll
                        for (int y = 0; y < 4; ++y) x[y] = fmaf(x[y], inv, x[y] - x[y]);       // NaN where not finite
                        uint32_t h, l;
                        k8_split(x[0], x[1], x[2], x[3], h, l);
                        words[n][i] = g & 1 ? l : h;
                    }
                }
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&q_empty[k & 1], (uint32_t)((k >> 1) & 1) ^ 1))) give_up();
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) s_query[k & 1][n][i][lane] = words[n][i];
                    s_query[k & 1][n][CHUNKS][lane] = __float_as_uint(factor[n]);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&q_full[k & 1]);
                w += at.end - at.tile;
                at.tile = at.end - 1;
                work.next(at, 1);
            }
        }
    } else if (warp == MERGE_WARP) {
        // ---- results: the working warps' sums of a pair are added up while they are at the next one ----
        uint32_t ph = 0;
        // The CTAs from cta_of(item0) on hold a cut pair's parts, in their second place where the pair starts in them, else in their
        // first.  Each says that its part is there and then looks whether all are: whoever finds them all adds them up.  (Two
        // may find so at once; they write the same numbers.)  Then the places are free for the next call.
        auto say = [&](int item0) {
            __threadfence();
            __syncwarp();
            if (lane == 0) ((volatile unsigned long long*)p.arrivals)[blockIdx.x * 2 + (item0 >= lo ? 1 : 0)] = p.nonce;
            __threadfence();
            __syncwarp();
        };
        auto all_there = [&](int item0, int nparts) {
            volatile unsigned long long* a = p.arrivals;
            const int i0 = work.cta_of(item0);
            bool all = true;
            for (int i = lane; i < nparts; i += 32) all = all && a[(i0 + i) * 2 + (i == 0 ? 1 : 0)] == p.nonce;
            all = __all_sync(0xffffffffu, all);
            __threadfence();
            if (all)
                for (int i = lane; i < nparts; i += 32) a[(i0 + i) * 2 + (i == 0 ? 1 : 0)] = 0ull;
            return all;
        };
        // Pairs of many parts (the first and the last of this CTA may be such) wait for the end, where the working warps can bring them:
        // then whoever adds them up does it in one and the same order.
        struct { int item0, nparts, nheads; bf16* out; } late[2];
        int n_late = 0;
        // (once on nothing, while the first tiles are on their way: a function's first call waits for its instructions)
        k8d_combine<NT>(merge, 0, nullptr, nullptr);
        for (int seg = 0; seg < 3; ++seg) {
            K8dAt at = work.at(min(run_from(seg), W - 1));
            for (int w = run_from(seg); w < run_to(seg); ph ^= 1) {
                const int kvh = (j0 + at.j) / p.n_chunks, chunk = j0 + at.j - kvh * p.n_chunks;
                const int head0 = kvh * group + chunk * p.heads, nheads = min(p.heads, group - chunk * p.heads);
                const int item0 = w - at.tile, item1 = item0 + at.end;
                const bool whole = item0 >= lo && item1 <= hi;
                bf16* out = p.out + ((size_t)(row0 + at.row) * p.nh + head0) * HD;
                if (!__all_sync(0xffffffffu, tc::mbar_wait(&dumped, ph))) give_up();
                float* part = CL ? own_part : p.parts + ((size_t)blockIdx.x * 2 + (item0 >= lo ? 1 : 0)) * p.heads * XROW;
                k8d_combine<NT>(merge, nheads, out, whole ? nullptr : part);
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&taken);
                if (!CL && !whole) {
                    const int nparts = work.cta_of(item1 - 1) - work.cta_of(item0) + 1;
                    say(item0);
                    if (nparts > K8D_FEW_PARTS) {
                        late[n_late++] = {item0, nparts, nheads, out};
                    } else if (all_there(item0, nparts)) {
                        k8d_add_few<NT>(p.parts, work.cta_of(item0), nparts, p.heads, nheads, out);
                    }
                }
                w = item1;
                at.tile = at.end - 1;
                work.next(at, 1);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (i >= n_late) break;
            const bool all = all_there(late[i].item0, late[i].nparts);
            if (lane == 0) s_join[i] = all ? 1 : 0;
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&join[i]);
            if (!all) continue;
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&dumped, ph))) {
                give_up();
                return;
            }
            ph ^= 1;
            k8d_combine<NT>(merge, late[i].nheads, late[i].out, nullptr);
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&taken);
        }
    } else {
        // ---- working: warps 2 i and 2 i + 1 take the two halves of every fourth tile (LANES) ----
        const int half = warp & 1, turn = warp >> 1;
        const int rows_shift = p.P < TILE ? p.P_shift : 6;     // rows of a page in a tile
        // rows of the tile that this lane's addresses of ldmatrix name (see above: row r of a product is key 2 r and 2 r + 1)
        const int r8 = lane & 7, mat = lane >> 3;
        const int key_a = 2 * r8 + (r8 >= 4 ? 1 : 0), key_b = 2 * r8 + (r8 >= 4 ? 0 : 1);
        const int k_key = half * 32 + (mat & 1 ? key_b : key_a);
        const int v_key = half * 32 + (mat & 1) * 16 + (mat & 2 ? 8 + (r8 ^ 1) : r8);
        const int my_a = half * 32 + 2 * g + (g >= 4 ? 1 : 0), my_b = half * 32 + 2 * g + (g >= 4 ? 0 : 1);   // and + 16
        bool ok = true;
        int s = 0;                                             // stage and phase of tile `w`
        uint32_t ph = 0;
        int k = 0, v = 0, n_late = 0, late0 = 0, late1 = 0, parts0 = 0, parts1 = 0;
        for (int seg = 0; seg < 3; ++seg) {
            K8dAt at = work.at(min(run_from(seg), W - 1));
            for (int w = run_from(seg); w < run_to(seg); ++k) {
                // one pair, or the part of it that is this CTA's
                const int item0 = w - at.tile, item1 = item0 + at.end, stop = item1 < hi ? item1 : hi;
                const int last = s_last[at.row], first = k8d_first(p, last);
                if (ok && !__all_sync(0xffffffffu, tc::mbar_wait(&q_full[k & 1], (uint32_t)((k >> 1) & 1)))) {
                    give_up();
                    ok = false;
                }
                uint32_t qf[NT][CHUNKS + 1];
                float rowfac[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) qf[n][i] = s_query[k & 1][n][i][lane];
                    qf[n][CHUNKS] = 0u;
                    rowfac[n] = __uint_as_float(s_query[k & 1][n][CHUNKS][lane]);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&q_empty[k & 1]);
                float o[NT][CHUNKS][4], m[NT], l[NT], top[NT];         // m: what the sums are relative to; top: the largest so far
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    m[n] = top[n] = -INFINITY;
                    l[n] = 0.f;
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
                }
                for (; w < stop; ++w, ++v) {
                    const int st = s;
                    const uint32_t sp = ph;
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                    const int tile = w - item0;
                    if ((v & (LANES - 1)) != turn) continue;
                    if (ok && !__all_sync(0xffffffffu, tc::mbar_wait(&full[st], sp))) {
                        give_up();
                        ok = false;
                    }
                    if (!ok) continue;
                    uint8_t* stage = smem + (size_t)st * STAGE_BYTES;
                    const uint32_t base = tc::smem_addr(stage);
                    float sc[NT][2][4];
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
#pragma unroll
                        for (int n = 0; n < NT; ++n) sc[n][t][0] = sc[n][t][1] = sc[n][t][2] = sc[n][t][3] = 0.f;
#pragma unroll
                        for (int i = 0; i < CHUNKS; i += 2) {
                            uint32_t a[4];
                            if (i + 1 < CHUNKS) k8_ldmatrix(a, base + k8_at(k_key + t * 16, i + (mat >> 1), rows_shift, false));
                            else k8_ldmatrix_x2(a, base + k8_at(k_key + t * 16, i, rows_shift, false));
#pragma unroll
                            for (int n = 0; n < NT; ++n) k8_mma(sc[n][t], a, qf[n][i], qf[n][i + 1]);
                        }
                    }
                    // scale bytes of this lane's keys: 2 g and 2 g + 1 (the other way round from g = 4 on), 16 further on the same; 0 where there
                    // is no page
                    uint32_t kb[4], vb[4];
                    {
                        const uint8_t* bytes = scales + st * SCALE_BYTES;
#pragma unroll
                        for (int t = 0; t < 2; ++t) {
                            const uint32_t k2 = *reinterpret_cast<const uint16_t*>(bytes + half * 32 + t * 16 + 2 * g);
                            const uint32_t v2 = *reinterpret_cast<const uint16_t*>(bytes + TILE + half * 32 + t * 16 + 2 * g);
                            const uint32_t k0 = k2 & 0xffu, k1 = k2 >> 8, v0 = v2 & 0xffu, v1 = v2 >> 8;
                            kb[2 * t] = g >= 4 ? k1 : k0;
                            kb[2 * t + 1] = g >= 4 ? k0 : k1;
                            vb[2 * t] = g >= 4 ? v1 : v0;
                            vb[2 * t + 1] = g >= 4 ? v0 : v1;
                        }
                    }
                    const int key0 = (first / TILE + tile) * TILE + half * 32;
                    const bool inside = key0 >= first && key0 + 31 <= last;
                    const bool every = __all_sync(0xffffffffu, inside && kb[0] && kb[1] && kb[2] && kb[3]);
                    uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                    if (!every) {
                        // keys before the first, behind the last, or without a page do not count, and what lies in the place of their values
                        // must not meet a weight of zero: it may be NaN.  (keep0, keep1: a byte to a key of the second product's
                        // operand in this lane)
                        uint32_t keep = 0u;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int kpos = key0 - half * 32 + (i & 1 ? my_b : my_a) + (i >> 1) * 16;
                            if (kpos < first || kpos > last) kb[i] = 0u;
                            if (!kb[i]) vb[i] = 0u;
                            keep |= kb[i] ? 0xffu << (8 * i) : 0u;
                        }
                        keep0 = __shfl_sync(0xffffffffu, keep, 4 * c);
                        keep1 = __shfl_sync(0xffffffffu, keep, 4 * c + 16);
                    }
                    uint32_t b0[NT], b1[NT];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float t[4], mx = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float* q2 = sc[n][i >> 1] + 2 * (i & 1);
                            t[i] = fmaf(q2[1], 0.0625f, q2[0]) * (rowfac[n] * kv8_scale(kb[i]));
                            t[i] = kb[i] ? t[i] : -INFINITY;
                            mx = fmaxf(mx, t[i] + ((float)vb[i] - 127.f));
                        }
                        // (heads, four of them, with a key that is near the reference from below)
                        uint32_t near = __ballot_sync(0xffffffffu, mx >= m[n] - K8D_NEAR);
                        near |= near >> 16;
                        near |= near >> 8;
                        near |= near >> 4;
                        if (__any_sync(0xffffffffu, mx > m[n]) || (near & 0xfu) != 0xfu) {
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            top[n] = fmaxf(top[n], mx);
                            float m_new = fmaxf(m[n], mx);
                            if (mx < m[n] - K8D_NEAR && mx > -INFINITY) m_new = fmaxf(mx, top[n] - K8D_FALL);
                            const float alpha = m_new == -INFINITY ? 0.f : k8_exp2(m[n] - m_new);
                            m[n] = m_new;
                            l[n] *= alpha;
#pragma unroll
                            for (int i = 0; i < CHUNKS; ++i) {
                                o[n][i][0] *= alpha; o[n][i][1] *= alpha; o[n][i][2] *= alpha; o[n][i][3] *= alpha;
                            }
                        }
                        const float m_use = m[n] == -INFINITY ? 0.f : m[n];
                        float wt[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = k8_exp2(t[i] - m_use);
                            l[n] += e;
                            wt[i] = e * kv8_scale(vb[i] + 8u);     // 2^8 times the weight
                        }
                        uint32_t hi4, lo4;
                        k8_split(wt[0], wt[1], wt[2], wt[3], hi4, lo4);
                        const int from = 4 * c + (g >> 1);
                        const uint32_t h0 = __shfl_sync(0xffffffffu, hi4, from), l0 = __shfl_sync(0xffffffffu, lo4, from);
                        const uint32_t h1 = __shfl_sync(0xffffffffu, hi4, from + 16), l1 = __shfl_sync(0xffffffffu, lo4, from + 16);
                        b0[n] = g & 1 ? l0 : h0;
                        b1[n] = g & 1 ? l1 : h1;
                    }
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i) {
                        uint32_t r[4], a[4];
                        k8_ldmatrix_trans(r, base + k8_at(v_key, i, rows_shift, true));
                        a[0] = __byte_perm(r[0], r[1], 0x6420);
                        a[1] = __byte_perm(r[0], r[1], 0x7531);
                        a[2] = __byte_perm(r[2], r[3], 0x6420);
                        a[3] = __byte_perm(r[2], r[3], 0x7531);
                        if (!every) {
                            a[0] &= keep0; a[1] &= keep0;
                            a[2] &= keep1; a[3] &= keep1;
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) k8_mma(o[n][i], a, b0[n], b1[n]);
                    }
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&empty[st]);
                }
                // ---- the pair's part is done: hand the sums over ----
                if (ok && k > 0 && !__all_sync(0xffffffffu, tc::mbar_wait(&taken, (uint32_t)((k - 1) & 1)))) {
                    give_up();
                    ok = false;
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 4);
                    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 8);
                    l[n] += __shfl_xor_sync(0xffffffffu, l[n], 16);
                    float* to = merge + (warp * 4 * NT + 4 * n + c) * XROW;
#pragma unroll
                    for (int i = 0; i < CHUNKS; ++i)
                        *reinterpret_cast<float2*>(to + i * 16 + 2 * g) = make_float2(fmaf(o[n][i][1], 0.0625f, o[n][i][0]) * 0x1p-8f,
                                                                                      fmaf(o[n][i][3], 0.0625f, o[n][i][2]) * 0x1p-8f);
                    if (g == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(m[n], l[n]);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&dumped);
                if (!CL && (item0 < lo || item1 > hi)) {
                    const int nparts = work.cta_of(item1 - 1) - work.cta_of(item0) + 1;
                    if (nparts > K8D_FEW_PARTS) {
                        late0 = n_late ? late0 : item0;
                        late1 = item0;
                        parts0 = n_late ? parts0 : nparts;
                        parts1 = nparts;
                        ++n_late;
                    }
                }
                at.tile = at.end - 1;
                work.next(at, 1);
            }
        }
        // pairs of many parts: where all are there, bring them, this warp every CWARPS-th
        for (int i = 0; i < n_late; ++i) {
            if (!ok || !__all_sync(0xffffffffu, tc::mbar_wait(&join[i], 0))) {
                give_up();
                return;
            }
            const bool all = s_join[i] != 0;
            const int nparts = i ? parts1 : parts0, i0 = work.cta_of(i ? late1 : late0);
            if (!all) continue;
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&taken, (uint32_t)((k - 1) & 1)))) {
                give_up();
                return;
            }
            ++k;
            gather(nparts, [&](int i, int h, int d, float2& ml, float4& po) {
                const float* row = p.parts + (((size_t)(i0 + i) * 2 + (i == 0 ? 1 : 0)) * p.heads + h) * XROW;
                ml = __ldcg(reinterpret_cast<const float2*>(row + HD));
                po = __ldcg(reinterpret_cast<const float4*>(row + d));
            });
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&dumped);
        }
    }
    if (CL && G > 1) {
        tc::cluster_sync();                                // every CTA's part is in its shared memory
        const int nparts = min(G, W);                      // (CTAs beyond hold nothing)
        if (blockIdx.x == 0 && nparts > 1) {
            if (warp < CWARPS)
                gather(nparts, [&](int i, int h, int d, float2& ml, float4& po) {
                    const uint32_t row = tc::map_to_rank(tc::smem_addr(own_part + h * XROW), (uint32_t)i);
                    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ml.x), "=f"(ml.y) : "r"(row + HD * 4));
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(po.x), "=f"(po.y), "=f"(po.z), "=f"(po.w) : "r"(row + d * 4));
                });
            __syncthreads();
            if (warp == MERGE_WARP) {
                const int kvh = j0 / p.n_chunks, chunk = j0 - kvh * p.n_chunks, head0 = kvh * group + chunk * p.heads;
                k8d_combine<NT>(merge, min(p.heads, group - chunk * p.heads), p.out + ((size_t)row0 * p.nh + head0) * HD, nullptr);
            }
        }
        tc::cluster_sync();                                // nobody leaves while its part may be read
    }
}

static int k8d_merge_bytes(int nt) { return (CWARPS + 1) * 4 * nt * XROW * (int)sizeof(float); }
#define K8D_STATIC (12 * (K8D_MAX_ROWS + 1) + 1024 + 4 * 2 * 2 * (CHUNKS + 1) * 32)      // the kernel's own shared memory, not quite
static int k8d_stages(int nt) {
    const int n = (227 * 1024 - 1024 - 1024 - K8D_STATIC - k8d_merge_bytes(nt)) / (STAGE_BYTES + SCALE_BYTES);
    return n > MAX_STAGES ? MAX_STAGES : n / LANES * LANES;                // a stage belongs to one loading warp and its pair of working ones
}

typedef CUresult (*K8dEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                CUtensorMapFloatOOBfill);

static K8dEncodeFn k8d_encode_fn() {
    static K8dEncodeFn fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = (K8dEncodeFn)ptr;
    }
    return fn;
}

// 1 where ap_attention_kv8_decode takes pages of P rows: 8, 16, 32, or whole tiles (scale words and swizzle atoms do not straddle pages)
AP_EXPORT int ap_attention_kv8_decode_takes(int P) { return (P == 8 || P == 16 || P == 32 || (P > 0 && P % TILE == 0 && P <= 65536)) && k8d_encode_fn(); }

// Query heads of a product's columns: a KV head's, up to eight.
static int k8d_heads(int nh, int nkv) { const int g = nh / nkv; return g < 8 ? g : 8; }

// The attributes of the kernels, once on every device
static int k8d_configure() {
    static bool configured[64];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return AP_ERR_LAUNCH;
    if (configured[dev]) return AP_OK;
    const void* kernels[4] = {(const void*)attention_kv8_decode_kernel<1, false>, (const void*)attention_kv8_decode_kernel<2, false>,
                              (const void*)attention_kv8_decode_kernel<1, true>, (const void*)attention_kv8_decode_kernel<2, true>};
    for (int i = 0; i < 4; ++i) {
        const int n = 1 + (i & 1);
        if (cudaFuncSetAttribute(kernels[i], cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 k8d_stages(n) * (STAGE_BYTES + SCALE_BYTES) + k8d_merge_bytes(n) + 1024) != cudaSuccess ||
            (i >= 2 && cudaFuncSetAttribute(kernels[i], cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess))
            return AP_ERR_LAUNCH;
    }
    configured[dev] = true;
    return AP_OK;
}

// Clusters of `cluster` CTAs that the current device runs at a time (its SMs come in groups that a cluster does not straddle).
AP_EXPORT int ap_attention_kv8_decode_clusters(int nh, int nkv, int cluster) {
    if (cluster < 1 || cluster > 16 || nkv <= 0 || k8d_configure() != AP_OK) return 0;
    const int nt = k8d_heads(nh, nkv) > 4 ? 2 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster, 1);
    cfg.blockDim = dim3(K8D_THREADS);
    cfg.dynamicSmemBytes = k8d_stages(nt) * (STAGE_BYTES + SCALE_BYTES) + k8d_merge_bytes(nt) + 1024;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    const cudaError_t e = nt == 1 ? cudaOccupancyMaxActiveClusters(&n, attention_kv8_decode_kernel<1, true>, &cfg)
                                  : cudaOccupancyMaxActiveClusters(&n, attention_kv8_decode_kernel<2, true>, &cfg);
    if (e != cudaSuccess) cudaGetLastError();                  // (nothing to the next launch)
    return e == cudaSuccess ? n : 0;
}

// Bytes of scratch that ap_attention_kv8_decode needs for `ctas` CTAs.
AP_EXPORT long long ap_attention_kv8_decode_scratch(int nh, int nkv, int ctas) {
    return 16LL * ctas + 8LL * ctas * k8d_heads(nh, nkv) * XROW;
}

// One launch for T rows.  cluster 0: `ctas` CTAs share the work whatever its lengths.  cluster 1, 2, 4, 8 or 16: so many CTAs to every pair
// of a row and a KV head, which add up their parts through the cluster's shared memory (for few pairs; no scratch).  scratch:
// ap_attention_kv8_decode_scratch bytes, 16-byte aligned, of any contents but those of a call that runs at the same time; nonce: another one
// for every call on the same scratch (a call may be run again, as from a graph, once it has ended).
AP_EXPORT int ap_attention_kv8_decode(const void* q, void* out, const void* cache, long long num_pages, long long page_bytes,
                                      const int* block_table, int max_blocks, int nseq, const int* token_seq, const int* positions,
                                      int T, int nh, int nkv, int hd, int P, float scale, int window, int ctas, int cluster, void* scratch,
                                      long long scratch_bytes, long long nonce, cudaStream_t stream) {
    AP_REQUIRE(hd == HD, "attention_kv8: this library was compiled for head size %d, not %d", HD, hd);
    AP_REQUIRE(T >= 0 && T <= K8D_MAX_ROWS && nseq > 0 && nh > 0 && nkv > 0 && nh % nkv == 0 && P > 0 && max_blocks > 0,
               "attention_kv8: bad sizes T=%d heads=%d kv_heads=%d page=%d", T, nh, nkv, P);
    AP_REQUIRE(num_pages > 0 && num_pages < (1LL << 31) && page_bytes == kv8_page_bytes(nkv, P, HD) && num_pages * page_bytes < (1LL << 36),
               "attention_kv8: the pages do not match the heads, or hold 64 GB and more");
    AP_REQUIRE(((uintptr_t)cache & 15) == 0 && ((uintptr_t)q & 15) == 0, "attention_kv8: operands must be 16-byte aligned");
    AP_REQUIRE((long long)max_blocks * P < (1LL << 31) - 128, "attention_kv8: the block table names more than 2^31 keys");
    AP_REQUIRE(ap_attention_kv8_decode_takes(P), "attention_kv8: pages of %d rows are not taken by the kernel for single rows", P);
    AP_REQUIRE(ctas > 0 && ctas < 65536, "attention_kv8: bad number of CTAs %d", ctas);
    AP_REQUIRE(cluster >= 0 && cluster <= 16 && (cluster & (cluster - 1)) == 0, "attention_kv8: bad cluster size %d", cluster);
    AP_REQUIRE(cluster || ((uintptr_t)scratch & 15) == 0 && scratch && scratch_bytes >= ap_attention_kv8_decode_scratch(nh, nkv, ctas),
               "attention_kv8: %lld bytes of scratch are too few", scratch_bytes);
    const int heads = k8d_heads(nh, nkv), chunks = (nh / nkv + heads - 1) / heads;
    AP_REQUIRE((long long)T * nkv * chunks * ((long long)max_blocks * P / TILE + 2 + K8D_PAIR_COST) < (1LL << 31),
               "attention_kv8: %d rows over block tables of %d pages are more than 2^31 tiles", T, max_blocks);
    if (T == 0) return AP_OK;
    K8dParams p;
    p.q = (const bf16*)q; p.out = (bf16*)out; p.cache = (const uint8_t*)cache;
    p.block_table = block_table; p.token_seq = token_seq; p.positions = positions;
    p.arrivals = (unsigned long long*)scratch;
    p.parts = cluster ? nullptr : (float*)(p.arrivals + (size_t)ctas * 2);
    p.nonce = (unsigned long long)nonce;
    p.page_bytes = (size_t)page_bytes; p.num_pages = (int)num_pages; p.max_blocks = max_blocks; p.nseq = nseq; p.T = T;
    p.nh = nh; p.nkv = nkv; p.P = P; p.window = window; p.heads = heads; p.n_chunks = chunks;
    p.P_shift = -1;
    for (int i = 0; i < 31; ++i)
        if (P == 1 << i) p.P_shift = i;
    p.scale_log2 = scale * 1.4426950408889634f;
    const int nt = heads > 4 ? 2 : 1;
    p.stages = k8d_stages(nt);
    const int smem = p.stages * (STAGE_BYTES + SCALE_BYTES) + k8d_merge_bytes(nt) + 1024;
    AP_REQUIRE(k8d_configure() == AP_OK, "attention_kv8: cannot configure the kernel for single rows");
    CUtensorMap map;
    {
        // [page][keys, values][KV head and row][number]: a box is a page of one head, its keys and its values
        cuuint64_t dims[4] = {(cuuint64_t)HD, (cuuint64_t)nkv * P, 2, (cuuint64_t)num_pages};
        cuuint64_t strides[3] = {(cuuint64_t)HD, (cuuint64_t)nkv * P * HD, (cuuint64_t)page_bytes};
        cuuint32_t box[4] = {BOX, (cuuint32_t)(P < TILE ? P : TILE), 2, 1};
        cuuint32_t es[4] = {1, 1, 1, 1};
        const CUtensorMapSwizzle sw = BOX == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : BOX == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                      : BOX == 32 ? CU_TENSOR_MAP_SWIZZLE_32B : CU_TENSOR_MAP_SWIZZLE_NONE;
        AP_REQUIRE(k8d_encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<void*>(cache), dims, strides, box, es,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
                   "attention_kv8: cannot encode the cache tensor map");
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = cluster ? dim3(cluster, T * nkv * chunks) : dim3(ctas);
    cfg.blockDim = dim3(K8D_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = ap_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster ? cluster : 1;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    AP_REQUIRE(!cluster || (long long)T * nkv * chunks <= 65535, "attention_kv8: too many pairs for clusters");
    AP_CHECK_PDL_LAUNCH("attention_kv8_decode",
                        cluster ? (nt == 1 ? cudaLaunchKernelEx(&cfg, attention_kv8_decode_kernel<1, true>, map, p)
                                           : cudaLaunchKernelEx(&cfg, attention_kv8_decode_kernel<2, true>, map, p))
                                : (nt == 1 ? cudaLaunchKernelEx(&cfg, attention_kv8_decode_kernel<1, false>, map, p)
                                           : cudaLaunchKernelEx(&cfg, attention_kv8_decode_kernel<2, false>, map, p)));
    return AP_OK;
}

AP_EXPORT int ap_attention_kv8_decode_status(void) {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_k8d_status, sizeof(int)) != cudaSuccess) return -1;
    return v;
}
