// Causal grouped-query attention of portions over the 8-bit paged cache (kv8.cuh) on the 5th-generation tensor cores, for head sizes
// 64 and 128 (-DAP_HEAD_DIM): sequences that bring several new rows each, from two on, packed one behind the other.
//
// Two kernels.  The first widens the keys that the step's rows see, once: c * 2^e, exact in bfloat16, from pages into dense rows of
// scratch memory, a sequence's keys of one KV head one behind the other; what lies outside, or has no page, becomes zeros, and so do values
// that are not finite (their NaN is put back at the end, in the rows that see them: looking for them costs 0 to 3 % of the call).  The
// second has the arithmetic of attention_tcgen05_wide.cu: a CTA owns up to 256 rows, two tiles "a" and "b" of (128 / group) tokens x the
// `group` query heads of one KV head, and every tile of 128 keys serves both; S and O live in tensor memory, the two tiles take turns
// on the tensor cores while the other's softmax warps work (one row to a thread, P in bfloat16 over the S it came from, O scaled
// down only when a row's maximum has grown by more than 2^8 over its reference).  Its loads are one box to half a tile.
//
// Widening first costs 5 bytes of traffic to a number (one read, two written, two read again), the last four in L2 where the keys fit there.
// Widening inside the second kernel, every tile in every CTA that reads it, was built and measured: four to six warps needed 3400 to 5100
// cycles to a key tile, loading a box to a page 4400, where the products and the softmax need 3700: 1470 us for 2048 rows behind 30000 keys
// (1.04 TFLOP), the two kernels 1005; 17 rows behind 8191 keys 39 us, the two kernels 29.
//
// A query tile without a second one beside it (few rows) walks two key tiles at once, each half of the CTA its own: 17 rows behind 32000
// keys 77 us, one by one 104.  2048 rows behind 30000 keys run at 1.04 PFLOP/s, 0.62 of the measured peak of a dense bfloat16 product:
// the tensor pipe and the exponentials are each about half busy, taking turns on the same scores.  Few rows are bound by the way
// from one key tile to the next (2 us for two of them), the widening (6 us of 29 behind 8191 keys, 31 of 77 behind 32000) and the
// slices' meeting (7).
//
// Few rows leave most SMs idle: then the keys are cut into slices, a cluster of 2, 4 or 8 CTAs works on one set of rows, and the slices'
// sums are added up through distributed shared memory, every CTA taking its share of the rows: no third launch, no scratch for them.
//
// Every wait is bounded; when one runs out a status word is raised and the results are void.
//
// Reference counterpart: attention_qtile_kernel (cuda/src/kernels.cu:1801), causal rule :1583-1585.
#include "kv8.cuh"
#include "tcgen05.cuh"
#include <cuda.h>
#include <math.h>

#ifndef AP_HEAD_DIM
#error "compile with -DAP_HEAD_DIM=<head size>"
#endif

#if (AP_HEAD_DIM == 64 || AP_HEAD_DIM == 128)

#define HD AP_HEAD_DIM
#define NHALF (HD / 64)
#define BQ 128
#define BKV 128
#define SUB_BYTES (128 * 128)              // a [128 rows x 64 bf16] sub-tile
#define Q_BYTES (NHALF * SUB_BYTES)        // one query tile
#define KV_BYTES (NHALF * SUB_BYTES)       // K (or V) of one tile
// One query tile (NX = 1) or two to a CTA: threads (four softmax warps to a tile; loading warp, MMA warp, two idle ones), stages of K and V,
// columns of tensor memory (S: 128 to a tile, O: HD)
#define T8_THREADS(NX) ((NX) * 128 + 128)
#define T8_STAGES(NX) (NX)
#define T8_TMEM_COLS(NX) ((NX) * 256)
#define T8_O_COL(NX) ((NX) * 128)
#define T8_PITCH (HD + 4)                  // a row of sums that slices exchange, in floats
#define LOG2E_F 1.4426950408889634f
#define T8_ERR_WAIT 9

static __device__ int g_t8_status;

__device__ __forceinline__ float t8_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// 2^x by the special-function unit; exactly 0 for x = -inf
__device__ __forceinline__ float t8_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct AttnT8Params {
    bf16* out;
    const uint8_t* cache;
    size_t page_bytes;
    int* spoiled;                                         // [sequence][KV head][tile of its keys]: a value in it is not finite
    const int* block_table;
    const int* seq_start;
    const int* positions;
    int num_pages, max_blocks, nseq, nh, nkv, P, window, group, tokens_per_tile;   // tokens_per_tile: of one query tile
    int nsplit, tiles;                                    // tiles: dense ones of a sequence's keys in one KV head
    float scale_log2;
};

// The keys kmin .. kmax that `ntok` rows from row0 on see (kmax < 0: none)
__device__ __forceinline__ void t8_span(const int* positions, int row0, int ntok, int window, int last_key, int& kmin, int& kmax) {
    kmax = min(positions[row0 + ntok - 1], last_key);
    const int first = min(positions[row0], last_key);
    kmin = (window > 0 && first - window + 1 > 0) ? first - window + 1 : 0;
}

// A sequence's dense tiles hold its keys from tile t0 on, the first that its rows see, up to last_key
__device__ __forceinline__ void t8_dense(const AttnT8Params& p, int first_row, int& t0, int& last_key) {
    const int last = p.max_blocks * p.P - 1;
    t0 = p.window > 0 ? max(min(p.positions[first_row], last) - p.window + 1, 0) / BKV : 0;
    last_key = (int)min((long long)last, ((long long)t0 + p.tiles) * BKV - 1);
}

// 0x80 in the bytes of a word of e4m3 numbers that are NaN
__device__ __forceinline__ uint32_t t8_not_finite(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// ---- widening: grid (tiles of a sequence's keys, keys and values of every KV head, sequences) ----
// Values that are not finite become zeros here, since the product with the values takes every row of a query tile at once and a weight of
// zero does not undo a NaN; the tile is noted, and the rows that do see the value get their NaN at the second kernel's end.
#define T8_WIDEN_THREADS 256
__global__ void __launch_bounds__(T8_WIDEN_THREADS)
kv8_widen_kernel(const __grid_constant__ AttnT8Params p, bf16* __restrict__ dense) {
    const uint8_t* __restrict__ const cache = p.cache;
    const size_t page_bytes = p.page_bytes;
    __shared__ long long at_s[BKV];                       // where a key's numbers lie (-1: nowhere)
    __shared__ float scale_s[BKV];
    const int s = blockIdx.z, plane = blockIdx.y;
    // the second kernel may start once everything before this one has ended: it reads all but this one's result ahead of its own wait
    ap_pdl_wait();
    ap_pdl_trigger();
    const int row0 = p.seq_start[s], ntok = p.seq_start[s + 1] - row0;
    if (ntok <= 0) return;
    int kmin, kmax, t0, last_key;
    t8_dense(p, row0, t0, last_key);
    t8_span(p.positions, row0, ntok, p.window, last_key, kmin, kmax);
    const int t = t0 + blockIdx.x;
    if (kmax < 0 ? t > 0 : t > kmax / BKV) return;                          // (rows that see nothing still multiply one tile)
    if (threadIdx.x < BKV) {
        const int kpos = t * BKV + threadIdx.x;
        long long at = -1;
        float scale = 0.f;
        if (kpos >= kmin && kpos <= kmax) {
            const int page = p.block_table[(size_t)s * p.max_blocks + kpos / p.P];
            if (page >= 0 && page < p.num_pages) {
                const size_t row = (size_t)plane * p.P + kpos % p.P;
                at = (long long)((size_t)page * page_bytes + row * HD);
                scale = kv8_scale(cache[(size_t)page * page_bytes + (size_t)2 * p.nkv * p.P * HD + row]);
            }
        }
        at_s[threadIdx.x] = at;
        scale_s[threadIdx.x] = scale;
    }
    __syncthreads();
    // eight numbers to a thread and turn: whole rows of 8-byte loads and 16-byte stores side by side
    bf16* to = dense + (((size_t)s * 2 * p.nkv + plane) * p.tiles + blockIdx.x) * BKV * HD;
    constexpr int kItems = BKV * HD / 8 / T8_WIDEN_THREADS;
    uint2 u[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int e = i * T8_WIDEN_THREADS + threadIdx.x, r = e / (HD / 8);
        const long long at = at_s[r];
        u[i] = at >= 0 ? *reinterpret_cast<const uint2*>(cache + at + (e - r * (HD / 8)) * 8) : make_uint2(0u, 0u);
    }
    if (plane >= p.nkv) {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const uint32_t x = t8_not_finite(u[i].x), y = t8_not_finite(u[i].y);
            u[i].x &= ~((x >> 7) * 0xffu);
            u[i].y &= ~((y >> 7) * 0xffu);
            bad |= x | y;
        }
        const int any = __syncthreads_or((int)bad);
        if (threadIdx.x == 0) p.spoiled[((size_t)s * p.nkv + plane - p.nkv) * p.tiles + blockIdx.x] = any ? 1 : 0;
    }
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int e = i * T8_WIDEN_THREADS + threadIdx.x, r = e / (HD / 8);
        const float f = scale_s[r];
        const float4 a = kv8_unpack(u[i].x), b = kv8_unpack(u[i].y);
        uint4 o;
        __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o);
        o2[0] = __floats2bfloat162_rn(a.x * f, a.y * f);
        o2[1] = __floats2bfloat162_rn(a.z * f, a.w * f);
        o2[2] = __floats2bfloat162_rn(b.x * f, b.y * f);
        o2[3] = __floats2bfloat162_rn(b.z * f, b.w * f);
        *reinterpret_cast<uint4*>(to + (size_t)e * 8) = o;
    }
}

template <int NX> struct T8Smem {
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + NX * Q_BYTES;
    static constexpr int kV = kK + T8_STAGES(NX) * KV_BYTES;
    static constexpr int kBars = kV + T8_STAGES(NX) * KV_BYTES;
    static constexpr int kTotal = kBars + 256 + 1024;             // + alignment slack
    // slices: [row of the tiles][T8_PITCH], then [row][maximum, sum], over Q, K and V when all is done
    static constexpr int kSums = 0;
    static constexpr int kStats = NX * BQ * T8_PITCH * 4;
    static_assert(kStats + NX * BQ * 8 <= kBars, "the slices' sums lie over the tiles");
};

template <bool SPLIT, int NX>
__global__ void __launch_bounds__(T8_THREADS(NX), NX == 1 ? 2 : 1)
attention_kv8_tcgen05_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_kv,
                             const AttnT8Params p) {
    using Smem = T8Smem<NX>;
    constexpr int kStages = T8_STAGES(NX), kLoadWarp = 4 * NX, kMmaWarp = kLoadWarp + 1, kOCol = T8_O_COL(NX);
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t* bars = (uint64_t*)(smem + Smem::kBars);
    uint64_t* q_full = bars + 0;
    uint64_t* k_full = bars + 1;                          // [stage]
    uint64_t* v_full = k_full + 2;                        // [stage]
    uint64_t* k_free = v_full + 2;                        // [stage]
    uint64_t* v_free = k_free + 2;                        // [stage]
    uint64_t* s_full = v_free + 2;                        // [query tile]
    uint64_t* p_ready = s_full + 2;                       // [query tile]
    uint64_t* o_full = p_ready + 2;                       // [query tile]: the last product into O is done
    uint32_t* tmem_slot = (uint32_t*)(o_full + 2);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    volatile int* s_seq = (volatile int*)(tmem_slot + 2);
    volatile int* s_tile = (volatile int*)(tmem_slot + 3);
    volatile int* s_spoiled = (volatile int*)(tmem_slot + 4);     // a value among the keys of the CTA's rows is not finite

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int per_cta = NX * p.tokens_per_tile;           // tokens of one CTA

    if (threadIdx.x == 0) {
        tc::mbar_init(q_full, 1);
        for (int x = 0; x < 2; ++x) {
            tc::mbar_init(&k_full[x], 1);
            tc::mbar_init(&v_full[x], 1);
            tc::mbar_init(&k_free[x], 1);
            tc::mbar_init(&v_free[x], 1);
            tc::mbar_init(&s_full[x], 1);
            tc::mbar_init(&p_ready[x], 4);                // one arrival per warp of the tile's group
            tc::mbar_init(&o_full[x], 1);
        }
        *abort_flag = 0;
        *s_spoiled = 0;
        tc::fence_barrier_init();
        tc::prefetch_tensormap(&tmap_q);
        tc::prefetch_tensormap(&tmap_kv);
    }
    // the second query tile starts as zeros: it may not exist
    for (int i = threadIdx.x; NX == 2 && i < Q_BYTES / 16; i += T8_THREADS(NX))
        reinterpret_cast<uint4*>(smem + Smem::kQ + Q_BYTES)[i] = make_uint4(0, 0, 0, 0);
    tc::fence_proxy_async();
    if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, T8_TMEM_COLS(NX));
    if (warp == 0) {
        // late portions of a sequence have the most keys to walk: hand them out first
        // (the KV head is the fast index of the grid: all heads of the longest portions start first)
        int t = (int)((gridDim.x - 1 - blockIdx.x) / (unsigned)p.nkv), found = -1;
        for (int s0 = 0; s0 < p.nseq && found < 0; s0 += 32) {         // 32 sequences' CTAs at once
            const int s = s0 + lane;
            int n = s < p.nseq ? (p.seq_start[s + 1] - p.seq_start[s] + per_cta - 1) / per_cta : 0, upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto > t);
            if (past) {
                found = s0 + __ffs(past) - 1;
                t -= __shfl_sync(0xffffffffu, upto - n, __ffs(past) - 1);
            } else {
                t -= __shfl_sync(0xffffffffu, upto, 31);
            }
        }
        if (lane == 0) {
            *s_seq = *(volatile int*)&g_t8_status != 0 ? -1 : found;   // (after an earlier failure: nothing, but the barriers)
            *s_tile = t;
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const int seq = *s_seq;
    const uint32_t tmem_base = *tmem_slot;
    const bool active = seq >= 0;

    // geometry of this CTA (identical in every thread)
    const int G = p.group;
    int row0 = 0, ntok = 0, kmax = -1, kmin = 0, kvh = 0, head0 = 0, t0 = 0, last_key = -1;
    if (active) {
        row0 = p.seq_start[seq] + *s_tile * per_cta;
        ntok = min(per_cta, p.seq_start[seq + 1] - row0);
        kvh = (int)(blockIdx.x % (unsigned)p.nkv);
        head0 = kvh * G;
    }
    const bool has_b = NX == 2 && ntok > p.tokens_per_tile;          // the second query tile holds rows
    // Where there is no second tile its place takes every other key tile of the first one's rows, as one more slice
    const bool halves = SPLIT && NX == 2 && !has_b;
    if (active) {
        t8_dense(p, p.seq_start[seq], t0, last_key);
        t8_span(p.positions, row0, ntok, p.window, last_key, kmin, kmax);
        kmin = max(kmin, t0 * BKV);                        // (positions that do not rise find no tile before the first)
    }
    int t_lo = kmin / BKV, t_hi = active ? kmax / BKV : -1;
    if (SPLIT) {
        const int each = (t_hi - t_lo + 1 + p.nsplit - 1) / p.nsplit;
        t_lo += (int)blockIdx.y * each;
        t_hi = min(t_hi, t_lo + each - 1);
    }
    const int ntiles = max(t_hi - t_lo + 1, 0);
    const int* table = p.block_table + (size_t)(active ? seq : 0) * p.max_blocks;
    // The pages of a tile's keys, one to a lane (a page larger than a tile: lane 0's), are looked at only to know which are not there
    const int page_rows = min(p.P, BKV), n_pages = BKV / page_rows;
    auto page_of = [&](int it) {
        const int key0 = (t_lo + it) * BKV + lane * page_rows;
        if (it >= ntiles || lane >= n_pages || key0 > kmax || key0 + page_rows - 1 < kmin) return 0;
        const int page = table[key0 / p.P];
        return page < p.num_pages ? page : -1;
    };

    float mref = -INFINITY, l = 0.f;                   // a softmax thread's row: its reference maximum (log2 units) and sum
    bool ok = true;                                    // the same in all lanes of a warp

    // Registers move from the warps that only issue copies and products to the softmax warps, which hold a row of 128 scores each (the
    // unit of such a move is four warps): 2 x 224 + 56 = 504 to a thread of each, or 192 + 64 = 256, what the launch holds.
    if (warp >= kLoadWarp) {
    if (NX == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == kLoadWarp) {
        if (!(active && ntiles > 0)) {
            ap_pdl_wait();                                 // (no CTA ends before the widening has)
        } else {
            if (lane == 0) {
                tc::mbar_expect_tx(q_full, (uint32_t)((has_b ? 2 : 1) * Q_BYTES));
                for (int x = 0; x < (has_b ? 2 : 1); ++x)
                    for (int h = 0; h < NHALF; ++h)
                        tc::tma_load_3d(smem + Smem::kQ + x * Q_BYTES + h * SUB_BYTES, &tmap_q, h * 64, head0,
                                        row0 + x * p.tokens_per_tile, q_full);
                ap_pdl_wait();                             // the widened keys and values
                const int k_row = ((seq * 2 * p.nkv + kvh) * p.tiles + t_lo - t0) * BKV, v_row = k_row + p.nkv * p.tiles * BKV;
                auto load = [&](int it, int row, uint64_t* full, uint64_t* free, int base) -> bool {
                    const int s = it % kStages;
                    if (*abort_flag) return false;
                    if (!tc::mbar_wait(&free[s], (uint32_t)((it / kStages) & 1) ^ 1)) {
                        *abort_flag = 1;
                        atomicExch(&g_t8_status, T8_ERR_WAIT);
                        return false;
                    }
                    tc::mbar_expect_tx(&full[s], KV_BYTES);
                    for (int h = 0; h < NHALF; ++h)
                        tc::tma_load_2d(smem + base + s * KV_BYTES + h * SUB_BYTES, &tmap_kv, h * 64, row + it * BKV, &full[s]);
                    return true;
                };
                // K runs one tile ahead of V
                bool fine = load(0, k_row, k_full, k_free, Smem::kK);
                for (int it = 0; it < ntiles && fine; ++it) {
                    if (NX == 1) fine = load(it, v_row, v_full, v_free, Smem::kV);       // (one stage: V of this tile is free first)
                    if (fine && it + 1 < ntiles) fine = load(it + 1, k_row, k_full, k_free, Smem::kK);
                    if (NX == 2 && fine) fine = load(it, v_row, v_full, v_free, Smem::kV);
                }
            }
        }
    } else if (warp == kMmaWarp + 1) {
        if (active) {
            ap_pdl_wait();                                 // the widened keys and values
            const int* flags = p.spoiled + ((size_t)seq * p.nkv + kvh) * p.tiles - t0;
            int bad = 0;
            for (int t = kmin / BKV + lane; t <= kmax / BKV; t += 32) bad |= __ldcg(flags + t);
            bad = __any_sync(0xffffffffu, bad != 0);
            if (lane == 0) *s_spoiled = bad;
        }
    } else if (warp == kMmaWarp) {
        if (lane == 0 && active && ntiles > 0) {
            constexpr uint32_t idesc_s = tc::instr_desc_bf16_f32(BQ, BKV);
            constexpr uint32_t idesc_o = tc::instr_desc_bf16_f32_b_mn(BQ, HD);
            const int nx = has_b ? 2 : 1;
            // S_x = Q_x K^T of key tile `it`
            auto scores = [&](int it, int x) {
                const int of = halves ? 0 : x;
                const int s = it % kStages;
#pragma unroll
                for (int h = 0; h < NHALF; ++h) {
                    const uint64_t qd = tc::smem_desc_k_major_sw128(smem + Smem::kQ + of * Q_BYTES + h * SUB_BYTES);
                    const uint64_t kd = tc::smem_desc_k_major_sw128(smem + Smem::kK + s * KV_BYTES + h * SUB_BYTES);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        tc::mma_bf16(tmem_base + (uint32_t)(x * BKV), qd + 2 * k, kd + 2 * k, idesc_s, (h > 0 || k > 0) ? 1u : 0u);
                }
                tc::mma_commit(&s_full[x]);
            };
            // O_x += P_x V of key tile `it`, the first of x's or not
            auto values = [&](int it, int x, bool first) {
                const uint64_t vd = tc::smem_desc_mn_major_sw128(smem + Smem::kV + it % kStages * KV_BYTES, SUB_BYTES);
                const uint32_t pt = tmem_base + (uint32_t)(x * BKV);      // P_x lies over S_x
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                    tc::mma_bf16_a_tmem(tmem_base + (uint32_t)(kOCol + x * HD), pt + (uint32_t)(ks * 8),
                                        vd + (uint64_t)(ks * (16 * 128 / 16)), idesc_o, (!first || ks > 0) ? 1u : 0u);
            };
            ok = tc::mbar_wait(q_full, 0);
            if (halves) {
                // two chains of their own: tile `it` is x = it % 2's, and so are its stages
                for (int x = 0; x < 2 && x < ntiles && ok; ++x) {
                    ok = tc::mbar_wait(&k_full[x], 0);
                    if (!ok) break;
                    tc::fence_after_sync();
                    scores(x, x);
                    tc::mma_commit(&k_free[x]);
                }
                for (int it = 0; it < ntiles && ok; ++it) {
                    const int x = it & 1;
                    const uint32_t ph = (uint32_t)((it >> 1) & 1);
                    const bool more = it + 2 < ntiles;
                    ok = tc::mbar_wait(&v_full[x], ph) && (!more || tc::mbar_wait(&k_full[x], ph ^ 1u)) && tc::mbar_wait(&p_ready[x], ph);
                    if (!ok || *abort_flag) break;
                    tc::fence_after_sync();
                    values(it, x, it < 2);
                    tc::mma_commit(more ? &v_free[x] : &o_full[x]);
                    if (more) {
                        scores(it + 2, x);
                        tc::mma_commit(&k_free[x]);
                    }
                }
            }
            if (ok && !halves) ok = tc::mbar_wait(&k_full[0], 0);
            if (ok && !halves) {
                tc::fence_after_sync();
                for (int x = 0; x < nx; ++x) scores(0, x);
                tc::mma_commit(&k_free[0]);
            }
            for (int it = 0; it < ntiles && ok && !halves; ++it) {
                const int sv = it % kStages, sk = (it + 1) % kStages;
                const bool more = it + 1 < ntiles;
                ok = tc::mbar_wait(&v_full[sv], (uint32_t)((it / kStages) & 1)) &&
                     (!more || tc::mbar_wait(&k_full[sk], (uint32_t)(((it + 1) / kStages) & 1)));
                if (!ok || *abort_flag) break;
                for (int x = 0; x < nx && ok; ++x) {
                    // O_x += P_x V as soon as the tile's group has written P_x (and scaled O_x down where a row's reference
                    // maximum moved); then S_x of the next key tile, which the group turns to while the other tile's products run
                    ok = tc::mbar_wait(&p_ready[x], (uint32_t)(it & 1));
                    if (!ok) break;
                    tc::fence_after_sync();
                    values(it, x, it == 0);
                    if (!more) tc::mma_commit(&o_full[x]);
                    if (NX == 1) tc::mma_commit(&v_free[sv]);
                    if (more) scores(it + 1, x);
                }
                if (!ok) break;
                if (more) {
                    if (NX == 2) tc::mma_commit(&v_free[sv]);
                    tc::mma_commit(&k_free[sk]);
                }
            }
            if (!ok && !*abort_flag) {
                *abort_flag = 1;
                atomicExch(&g_t8_status, T8_ERR_WAIT);
            }
        }
    }
    } else {
    if (NX == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    if (active && (warp < 4 || has_b || halves)) {
        // ---- softmax: warps 0..3 own query tile a, warps 4..7 tile b; one row per thread ----
        const int x = warp >> 2;
        const int qtr = warp & 3;
        const int r = qtr * 32 + lane;                 // row of the tile = (token r / G, head r % G)
        const int tok = (halves ? 0 : x * p.tokens_per_tile) + r / G, hq = r % G;
        const int it0 = halves ? x : 0, step = halves ? 2 : 1;         // the key tiles of this query tile
        const bool rvalid = tok < ntok;
        const uint32_t lane_base = tmem_base + ((uint32_t)(qtr * 32) << 16);
        const uint32_t s_cols = lane_base + (uint32_t)(x * BKV);
        const uint32_t o_cols = lane_base + (uint32_t)(kOCol + x * HD);
        const int qpos = min(p.positions[row0 + (rvalid ? tok : 0)], last_key);
        int page = page_of(it0);
        uint32_t ph = 0;
        for (int it = it0; it < ntiles; it += step, ph ^= 1u) {
            const int k0 = (t_lo + it) * BKV;
            // pages that are not there (rare: a caller gives them back behind a window)
            const uint32_t gone = __ballot_sync(0xffffffffu, page < 0);
            page = page_of(it + step);
            // tcgen05.ld and .st are warp-wide instructions: whatever decides whether one runs is a vote
            if (!__all_sync(0xffffffffu, tc::mbar_wait(&s_full[x], ph))) { ok = false; break; }
            tc::fence_after_sync();
            // (rows that are none see everything: their sums go nowhere)
            const bool row_all = !rvalid || (k0 + BKV - 1 <= qpos && (p.window <= 0 || qpos - k0 < p.window));
            const bool row_none = !rvalid || k0 > qpos || (p.window > 0 && qpos - (k0 + BKV - 1) >= p.window);
            const bool all_visible = __all_sync(0xffffffffu, row_all) && gone == 0;
            const bool none_visible = __all_sync(0xffffffffu, row_none);
            float lsum = 0.f;
            if (none_visible) {
                // nothing of this tile is for this warp's rows: P = 0
                uint32_t zero[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) zero[j] = 0u;
                tc::tmem_st_x32(s_cols, zero);
                tc::tmem_st_x32(s_cols + 32u, zero);
            } else {
                // the row's 128 scores, masked ones as -inf (their probability below is exactly zero)
                uint32_t v[128];
#pragma unroll
                for (int c = 0; c < 128; c += 32) tc::tmem_ld_x32(s_cols + (uint32_t)c, v + c);
                tc::tmem_ld_wait();
                if (!all_visible) {
#pragma unroll
                    for (int j = 0; j < 128; ++j) {
                        const int kpos = k0 + j;
                        const bool vis = kpos <= qpos && (p.window <= 0 || qpos - kpos < p.window);
                        v[j] = vis ? v[j] : 0xff800000u;
                    }
                    if (gone != 0) {
#pragma unroll
                        for (int j = 0; j < 128; j += 8) {                 // (pages are of eight rows at least)
                            if (gone >> (j / page_rows) & 1u) {
#pragma unroll
                                for (int e = 0; e < 8; ++e) v[j + e] = 0xff800000u;
                            }
                        }
                    }
                }
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < 128; j += 2)
                    mx4[(j >> 1) & 3] = t8_max3(mx4[(j >> 1) & 3], __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                // the scale is positive: the maximum of the scaled scores is the scaled maximum
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
                const bool grow = mx > mref + 8.0f;            // also the row's first visible key
                float alpha = 1.f;
                if (grow) {
                    alpha = t8_exp2(mref - mx);                // 0 when the row had no key yet
                    mref = mx;
                    l *= alpha;
                }
                if (it > it0 && __any_sync(0xffffffffu, grow)) {
                    // scale this warp's rows of O_x down.  The product of the tile before into O_x is in: it was issued before the
                    // scores whose arrival (s_full) this warp has seen, and an arrival stands for everything issued before it
#pragma unroll 1
                    for (int c = 0; c < HD; c += 32) {
                        uint32_t w[32];
                        tc::tmem_ld_x32(o_cols + (uint32_t)c, w);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; ++j) w[j] = __float_as_uint(__uint_as_float(w[j]) * alpha);
                        tc::tmem_st_x32(o_cols + (uint32_t)c, w);
                    }
                    tc::tmem_st_wait();
                }
                // probabilities, two bfloat16 to a column, over the first half of S
                const float muse = mref == -INFINITY ? 0.f : mref;
                const float2 scale2 = make_float2(p.scale_log2, p.scale_log2), shift2 = make_float2(-muse, -muse);
                float2 l2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int j = 0; j < 128; j += 2) {
                    const float2 a = __ffma2_rn(make_float2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), scale2, shift2);
                    const float2 e = make_float2(t8_exp2(a.x), t8_exp2(a.y));
                    l2[(j >> 1) & 1] = __fadd2_rn(l2[(j >> 1) & 1], e);
                    __nv_bfloat162 b2 = __floats2bfloat162_rn(e.x, e.y);
                    v[j >> 1] = *reinterpret_cast<uint32_t*>(&b2);
                }
                lsum = (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
                tc::tmem_st_x32(s_cols, v);
                tc::tmem_st_x32(s_cols + 32u, v + 32);
            }
            l += lsum;
            tc::tmem_st_wait();
            tc::fence_before_sync();
            __syncwarp();                       // every lane's part of P is written: one arrival for the warp
            if (lane == 0) tc::mbar_arrive(&p_ready[x]);
        }
        // the last product into O_x, then the row goes out, or to the other slices
        if (ok && ntiles > it0 && !__all_sync(0xffffffffu, tc::mbar_wait(&o_full[x], 0))) ok = false;
        tc::fence_after_sync();
        if (!ok) {
            if (!*abort_flag) {
                *abort_flag = 1;
                atomicExch(&g_t8_status, T8_ERR_WAIT);
            }
        } else if (SPLIT) {
            // (this tile's products may be done before the other's, whose operands the sums are about to lie over)
            if ((has_b || halves) && ntiles > (halves ? x ^ 1 : 0)) ok = __all_sync(0xffffffffu, tc::mbar_wait(&o_full[x ^ 1], 0));
        } else {
            const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;     // (a sum that is not a number stays one)
            bf16* dst = p.out + ((size_t)(row0 + (rvalid ? tok : 0)) * p.nh + head0 + hq) * HD;
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t w[32];
                if (ntiles > 0) {
                    tc::tmem_ld_x32(o_cols + (uint32_t)c, w);
                    tc::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int d = 0; d < 32; ++d) w[d] = 0u;
                }
                if (rvalid) {
#pragma unroll
                    for (int d = 0; d < 32; d += 8) {
                        uint4 o8;
                        __nv_bfloat162* o2 = reinterpret_cast<__nv_bfloat162*>(&o8);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            o2[e] = __floats2bfloat162_rn(__uint_as_float(w[d + 2 * e]) * inv, __uint_as_float(w[d + 2 * e + 1]) * inv);
                        *reinterpret_cast<uint4*>(dst + c + d) = o8;
                    }
                }
            }
        }
    }
    }
    if (SPLIT) {
        // The slices' sums meet in CTA i % nsplit for row i, over the tiles (the cluster's products are all done): every thread sends its
        // row there (halves: source 2 z + x is tile x of slice z).  Then a thread to a row turns its sources' maxima and sums into weights,
        // and all threads add up, four numbers each, in the sources' order.  3.2 us to send and 2 to add for 17 rows of 4 heads, 4 and 4 for
        // 512 rows in two slices: barriers and code that runs for the first time, not bytes (unrolled four times it adds no faster,
        // a row to a warp at a time, 10 us).
        const int ns = p.nsplit, shift = __ffs(ns) - 1, rank = (int)blockIdx.y, x = warp >> 2;
        const int sources = halves ? 2 * ns : ns, rows = (halves ? BQ : NX * BQ) >> shift;       // rows of a source that meet here
        tc::cluster_sync();
        if (warp < kLoadWarp && active && (warp < 4 || has_b || halves)) {
            const int r = (warp & 3) * 32 + lane, i = halves ? r : x * BQ + r;
            const uint32_t o_cols = tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(kOCol + x * HD);
            const int slot = (halves ? 2 * rank + x : rank) * rows + (i >> shift);
            const uint32_t to = (uint32_t)(i & (ns - 1));
            const uint32_t sums = tc::map_to_rank(tc::smem_addr(smem + Smem::kSums) + (uint32_t)(slot * T8_PITCH) * 4u, to);
            const uint32_t stats = tc::map_to_rank(tc::smem_addr(smem + Smem::kStats) + (uint32_t)slot * 8u, to);
            const bool sends = i < ntok * G, some = ntiles > (halves ? x : 0);
            if (sends) asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(stats), "f"(mref), "f"(l) : "memory");
#pragma unroll 1
            for (int c = 0; c < HD; c += 32) {
                uint32_t w[32];
                if (some) {
                    tc::tmem_ld_x32(o_cols + (uint32_t)c, w);
                    tc::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int d = 0; d < 32; ++d) w[d] = 0u;
                }
#pragma unroll
                for (int d = 0; d < 32; d += 4)
                    if (sends)
                        asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(sums + (uint32_t)(c + d) * 4u), "r"(w[d]),
                                     "r"(w[d + 1]), "r"(w[d + 2]), "r"(w[d + 3])
                                     : "memory");
            }
        }
        tc::cluster_sync();
        const int mine = (ntok * G - rank + ns - 1) >> shift;
        float2* all_stats = reinterpret_cast<float2*>(smem + Smem::kStats);
        if ((int)threadIdx.x < mine) {
            float2* stat = all_stats + threadIdx.x;
            float M = -INFINITY, L = 0.f;
#pragma unroll 1
            for (int z = 0; z < sources; ++z) M = fmaxf(M, stat[z * rows].x);
            const float use = M == -INFINITY ? 0.f : M;
#pragma unroll 1
            for (int z = 0; z < sources; ++z) L += stat[z * rows].y * t8_exp2(stat[z * rows].x - use);
            const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
            for (int z = 0; z < sources; ++z) stat[z * rows].x = t8_exp2(stat[z * rows].x - use) * inv;
        }
        __syncthreads();
#pragma unroll 1
        for (int k = threadIdx.x; k < mine * (HD / 4); k += T8_THREADS(NX)) {
            const int n = k / (HD / 4), d = k % (HD / 4) * 4;
            const float* v = reinterpret_cast<const float*>(smem + Smem::kSums) + (size_t)n * T8_PITCH + d;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int z = 0; z < sources; ++z) {
                const float w = all_stats[z * rows + n].x;
                const float4 o = *reinterpret_cast<const float4*>(v + (size_t)z * rows * T8_PITCH);
                acc.x = fmaf(w, o.x, acc.x); acc.y = fmaf(w, o.y, acc.y);
                acc.z = fmaf(w, o.z, acc.z); acc.w = fmaf(w, o.w, acc.w);
            }
            const int i = (n << shift) + rank, tok = i / G, hq = i - tok * G;
            uint2 u;
            __nv_bfloat162* u2 = reinterpret_cast<__nv_bfloat162*>(&u);
            u2[0] = __floats2bfloat162_rn(acc.x, acc.y);
            u2[1] = __floats2bfloat162_rn(acc.z, acc.w);
            *reinterpret_cast<uint2*>(p.out + ((size_t)(row0 + tok) * p.nh + head0 + hq) * HD + d) = u;
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (*s_spoiled && warp < kLoadWarp) {
        // Rows that see a value which is not finite: its column becomes NaN.  A row to a lane, among those that this CTA wrote; the 32 lanes
        // look at 32 keys at a time and tell one another which of them are spoiled, column by column, until all columns are (2048 rows behind
        // 30000 keys: 1.15 ms where every value is, 4.2 where one in every tile is, 1.0 where none is).  Whose rows they are is looked up
        // again: the registers were the softmax's.
        const int s = *s_seq, first_row = p.seq_start[s] + *s_tile * per_cta, n = min(per_cta, p.seq_start[s + 1] - first_row);
        const int head = (int)(blockIdx.x % (unsigned)p.nkv), i = (SPLIT ? p.nsplit : 1) * (int)threadIdx.x + (SPLIT ? (int)blockIdx.y : 0);
        const bool row = i < n * p.group;
        const int tok = row ? i / p.group : 0;
        int k_first, k_last, t_first, last;
        t8_dense(p, p.seq_start[s], t_first, last);
        t8_span(p.positions, first_row, n, p.window, last, k_first, k_last);
        uint32_t done[HD / 32];                            // columns that are NaN already
#pragma unroll
        for (int j = 0; j < HD / 32; ++j) done[j] = row ? 0u : 0xffffffffu;
        const int pos = row ? min(p.positions[first_row + tok], last) : -1;
        bf16* dst = p.out + ((size_t)(first_row + tok) * p.nh + head * p.group + (row ? i - tok * p.group : 0)) * HD;
        const int* flags = p.spoiled + ((size_t)s * p.nkv + head) * p.tiles - t_first;
        for (int t = max(k_first / BKV, t_first); t <= k_last / BKV; ++t) {
            if (__ldcg(flags + t) == 0) continue;
            for (int k0 = t * BKV; k0 < (t + 1) * BKV; k0 += 32) {
                const int key = k0 + lane;
                const int page = key >= k_first && key <= k_last ? p.block_table[(size_t)s * p.max_blocks + key / p.P] : -1;
                const bool there = page >= 0 && page < p.num_pages;
                const uint8_t* v = p.cache + (there ? (size_t)page * p.page_bytes + ((size_t)(p.nkv + head) * p.P + key % p.P) * HD : 0);
                // of these keys the row sees lo .. hi
                const int lo = p.window > 0 ? max(pos - p.window + 1 - k0, 0) : 0, hi = min(pos - k0, 31);
                const uint32_t sees = hi < lo ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
#pragma unroll
                for (int j = 0; j < HD / 32; ++j) {
#pragma unroll 1
                    for (int w = 0; w < 32; w += 4) {
                        const uint32_t bad = there ? t8_not_finite(*reinterpret_cast<const uint32_t*>(v + 32 * j + w)) : 0u;
                        if (!__any_sync(0xffffffffu, bad != 0)) continue;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool sees_one = (__ballot_sync(0xffffffffu, bad >> (8 * e) & 0x80u) & sees) != 0;
                            if (sees_one && !(done[j] >> (w + e) & 1u)) {
                                dst[32 * j + w + e] = __float2bfloat16(NAN);
                                done[j] |= 1u << (w + e);
                            }
                        }
                    }
                }
            }
            bool all = true;
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) all = all && done[j] == 0xffffffffu;
            if (__all_sync(0xffffffffu, all)) break;
        }
    }
    ap_pdl_trigger();
    if (warp == kMmaWarp) {
        __syncwarp();
        tc::tmem_dealloc(tmem_base, T8_TMEM_COLS(NX));
    }
}

// ---------------------------------------------------------------------------
typedef CUresult (*T8EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                               CUtensorMapFloatOOBfill);

static T8EncodeFn t8_encode_fn() {
    static T8EncodeFn fn = nullptr;
    if (!fn) {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
            fn = (T8EncodeFn)ptr;
    }
    return fn;
}

// 1 when ap_attention_kv8_tcgen05 takes this shape, else 0
AP_EXPORT int ap_attention_kv8_tcgen05_takes(int nh, int nkv, int hd, int P) {
    if (hd != HD || nkv <= 0 || nh % nkv) return 0;
    const int g = nh / nkv;
    if (g > 128 || 128 % g) return 0;
    if (P < 8 || (P < BKV ? BKV % P : P % BKV)) return 0;
    return t8_encode_fn() != nullptr;
}

// tokens of one sequence in a query tile
AP_EXPORT int ap_attention_kv8_tcgen05_tokens(int nh, int nkv) { return 128 / (nh / nkv); }

// Bytes of scratch for `tiles` tiles of 128 keys, of all sequences together
AP_EXPORT long long ap_attention_kv8_tcgen05_scratch(long long tiles, int nkv) {
    return (tiles * nkv * (2 * 2 * BKV * HD + 4) + 15) / 16 * 16;
}

// q: [T][nh][HD]; query_tiles: 1 or 2 to a CTA; total_ctas: the sum over the sequences of ceil(rows / tokens of a CTA); nsplit: 1, 2, 4 or
// 8 key slices; scale > 0; tiles: tiles of 128 keys that a sequence's rows see at most, from the first one that they see on (keys beyond
// them are not seen); scratch: ap_attention_kv8_tcgen05_scratch(nseq * tiles, nkv) bytes of any contents, 16-byte aligned, of no call that runs
// at the same time.
AP_EXPORT int ap_attention_kv8_tcgen05(const void* q, void* out, const void* cache, long long num_pages, long long page_bytes,
                                       const int* block_table, int max_blocks, const int* seq_start, const int* positions, int nseq, int T,
                                       int nh, int nkv, int hd, int P, float scale, int window, int query_tiles, int total_ctas, int nsplit, int tiles, void* scratch,
                                       long long scratch_bytes, cudaStream_t stream) {
    AP_REQUIRE(ap_attention_kv8_tcgen05_takes(nh, nkv, hd, P), "attention_kv8 (tcgen05): shape not supported: heads=%d kv_heads=%d "
               "head_dim=%d page=%d", nh, nkv, hd, P);
    AP_REQUIRE(T > 0 && nseq > 0 && total_ctas > 0 && max_blocks > 0, "attention_kv8 (tcgen05): bad sizes");
    AP_REQUIRE(num_pages >= 0 && num_pages < (1LL << 31) && page_bytes == kv8_page_bytes(nkv, P, HD), "attention_kv8: the pages do not match the heads");
    AP_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)cache & 15) == 0 && ((uintptr_t)out & 15) == 0 && ((uintptr_t)scratch & 15) == 0,
               "attention_kv8 (tcgen05): operands must be 16-byte aligned");
    AP_REQUIRE((long long)max_blocks * P < (1LL << 31) - 128, "attention_kv8 (tcgen05): the block table names more than 2^31 keys");
    AP_REQUIRE(tiles > 0 && tiles < (1 << 24), "attention_kv8 (tcgen05): %d tiles of keys", tiles);
    const long long dense_rows = (long long)nseq * 2 * nkv * tiles * BKV;
    AP_REQUIRE(dense_rows < (1LL << 31) - 256, "attention_kv8 (tcgen05): %lld rows of keys and values are too many", dense_rows);
    AP_REQUIRE(scratch && scratch_bytes >= ap_attention_kv8_tcgen05_scratch((long long)nseq * tiles, nkv), "attention_kv8 (tcgen05): %lld bytes of "
               "scratch are too few", scratch_bytes);
    AP_REQUIRE(query_tiles == 1 || query_tiles == 2, "attention_kv8 (tcgen05): %d query tiles", query_tiles);
    AP_REQUIRE(scale > 0.f, "attention_kv8 (tcgen05): the scale must be positive");
    AP_REQUIRE(nsplit >= 1 && nsplit <= 8 && (nsplit & (nsplit - 1)) == 0, "attention_kv8: bad number of key slices %d", nsplit);
    AP_REQUIRE(nseq <= 65535 && 2 * nkv <= 65535, "attention_kv8 (tcgen05): %d sequences of %d KV heads exceed the grid", nseq, nkv);
    const int G = nh / nkv;
    CUtensorMap mq, mkv;
    {
        cuuint64_t dims[3] = {(cuuint64_t)HD, (cuuint64_t)nh, (cuuint64_t)T};
        cuuint64_t strides[2] = {(cuuint64_t)HD * 2, (cuuint64_t)nh * HD * 2};
        cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)(128 / G)};
        cuuint32_t es[3] = {1, 1, 1};
        AP_REQUIRE(t8_encode_fn()(&mq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, es,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
                   "attention_kv8 (tcgen05): cannot encode the query tensor map");
    }
    {
        cuuint64_t dims[2] = {(cuuint64_t)HD, (cuuint64_t)dense_rows};
        cuuint64_t strides[1] = {(cuuint64_t)HD * 2};
        cuuint32_t box[2] = {64, BKV};
        cuuint32_t es[2] = {1, 1};
        AP_REQUIRE(t8_encode_fn()(&mkv, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, scratch, dims, strides, box, es,
                                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS,
                   "attention_kv8 (tcgen05): cannot encode the tensor map of keys and values");
    }
    static bool configured[64];
    int dev = 0;
    AP_REQUIRE(cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64, "attention_kv8: cannot tell the current device");
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(attention_kv8_tcgen05_kernel<false, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, T8Smem<1>::kTotal);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attention_kv8_tcgen05_kernel<true, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, T8Smem<1>::kTotal);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attention_kv8_tcgen05_kernel<false, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, T8Smem<2>::kTotal);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(attention_kv8_tcgen05_kernel<true, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, T8Smem<2>::kTotal);
        AP_REQUIRE(e == cudaSuccess, "attention_kv8 (tcgen05): cannot reserve %d bytes of shared memory: %s", T8Smem<2>::kTotal,
                   cudaGetErrorString(e));
        configured[dev] = true;
    }
    AttnT8Params p;
    p.cache = (const uint8_t*)cache; p.page_bytes = (size_t)page_bytes; p.spoiled = (int*)((bf16*)scratch + (size_t)dense_rows * HD);
    p.out = (bf16*)out; p.block_table = block_table; p.seq_start = seq_start; p.positions = positions;
    p.tiles = tiles; p.num_pages = (int)num_pages; p.max_blocks = max_blocks; p.nseq = nseq; p.nh = nh; p.nkv = nkv;
    p.P = P; p.window = window; p.group = G; p.tokens_per_tile = 128 / G; p.nsplit = nsplit;
    p.scale_log2 = scale * LOG2E_F;
    AP_REQUIRE((long long)total_ctas * nkv < (1LL << 31), "attention_kv8 (tcgen05): too many CTAs for the grid");
    AP_CHECK_PDL_LAUNCH("kv8_widen", ap_launch_pdl(kv8_widen_kernel, dim3((unsigned)tiles, 2 * nkv, nseq), dim3(T8_WIDEN_THREADS), 0, stream, p, (bf16*)scratch));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(total_ctas * nkv), nsplit);
    cfg.blockDim = dim3(T8_THREADS(query_tiles));
    cfg.dynamicSmemBytes = query_tiles == 1 ? T8Smem<1>::kTotal : T8Smem<2>::kTotal;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = ap_pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1;
    attr[1].val.clusterDim.y = nsplit;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = nsplit > 1 ? 2 : 1;
    AP_CHECK_PDL_LAUNCH("attention_kv8_tcgen05",
                        query_tiles == 1 ? (nsplit > 1 ? cudaLaunchKernelEx(&cfg, attention_kv8_tcgen05_kernel<true, 1>, mq, mkv, p)
                                                       : cudaLaunchKernelEx(&cfg, attention_kv8_tcgen05_kernel<false, 1>, mq, mkv, p))
                                         : (nsplit > 1 ? cudaLaunchKernelEx(&cfg, attention_kv8_tcgen05_kernel<true, 2>, mq, mkv, p)
                                                       : cudaLaunchKernelEx(&cfg, attention_kv8_tcgen05_kernel<false, 2>, mq, mkv, p)));
    return AP_OK;
}

AP_EXPORT int ap_attention_kv8_tcgen05_status(void) {
    int v = -1;
    if (cudaMemcpyFromSymbol(&v, g_t8_status, sizeof(int)) != cudaSuccess) return -1;
    return v;
}

#else   // head sizes this kernel is not built for

AP_EXPORT int ap_attention_kv8_tcgen05_takes(int, int, int, int) { return 0; }

#endif
