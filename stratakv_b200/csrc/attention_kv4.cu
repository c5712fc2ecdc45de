// Causal grouped-query attention of one or a few new tokens a sequence over a paged cache held in 4 bits (kv4.cuh).
//
// The mathematics is that of attention_decode.cu: scores (q.k) * scale over the sequence's visible positions, a softmax whose maximum
// and sum run along with one pass over the keys, and the weighted sum of values, in float.  The products take half precision,
// in which what the cache holds is exact: a query head is brought to a largest magnitude between 2^15 and 2^16 by a power of two (a half
// ends at 65,504, a bfloat16 below 2^16 at 65,280), so that its numbers down to 2^-32 of the largest keep their 8 bits and smaller ones are
// off by 2^-40 of it at most; and the probabilities keep 11 bits.
//
// An item is a key head of a sequence and up to 8 NT rows (a row: a query head of one new token; the heads that share a key head lie side by side); a warp
// takes 32 keys of it at a time (16 where a cache block is no multiple of 32), which asynchronous copies have brought to its own part of shared memory.
// Both products are turned so that the keys are the rows of mma.sync m16n8k16: S^T = K Q^T, O^T = V^T P^T.  Eight rows
// then fill an instruction, and a lane has eight keys' or values' numbers for each instead of four.  Which number of
// a head is which index of the sum is free as long as both operands agree: lane t of four has a quarter of a key's numbers, one after
// the other, so it reads its codes in one piece and one scale byte serves sixteen of them.  For the second product a lane has
// a run of numbers of four keys; the bytes of two keys are put side by side ahead of the unpacking, which then yields the pairs of keys
// that the instruction wants.  P goes from one product to the other by movmatrix.
//
// Over many positions it is bound by issue: a chunk of 32 keys of a head of 128 is 688 instructions of a warp, 352 of them unpacking (11 for eight codes),
// and takes 1,000 cycles of a scheduler.  64 sequences of 4,096 positions, 32 heads over 8 of 128, 73 us, 4.1 TB/s of codes and scales; copies alone
// 58, all but the copies 60.  (Loads by each lane 130 us; copies through shared memory, 16 keys at a time 101; 32 keys, packed float arithmetic, masks only
// where a row needs them 83; one logic operation a code 74.  16 warps an SM at 128 registers: 18 to 20 spill, 97 to 106.)  On tcgen05 the unpacked codes
// would go through shared memory first; the products here are a quarter of the time at most.
// Over few positions it is a chain of latencies: lengths, block table, one or two chunks, and the sum over the warps.
#include "head_size.cuh"

#include "kv4.cuh"

#include <array>
#include <type_traits>

#if SKV_DTYPE == SKV_BF16

namespace skv {

constexpr int FHD = SKV_HEAD_DIM;
constexpr int FPAD = (FHD + 63) / 64 * 64;        // a lane has whole groups of 16 of a key, and whole words of a value
constexpr int KWORDS = FPAD / 32, VWORDS4 = FPAD / 64;      // words of eight codes a lane reads per key, per value
constexpr int KSTEP4 = FPAD / 16, OTILE4 = FPAD / 16;       // k16 steps of K Q^T; m16 tiles of V^T P^T
// Scale bytes of a lane's words of a value: one where they lie in one group, one for two words or one each.
constexpr int VGROUPS = FPAD == 192 ? 3 : FPAD == 256 ? 2 : 1, VWORDS_OF_GROUP = VWORDS4 / VGROUPS;
constexpr int KV4_WARPS = 8, KV4_SEQS = 1024;     // (sequences of a call)
// A warp's chunk of CK keys (32, or 16 where a cache block is no multiple of 32) on its way: codes of keys and values, then their scales.
constexpr int KROW = FHD / 2, SROW = FHD / 16, KV4_STAGES = FHD > 64 ? 2 : 3;
template <int CK> constexpr int CHUNK_OF = CK * 2 * (KROW + SROW);
template <int CK> constexpr int RING_OF = KV4_WARPS * KV4_STAGES * CHUNK_OF<CK>;

// Index i of the sums over keys is key (i >> 1) + 4 (i & 1) of its eight: the four lanes that read values of one index then read four
// neighbouring rows, which lie in different banks.  Keys are laid down in the order of the indices, where a row is whole pieces of 16
// bytes (head sizes that are multiples of 32; of others a piece has the end of one row and the start of the next).
constexpr bool KEYS_BY_INDEX = FHD % 32 == 0;
constexpr int KREAD = FHD == 128 ? 4 : 2;         // words of a key a lane reads at once
__device__ __forceinline__ int key_of_index(int i) { return (i & ~7) + ((i & 7) >> 1) + 4 * (i & 1); }
__device__ __forceinline__ int index_of_key(int k) { return (k & ~7) + 2 * (k & 3) + ((k & 7) >> 2); }
__device__ __forceinline__ void chunk_copy(uint32_t to, const uint8_t* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(from) : "memory");
}
// Where 16 bytes of a value's codes go (heads of 128: 64 bytes a row, of which two rows would share their banks).
__device__ __forceinline__ int value_piece(int row, int piece) { return FHD == 128 ? piece ^ (row & 2) : piece; }

__device__ __forceinline__ void mma_f16_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn_8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *(const uint32_t*)&v;
}
__device__ __forceinline__ float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// Probabilities are taken against a maximum that is raised when a score exceeds it by 2^8, and carry a factor 2^7: they stay
// below 2^15 (a half ends at 65,504), and one 2^-21 of the largest still has all its 11 bits.
constexpr float KV4_MARGIN = 8.0f, KV4_LIFT = 7.0f;

// The weight of a part whose maximum is m next to a common maximum: one that saw no finite score has sums of zero, or NaN if a
// NaN was among them, which must not get lost.
__device__ __forceinline__ float part_weight(float m, float top) { return m == -INFINITY ? 1.0f : kv4_exp2(m - top); }

// How a step's work is cut, in one of two ways (kv4_plan has the rule).  Either a cluster of one to eight blocks has an item and adds its warps' results
// up in shared memory: one launch.  Or the chunks of all items, one item behind the other, are dealt
// out to the warps in runs of equal length, whatever the sequences' lengths.  A run that begins or ends inside an item leaves a partial result, at most two a warp; an item that
// one run holds whole is finished by it.  (Runs of blocks, whose warps take chunks in turn and add up in shared memory: 64 x 4,096 positions 79.6 us
// against 73.9, 12 ragged sequences of 32 key heads 52.4 against 46.4.)
struct Kv4Cut {
    int n_seqs, num_heads, num_kv_heads, window, least;     // a run has at least `least` chunks
    int most_positions, most_new, most_tiles;               // what the call has room for: lengths beyond it are cut
    int group;                                              // query heads of a key head, and 2^32 / group, rounded up
    uint32_t group_magic;
    // x / group, as the upper half of a product (exact while x * group stays below 2^32)
    __device__ __forceinline__ int of_group(int x) const { return group == 1 ? x : (int)__umulhi((uint32_t)x, group_magic); }
};
struct Kv4Share {
    int q_begin, q_len, ctx, tiles, first_chunk, chunks;    // chunks of an item
    __device__ __forceinline__ int all(const Kv4Cut& cut) const { return chunks * cut.num_kv_heads * tiles; }
};
template <int ROWS, int CK>
__device__ __forceinline__ Kv4Share kv4_share(const Kv4Cut& cut, const int* cu_q, const int* ctx_after, int seq) {
    Kv4Share s = {};
    if (seq >= cut.n_seqs) return s;
    s.q_begin = cu_q[seq];
    s.q_len = min(cu_q[seq + 1] - s.q_begin, cut.most_new);
    s.ctx = max(0, min(ctx_after[seq], cut.most_positions));
    s.tiles = (s.q_len * cut.group + ROWS - 1) / ROWS;
    s.first_chunk = cut.window > 0 ? max(0, s.ctx - s.q_len - cut.window + 1) / CK : 0;
    s.chunks = s.q_len > 0 ? (s.ctx + CK - 1) / CK - s.first_chunk : 0;
    return s;
}

// Bytes that the partial results of a block's warps take, and behind them those of the block.
template <int NT> constexpr int ITEM_OF = (KV4_WARPS + 1) * NT * (OTILE4 * 512 + 64);
template <int NT, int CK, bool ITEM> constexpr int KV4_SMEM = ITEM && ITEM_OF<NT> > RING_OF<CK> ? ITEM_OF<NT> : RING_OF<CK>;

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;\n" ::: "memory");
}
// The same place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ float4 of_block(uint32_t at, int rank) {
    float4 v;
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %4, %5;\n ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at), "r"(rank) : "memory");
    return v;
}

// `parts` partial results of a tile of 16 numbers, brought to their common maximum and added up in their order.
template <class Load>
__device__ __forceinline__ void kv4_add_up(int parts, const Load& load, float4& acc, float4& ml) {
    constexpr int AHEAD = 8;
    acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    ml = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
    for (int p0 = 0; p0 < parts; p0 += AHEAD) {
        float4 o[AHEAD], of[AHEAD];                   // (maximum and sum of rows 2t and 2t + 1)
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            o[u] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            of[u] = make_float4(-INFINITY, 0.0f, -INFINITY, 0.0f);
            if (p0 + u < parts) load(p0 + u, o[u], of[u]);
        }
        float2 now = make_float2(ml.x, ml.z);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) now = make_float2(fmaxf(now.x, of[u].x), fmaxf(now.y, of[u].z));
        const float2 by = make_float2(part_weight(ml.x, now.x), part_weight(ml.z, now.y));
        acc = make_float4(acc.x * by.x, acc.y * by.y, acc.z * by.x, acc.w * by.y);
        ml = make_float4(now.x, ml.y * by.x, now.y, ml.w * by.y);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const float a = part_weight(of[u].x, now.x), b = part_weight(of[u].z, now.y);
            acc = make_float4(acc.x + o[u].x * a, acc.y + o[u].y * b, acc.z + o[u].z * a, acc.w + o[u].w * b);
            ml.y += of[u].y * a;
            ml.w += of[u].w * b;
        }
    }
}

// ITEM: a cluster of blocks has one item, whose chunks its warps share out and whose partial results it adds up itself.
template <int NT, int CK, bool ITEM>
__global__ void __launch_bounds__(KV4_WARPS * 32, NT == 1 && FHD <= 128 ? 2 : 1)
kv4_attention_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes,
                     const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale, const int* __restrict__ block_table,
                     int table_width, const int* __restrict__ cu_q, const int* __restrict__ ctx_after, __nv_bfloat16* __restrict__ out,
                     float4* __restrict__ partial_o, float2* __restrict__ partial_ml, const Kv4Cut cut, int block_size, float scale,
                     uint32_t chunks_magic, uint32_t ones, int cluster) {
    extern __shared__ __align__(16) uint8_t kv4_smem[];
    __shared__ int upto_all[ITEM ? 1 : KV4_SEQS], warp_all[KV4_WARPS];
    constexpr int ROWS = 8 * NT;
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int num_heads = cut.num_heads, num_kv_heads = cut.num_kv_heads, window = cut.window, group = cut.group;
    int total = 0;
    // upto[s]: the chunks up to and with sequence s.  Up to 32 sequences every warp adds up by itself, which needs no barrier.
    const bool few = cut.n_seqs <= 32;
    const int* upto = few ? upto_all + 32 * warp : upto_all;
    for (int s0 = 0; !ITEM && s0 < cut.n_seqs; s0 += KV4_WARPS * 32) {
        int sum = kv4_share<ROWS, CK>(cut, cu_q, ctx_after, s0 + (few ? lane : (int)threadIdx.x)).all(cut);
#pragma unroll
        for (int o2 = 1; o2 < 32; o2 *= 2) {
            const int before = __shfl_up_sync(0xffffffffu, sum, o2);
            if (lane >= o2) sum += before;
        }
        if (few) {
            upto_all[32 * warp + lane] = sum;
            total = __shfl_sync(0xffffffffu, sum, 31);
            __syncwarp();
            break;
        }
        if (lane == 31) warp_all[warp] = sum;
        __syncthreads();
        for (int w = 0; w < KV4_WARPS; ++w) {
            const int v = warp_all[w];
            if (w < warp) sum += v;
        }
        if (s0 + threadIdx.x < cut.n_seqs) upto_all[s0 + threadIdx.x] = total + sum;
        __syncthreads();
        total = upto_all[min(s0 + KV4_WARPS * 32, cut.n_seqs) - 1];
    }
    const int workers = (int)gridDim.x * KV4_WARPS, run = max(cut.least, (total + workers - 1) / workers);
    const int worker = blockIdx.x + gridDim.x * warp;       // (runs that follow each other lie on different SMs)
    const long long run_begin = (long long)worker * run;
    if (!ITEM && run_begin >= total) return;
    const int run_end = ITEM ? 1 : (int)min((long long)total, run_begin + run);
    int seq = 0;                                            // the first whose chunks reach beyond run_begin
    for (int step = few ? 16 : KV4_SEQS / 2; !ITEM && step > 0; step /= 2)
        if (seq + step <= cut.n_seqs && upto[seq + step - 1] <= (int)run_begin) seq += step;

    for (int done = ITEM ? 0 : (int)run_begin; done < run_end;) {
    const int of_cluster = ITEM ? blockIdx.x / cluster : 0, rank = blockIdx.x - of_cluster * cluster, items = num_kv_heads * cut.most_tiles;
    if (ITEM) seq = of_cluster / items;
    else
        while (upto[seq] <= done) ++seq;                    // (sequences without tokens have no chunks)
    const Kv4Share share = kv4_share<ROWS, CK>(cut, cu_q, ctx_after, seq);
    const int q_begin = share.q_begin, q_len = share.q_len, tiles = share.tiles;
    const int in_seq = ITEM ? 0 : done - (seq ? upto[seq - 1] : 0), item = ITEM ? of_cluster - seq * items : in_seq / share.chunks;
    const int kv_head = item / (ITEM ? cut.most_tiles : tiles), at_tile = item - kv_head * (ITEM ? cut.most_tiles : tiles);
    // (ITEM: a tile behind the sequence's last has no chunks)
    const int mine = ITEM && at_tile < tiles ? (share.chunks + cluster * KV4_WARPS - 1) / (cluster * KV4_WARPS) : 0;
    const int from = ITEM ? (rank * KV4_WARPS + warp) * mine : in_seq - item * share.chunks;
    const int count = ITEM ? max(0, min(mine, share.chunks - from)) : min(run_end - done, share.chunks - from);
    const bool whole = !ITEM && count == share.chunks;
    const size_t slot = (size_t)2 * worker + (done != (int)run_begin);
    done += ITEM ? 1 : count;
    const int row0 = at_tile * ROWS, rows = q_len * group, before = share.ctx - q_len;
    const int last_query = min(rows, row0 + ROWS) - 1;
    const int end = before + cut.of_group(last_query) + 1;                        // keys that any row of the tile sees lie before it
    const int my_first = share.first_chunk + from, my_end = min(my_first + count, (end + CK - 1) / CK);
    const int* table = block_table + (size_t)seq * table_width;

    // Queries on their way: lane (g, t) has a quarter of row g of each tile of eight.
    uint4 raw[NT][KWORDS];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = row0 + 8 * n + g, token = cut.of_group(min(r, rows - 1));
        const __nv_bfloat16* at = q + ((size_t)(q_begin + token) * num_heads + kv_head * group + min(r, rows - 1) - token * group) * FHD;
#pragma unroll
        for (int j = 0; j < KWORDS; ++j) {
            const int d = t * (FPAD / 4) + 8 * j;
            raw[n][j] = r < rows && d < FHD ? *(const uint4*)(at + d) : make_uint4(0u, 0u, 0u, 0u);
        }
    }

    // Copies of a chunk: pieces of 16 bytes, a lane one after the other.
    constexpr int CHUNK_BYTES = CHUNK_OF<CK>, PIECES = FHD % 32 ? 1 : FHD / 32;      // (of a row)
    const uint32_t ring = smem_u32(kv4_smem) + (uint32_t)(warp * KV4_STAGES * CHUNK_BYTES);
    const uint32_t block_bytes = (uint32_t)num_kv_heads * block_size * KROW;
    const uint8_t* k_from = k_codes + (size_t)kv_head * block_size * KROW + 16 * lane;
    const uint8_t* v_from = v_codes + (size_t)kv_head * block_size * KROW + 16 * lane;
    constexpr int SCALE_PIECES = CK * SROW / 16;
    const uint8_t* s_from = (lane < SCALE_PIECES || SCALE_PIECES > 16 ? k_scale + 16 * lane : v_scale + 16 * (lane - SCALE_PIECES)) + (size_t)kv_head * block_size * SROW;
    const uint32_t k_to = KEYS_BY_INDEX ? index_of_key(lane / PIECES) * KROW + 16 * (lane % PIECES) : 16 * lane;
    const uint32_t v_to = CK * KROW + (KEYS_BY_INDEX ? lane / PIECES * KROW + 16 * value_piece(lane / PIECES, lane % PIECES) : 16 * lane);
    auto block_of = [&](int chunk) { return chunks_magic ? (int)__umulhi((uint32_t)chunk, chunks_magic) : chunk; };
    auto fetch = [&](int chunk, int block, uint32_t to) {
        const uint32_t inside = (uint32_t)(chunk * CK - block_of(chunk) * block_size);
        const uint8_t* kc = k_from + ((size_t)(uint32_t)block * block_bytes + inside * KROW);
        const uint8_t* vc = v_from + ((size_t)(uint32_t)block * block_bytes + inside * KROW);
        const uint8_t* sc = s_from + ((size_t)(uint32_t)block * (block_bytes / 8) + inside * SROW);
#pragma unroll
        for (int u = 0; u < CK * KROW / 16; u += 32) {
            if (CK * KROW / 16 % 32 && u + lane >= CK * KROW / 16) break;
            if (!KEYS_BY_INDEX || (32 % PIECES == 0 && 32 / PIECES % 8 == 0)) {
                chunk_copy(to + k_to + 16 * u, kc + 16 * u);         // (whole groups of eight keys further)
                chunk_copy(to + v_to + 16 * u, vc + 16 * u);
            } else {
                const int key = (u + lane) / PIECES, piece = u + lane - key * PIECES;
                chunk_copy(to + index_of_key(key) * KROW + 16 * piece, kc + 16 * u);
                chunk_copy(to + CK * KROW + key * KROW + 16 * piece, vc + 16 * u);
            }
        }
        const uint32_t scales_to = to + 2 * CK * KROW + 16 * lane;
        if (SCALE_PIECES <= 16) {                     // both sorts at once
            if (lane < 2 * SCALE_PIECES) chunk_copy(scales_to, sc);
        } else if (lane < SCALE_PIECES) {
            chunk_copy(scales_to, sc);
            chunk_copy(scales_to + CK * SROW, v_scale + (sc - k_scale));
        }
    };

    int ahead = my_first;                             // the chunk that is fetched next, and its block
    auto entry = [&](int chunk) { return chunk < my_end ? table[block_of(chunk)] : 0; };
    int block = entry(ahead);
#pragma unroll
    for (int st = 0; st < KV4_STAGES - 1; ++st) {
        const int following = entry(ahead + 1);
        if (ahead < my_end) fetch(ahead, block, ring + st * CHUNK_BYTES);
        ring_commit();
        ++ahead;
        block = following;
    }

    // Queries as halves: word j's codes p and p + 4 meet numbers 8j + p and 8j + p + 4.
    uint32_t qb[NT][KSTEP4][2];
    float2 factor[NT];                                // of rows 2t and 2t + 1: scale * log2 e * the power of two taken off the query
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float most = 0.0f;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < KWORDS; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = (&raw[n][j].x)[e];
                const float a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
                most = fmaxf(most, fmaxf(fabsf(a), fabsf(b)));
                finite = finite && isfinite(a) && isfinite(b);
            }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        finite = (__ballot_sync(0xffffffffu, finite) >> (lane & 28) & 15u) == 15u;
        // most = 2^(power + 15) (1 + ...); what is not finite stays so in a half
        const int power = most > 0.0f && finite ? max((int)(__float_as_uint(most) >> 23) - 127 - 15, -115) : 0;          // (at most 112)
        const float down = __uint_as_float((uint32_t)(127 - power) << 23);
#pragma unroll
        for (int j = 0; j < KWORDS; ++j) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = (&raw[n][j].x)[e];
                x[2 * e] = __uint_as_float(w << 16) * down;
                x[2 * e + 1] = __uint_as_float(w & 0xffff0000u) * down;
            }
            qb[n][2 * j][0] = pack_half(x[0], x[4]); qb[n][2 * j][1] = pack_half(x[1], x[5]);
            qb[n][2 * j + 1][0] = pack_half(x[2], x[6]); qb[n][2 * j + 1][1] = pack_half(x[3], x[7]);
        }
        const float up = scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + power) << 23);
        factor[n] = make_float2(__shfl_sync(0xffffffffu, up, 8 * t), __shfl_sync(0xffffffffu, up, 8 * t + 4));
    }

    float o[OTILE4][NT][4];
#pragma unroll
    for (int j = 0; j < OTILE4; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
    float2 lift[NT], sum[NT];                         // KV4_LIFT less the maximum in use of rows 2t and 2t + 1; their sums
#pragma unroll
    for (int n = 0; n < NT; ++n) { lift[n] = make_float2(INFINITY, INFINITY); sum[n] = make_float2(0.0f, 0.0f); }

    // One chunk.  MASKED: some row of the block does not see all of its keys.
    const uint32_t k_lane = (KEYS_BY_INDEX ? g : key_of_index(g)) * KROW + t * (FPAD / 8);
    const uint32_t ks_lane = 2 * CK * KROW + key_of_index(g) * SROW + t * (FPAD / 64), vs_lane = 2 * CK * KROW + CK * SROW + t * SROW;
    auto attend = [&](auto masked_, int j0, const uint8_t* tile) {
        constexpr bool MASKED = decltype(masked_)::value;
        constexpr int HALVES = CK / 16;
        int position[NT][2];                          // where rows 2t and 2t + 1 sit (-1: no such row)
        if (MASKED) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int r = row0 + 8 * n + 2 * t + c;
                    position[n][c] = r < rows ? before + cut.of_group(r) : -1;
                }
        }
        // S^T: keys of indices g, g + 8 by rows 2t, 2t + 1
        float s[HALVES][NT][4];
        uint32_t kw[HALVES][2][KWORDS];
#pragma unroll
        for (int h16 = 0; h16 < HALVES; ++h16) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[h16][n][c] = 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < KWORDS; j += KREAD) {
                    const bool there = FHD == FPAD || t * (FPAD / 4) + 8 * j < FHD;
                    const uint8_t* from = tile + k_lane + (16 * h16 + 8 * i) * KROW + 4 * j;
                    if (KREAD == 4) {
                        const uint4 w = *(const uint4*)from;
                        kw[h16][i][j] = w.x; kw[h16][i][j + 1] = w.y; kw[h16][i][j + 2] = w.z; kw[h16][i][j + KREAD - 1] = w.w;
                    } else {
                        const uint2 w = there ? *(const uint2*)from : make_uint2(0u, 0u);
                        kw[h16][i][j] = w.x; kw[h16][i][j + 1] = w.y;
                    }
                }
        }
#pragma unroll
        for (int h16 = 0; h16 < HALVES; ++h16)
#pragma unroll
            for (int j = 0; j < KWORDS; j += 2) {
                const bool there = FHD == FPAD || t * (FPAD / 4) + 8 * j < FHD;
                Kv4Scale of[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    of[i] = kv4_pair_of_scales((there ? (uint32_t)tile[ks_lane + (16 * h16 + 8 * i) * SROW + j / 2] : 0u) * 0x00800080u);
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    uint32_t a[2][4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) kv4_unpack(kw[h16][i][j + w], of[i], ones, a[i]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_f16_16816(s[h16][n], a[0][0], a[1][0], a[0][1], a[1][1], qb[n][2 * (j + w)][0], qb[n][2 * (j + w)][1]);
                        mma_f16_16816(s[h16][n], a[0][2], a[1][2], a[0][3], a[1][3], qb[n][2 * (j + w) + 1][0], qb[n][2 * (j + w) + 1][1]);
                    }
                }
            }
        auto sees = [&](int h16, int n, int c) {
            const int key = j0 + 16 * h16 + key_of_index(g) + 8 * (c >> 1), pos = position[n][c & 1];
            return key <= pos && (window == 0 || key > pos - window);
        };
        // Scores in units of log2, above the maximum in use and with its lift.  (Nothing seen before: +infinity, which raises it.)
        float y[HALVES][NT][4];
        auto place = [&] {
#pragma unroll
            for (int h16 = 0; h16 < HALVES; ++h16)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; c += 2) {
                        const float2 v = fma2(make_float2(s[h16][n][c], s[h16][n][c + 1]), factor[n], lift[n]);
                        y[h16][n][c] = !MASKED || sees(h16, n, c) ? v.x : -INFINITY;
                        y[h16][n][c + 1] = !MASKED || sees(h16, n, c + 1) ? v.y : -INFINITY;
                    }
        };
        place();
        float top = -INFINITY;
#pragma unroll
        for (int h16 = 0; h16 < HALVES; ++h16)
#pragma unroll
            for (int n = 0; n < NT; ++n) top = max3(max3(top, y[h16][n][0], y[h16][n][1]), y[h16][n][2], y[h16][n][3]);
        if (__any_sync(0xffffffffu, top > KV4_MARGIN + KV4_LIFT)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float by[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float f = c ? factor[n].y : factor[n].x;
                    float m = -INFINITY;
#pragma unroll
                    for (int h16 = 0; h16 < HALVES; ++h16)
#pragma unroll
                        for (int i = 0; i < 4; i += 2) m = fmaxf(m, !MASKED || sees(h16, n, c + i) ? s[h16][n][c + i] * f : -INFINITY);
#pragma unroll
                    for (int o2 = 4; o2 < 32; o2 *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o2));
                    const float was = c ? lift[n].y : lift[n].x, now = fminf(was, KV4_LIFT - m);
                    by[c] = now == was ? 1.0f : kv4_exp2(now - was);                 // (0 if nothing was seen before)
                    if (c) { lift[n].y = now; sum[n].y *= by[1]; } else { lift[n].x = now; sum[n].x *= by[0]; }
                }
#pragma unroll
                for (int j = 0; j < OTILE4; ++j) { o[j][n][0] *= by[0]; o[j][n][1] *= by[1]; o[j][n][2] *= by[0]; o[j][n][3] *= by[1]; }
            }
            place();
        }
        uint32_t pb[HALVES][NT][2];
#pragma unroll
        for (int h16 = 0; h16 < HALVES; ++h16)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float p[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) p[c] = kv4_exp2(y[h16][n][c]);
                sum[n] = add2(sum[n], add2(make_float2(p[0], p[1]), make_float2(p[2], p[3])));
                pb[h16][n][0] = turn_8x8(pack_half(p[0], p[1]));
                pb[h16][n][1] = turn_8x8(pack_half(p[2], p[3]));
            }
#pragma unroll
        for (int h16 = 0; h16 < HALVES; ++h16) {
            // Scales of the values of indices 2t, 2t + 1, 2t + 8 and 2t + 9: keys t, t + 4, t + 8 and t + 12.
            uint32_t vs[4][VGROUPS], spoiled = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < VGROUPS; ++j) {
                    const int d = g * (FPAD / 8) + 8 * VWORDS_OF_GROUP * j;
                    vs[i][j] = FHD == FPAD || d < FHD ? tile[vs_lane + (16 * h16 + 4 * i) * SROW + d / 16] : 0u;
                    if (MASKED) {
                        // Rows behind the sequence hold what earlier users of the block left.  A NaN among the values reaches the rows that
                        // see its key alone: times a masked key's zero it would reach all.
                        if (j0 + 16 * h16 + t + 4 * i >= end) vs[i][j] = 0u;
                        if (vs[i][j] > KV4_LARGEST) { spoiled |= 1u << (4 * j + i); vs[i][j] = 0u; }
                    }
                }
            // O^T += V^T P^T
            uint32_t words[4][VWORDS4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t* from = tile + CK * KROW + (16 * h16 + t + 4 * i) * KROW;
#pragma unroll
                for (int j = 0; j < VWORDS4; ++j) {
                    const int d = g * (FPAD / 8) + 8 * j;
                    if (FHD == 128) {
                        if (j == 0) {                  // (both words lie in one piece of 16 bytes)
                            const uint2 w = *(const uint2*)(from + 16 * value_piece(t, g / 2) + 8 * (g & 1));
                            words[i][0] = w.x; words[i][VWORDS4 - 1] = w.y;
                        }
                    } else {
                        words[i][j] = FHD == FPAD || d < FHD ? *(const uint32_t*)(from + d / 2) : 0u;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < VWORDS4; ++j) {
                const int of = j / VWORDS_OF_GROUP;
                const Kv4Scale of01 = kv4_pair_of_scales(vs[1][of] * 0x00800000u + vs[0][of] * 0x80u);
                const Kv4Scale of89 = kv4_pair_of_scales(vs[3][of] * 0x00800000u + vs[2][of] * 0x80u);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t x[4], z[4];
                    kv4_unpack(__byte_perm(words[0][j], words[1][j], half ? 0x7632 : 0x5410), of01, ones, x);
                    kv4_unpack(__byte_perm(words[2][j], words[3][j], half ? 0x7632 : 0x5410), of89, ones, z);
#pragma unroll
                    for (int p = 0; p < 4; p += 2)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            mma_f16_16816(o[4 * j + 2 * half + p / 2][n], x[p], x[p + 1], z[p], z[p + 1], pb[h16][n][0], pb[h16][n][1]);
                }
            }
            if (MASKED && __any_sync(0xffffffffu, spoiled != 0u)) {
                // how many NaN a row sees in a group of numbers: a product of ones
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const uint32_t b0 = turn_8x8(pack_half(sees(h16, n, 0) ? 1.0f : 0.0f, sees(h16, n, 1) ? 1.0f : 0.0f));
                    const uint32_t b1 = turn_8x8(pack_half(sees(h16, n, 2) ? 1.0f : 0.0f, sees(h16, n, 3) ? 1.0f : 0.0f));
#pragma unroll
                    for (int j = 0; j < VGROUPS; ++j) {
                        const uint32_t bits = spoiled >> (4 * j);
                        const uint32_t a01 = pack_half(bits & 1u ? 1.0f : 0.0f, bits & 2u ? 1.0f : 0.0f);
                        const uint32_t a89 = pack_half(bits & 4u ? 1.0f : 0.0f, bits & 8u ? 1.0f : 0.0f);
                        float count[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma_f16_16816(count, a01, a01, a89, a89, b0, b1);
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            if (count[c] > 0.0f) {
#pragma unroll
                                for (int w = 0; w < 4 * VWORDS_OF_GROUP; ++w) o[4 * VWORDS_OF_GROUP * j + w][n][c] = NAN;
                            }
                    }
                }
            }
        }
    };

    // every row of the block sees keys all_from .. all_to - 1
    const int all_to = before + cut.of_group(row0) + 1, all_from = window > 0 ? max(0, before + cut.of_group(last_query) - window + 1) : 0;
    int stage = 0, free_stage = KV4_STAGES - 1;
    for (int at = my_first; at < my_end; ++at) {
        ring_wait<KV4_STAGES - 2>();
        __syncwarp();                                 // the chunk is here for all lanes, and all have left the one before
        const int following = entry(ahead + 1);
        if (ahead < my_end) fetch(ahead, block, ring + free_stage * CHUNK_BYTES);
        ring_commit();
        ++ahead;
        block = following;
        const int j0 = at * CK;
        const uint8_t* tile = kv4_smem + (warp * KV4_STAGES + stage) * CHUNK_BYTES;
        if (j0 + CK <= all_to && j0 >= all_from) attend(std::false_type{}, j0, tile);
        else attend(std::true_type{}, j0, tile);
        free_stage = stage;
        stage = stage + 1 == KV4_STAGES ? 0 : stage + 1;
    }
    ring_wait<0>();
    __syncwarp();                                     // (the next item's chunks go where these were)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int o2 = 4; o2 < 32; o2 *= 2) {
            sum[n].x += __shfl_xor_sync(0xffffffffu, sum[n].x, o2);
            sum[n].y += __shfl_xor_sync(0xffffffffu, sum[n].y, o2);
        }
    if (ITEM) {
        // Partial results as they lie in the registers, where the chunks were: a tile's 32 lanes of four numbers, then maxima and sums, a row each.
        constexpr int TILES = NT * OTILE4, OF_WARP = NT * (OTILE4 * 512 + 64);
        float4* parts_o = (float4*)kv4_smem;
        float4* parts_ml = (float4*)(kv4_smem + (KV4_WARPS + 1) * TILES * 512);
        static_assert(ITEM_OF<NT> == (KV4_WARPS + 1) * OF_WARP, "tiles, then maxima and sums");
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int j = 0; j < OTILE4; ++j)
                parts_o[(warp * TILES + n * OTILE4 + j) * 32 + lane] = make_float4(o[j][n][0], o[j][n][1], o[j][n][2], o[j][n][3]);
            if (g == 0) parts_ml[(warp * NT + n) * 4 + t] = make_float4(-lift[n].x, sum[n].x, -lift[n].y, sum[n].y);
        }
        __syncthreads();
        float4 acc[(TILES + KV4_WARPS - 1) / KV4_WARPS], ml[(TILES + KV4_WARPS - 1) / KV4_WARPS];
#pragma unroll
        for (int u = 0; u * KV4_WARPS < TILES; ++u) {
            const int tile = u * KV4_WARPS + warp, n = tile / OTILE4;
            if (tile >= TILES) continue;
            kv4_add_up(KV4_WARPS, [&](int p, float4& v, float4& of) { v = parts_o[(p * TILES + tile) * 32 + lane]; of = parts_ml[(p * NT + n) * 4 + t]; }, acc[u], ml[u]);
            if (cluster > 1) {
                parts_o[(KV4_WARPS * TILES + tile) * 32 + lane] = acc[u];
                if (g == 0 && tile % OTILE4 == 0) parts_ml[(KV4_WARPS * NT + n) * 4 + t] = ml[u];
            }
        }
        if (cluster > 1) cluster_barrier();           // (every block of a cluster comes here, and to the one below)
#pragma unroll
        for (int u = 0; u * KV4_WARPS < TILES; ++u) {
            const int tile = u * KV4_WARPS + warp, n = tile / OTILE4, j = tile - n * OTILE4;
            if (tile >= TILES || tile % cluster != rank) continue;
            if (cluster > 1)
                kv4_add_up(cluster, [&](int p, float4& v, float4& of) {
                    v = of_block(smem_u32(parts_o + (KV4_WARPS * TILES + tile) * 32 + lane), p);
                    of = of_block(smem_u32(parts_ml + (KV4_WARPS * NT + n) * 4 + t), p);
                }, acc[u], ml[u]);
            const int d = g * (FPAD / 8) + 2 * j;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = row0 + 8 * n + 2 * t + c;
                if (r >= rows || d >= FHD || share.chunks == 0) continue;
                const int token = cut.of_group(r);
                const float by = 1.0f / (c ? ml[u].w : ml[u].y);
                *(__nv_bfloat162*)(out + ((size_t)(q_begin + token) * num_heads + kv_head * group + r - token * group) * FHD + d) =
                    __floats2bfloat162_rn((c ? acc[u].y : acc[u].x) * by, (c ? acc[u].w : acc[u].z) * by);
            }
        }
        if (cluster > 1) cluster_barrier();           // (a block's shared memory lasts until all have read it)
        return;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (!whole) {
            // left as they lie in the registers: a lane's four numbers of a tile
#pragma unroll
            for (int j = 0; j < OTILE4; ++j)
                partial_o[((slot * NT + n) * OTILE4 + j) * 32 + lane] = make_float4(o[j][n][0], o[j][n][1], o[j][n][2], o[j][n][3]);
            if (g == 0) {
                partial_ml[slot * ROWS + 8 * n + 2 * t] = make_float2(-lift[n].x, sum[n].x);
                partial_ml[slot * ROWS + 8 * n + 2 * t + 1] = make_float2(-lift[n].y, sum[n].y);
            }
        } else {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = row0 + 8 * n + 2 * t + c;
                if (r >= rows) continue;
                const int token = cut.of_group(r);
                __nv_bfloat16* to = out + ((size_t)(q_begin + token) * num_heads + kv_head * group + r - token * group) * FHD;
                const float by = 1.0f / (c ? sum[n].y : sum[n].x);
#pragma unroll
                for (int j = 0; j < OTILE4; ++j) {
                    const int d = g * (FPAD / 8) + 2 * j;
                    if (d < FHD) *(__nv_bfloat162*)(to + d) = __floats2bfloat162_rn(o[j][n][c] * by, o[j][n][c + 2] * by);
                }
            }
        }
    }
    }
}

// The partial results of an item, brought to their common maximum and added up in their order: a warp has a tile of 16 numbers.  SPREAD: eight warps have
// it, partial results in turn, for few items of many (1 x 131,072 positions, 296 partial results an item, attention and merge 43 us, 71 without;
// 16 x 4,096 28 us, 33 with it).
template <int NT, int CK, bool SPREAD>
__global__ void __launch_bounds__(KV4_WARPS * 32)
kv4_merge_kernel(const float4* __restrict__ partial_o, const float4* __restrict__ partial_ml, const int* __restrict__ cu_q,
                 const int* __restrict__ ctx_after, __nv_bfloat16* __restrict__ out, const Kv4Cut cut, int workers) {
    constexpr int ROWS = 8 * NT;
    __shared__ float4 shared_o[KV4_WARPS][32], shared_ml[KV4_WARPS][32];
    __shared__ int sums[2][KV4_WARPS];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int of_seq = cut.num_kv_heads * cut.most_tiles, seq = blockIdx.x / of_seq, item = blockIdx.x - seq * of_seq;
    const int kv_head = item / cut.most_tiles, at_tile = item - kv_head * cut.most_tiles, group = cut.group;
    const Kv4Share share = kv4_share<ROWS, CK>(cut, cu_q, ctx_after, seq);
    int total = 0, base = 0;                          // chunks of all sequences, and of those before this one
    for (int s = threadIdx.x; s < cut.n_seqs; s += KV4_WARPS * 32) {
        const int all = kv4_share<ROWS, CK>(cut, cu_q, ctx_after, s).all(cut);
        total += all;
        if (s < seq) base += all;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    base = __reduce_add_sync(0xffffffffu, base);
    if (lane == 0) { sums[0][warp] = total; sums[1][warp] = base; }
    __syncthreads();
    if (at_tile >= share.tiles || share.chunks == 0) return;
    total = base = 0;
#pragma unroll
    for (int w = 0; w < KV4_WARPS; ++w) { total += sums[0][w]; base += sums[1][w]; }
    const int run = max(cut.least, (total + workers - 1) / workers);
    const int begin = base + (kv_head * share.tiles + at_tile) * share.chunks, first = begin / run, parts = (begin + share.chunks - 1) / run - first + 1;
    if (parts == 1) return;                           // finished by the warp that had it
    auto slot_of = [&](int p) { return (size_t)2 * (first + p) + (p == 0 && begin != first * run); };
    for (int tile = SPREAD ? blockIdx.y : blockIdx.y * KV4_WARPS + warp; tile < OTILE4 * NT; tile += SPREAD ? OTILE4 * NT : KV4_WARPS * (int)gridDim.y) {
        const int n = tile / OTILE4, j = tile - n * OTILE4;
        float4 acc, ml;
        const int own = SPREAD ? warp : 0, step = SPREAD ? KV4_WARPS : 1;
        kv4_add_up((parts - own + step - 1) / step, [&](int p, float4& v, float4& of) {
            const size_t at = slot_of(own + p * step);
            v = partial_o[((at * NT + n) * OTILE4 + j) * 32 + lane];
            of = partial_ml[at * (ROWS / 2) + 4 * n + t];
        }, acc, ml);
        if (SPREAD) {
            shared_o[warp][lane] = acc;
            shared_ml[warp][lane] = ml;
            __syncthreads();
            if (warp != 0) return;
            kv4_add_up(KV4_WARPS, [&](int p, float4& v, float4& of) { v = shared_o[p][lane]; of = shared_ml[p][lane]; }, acc, ml);
        }
        const int d = g * (FPAD / 8) + 2 * j;
        if (d >= FHD) continue;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = at_tile * ROWS + 8 * n + 2 * t + c;
            if (r >= share.q_len * group) continue;
            const int token = cut.of_group(r);
            const float by = 1.0f / (c ? ml.w : ml.y);
            *(__nv_bfloat162*)(out + ((size_t)(share.q_begin + token) * cut.num_heads + kv_head * group + r - token * group) * FHD + d) =
                __floats2bfloat162_rn((c ? acc.y : acc.x) * by, (c ? acc.w : acc.z) * by);
        }
    }
}

// Clusters of `size` blocks that fit the GPU at once, by variant of the kernel (0 where there is no GPU).
template <int NT, int CK>
static int fitting_clusters(int size) {
    if (reserve_shared_once<kv4_attention_kernel<NT, CK, true>>("skv_attention_kv4", KV4_SMEM<NT, CK, true>)) return 0;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(size);
    config.blockDim = dim3(KV4_WARPS * 32);
    config.dynamicSmemBytes = KV4_SMEM<NT, CK, true>;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = size;
    attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = 1;
    int count = 0;
    return cudaOccupancyMaxActiveClusters(&count, kv4_attention_kernel<NT, CK, true>, &config) == cudaSuccess ? count : 0;
}
static int most_clusters(int variant, int size) {
    static const std::array<std::array<int, 4>, 4> fit = [] {
        std::array<std::array<int, 4>, 4> of;
        for (int i = 0; i < 4; ++i)
            of[0][i] = fitting_clusters<1, 32>(1 << i), of[1][i] = fitting_clusters<1, 16>(1 << i), of[2][i] = fitting_clusters<2, 32>(1 << i),
            of[3][i] = fitting_clusters<2, 16>(1 << i);
        return of;
    }();
    return fit[variant][size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3];
}

// How a step of these sizes is cut: as many runs as warps fit the GPU, and how many partial results an item has at most.
struct Kv4Plan {
    Kv4Cut cut;
    int chunk, tiles_of_8, blocks, cluster;           // (cluster: blocks of an item, 0 where runs are dealt out)
    long long items, chunks, parts, floats;
};

static Kv4Plan kv4_plan(int n_seqs, int max_q_len, int table_width, int num_heads, int num_kv_heads, int block_size, int window, int sms) {
    Kv4Plan plan;
    const long long rows = (long long)max_q_len * (num_heads / num_kv_heads);
    plan.tiles_of_8 = rows > 8 ? 2 : 1;
    plan.chunk = block_size % 32 == 0 ? 32 : 16;
    const int row_tiles = (int)((rows + 8 * plan.tiles_of_8 - 1) / (8 * plan.tiles_of_8));
    const long long most = (long long)table_width * block_size;
    if (window >= most) window = 0;                   // (one that no position can leave: sums of it and a length could pass 32 bits)
    const long long span = window > 0 && (long long)window + max_q_len - 1 < most ? (long long)window + max_q_len - 1 : most;
    const long long chunks = span < most ? (span + plan.chunk - 2) / plan.chunk + 1 : most / plan.chunk;       // of an item
    plan.items = (long long)n_seqs * num_kv_heads * row_tiles;
    plan.chunks = plan.items * chunks;
    const long long resident = (long long)sms * (plan.tiles_of_8 == 1 && FHD <= 128 ? 2 : 1);
    constexpr int least = 1;                          // (at least 4: 1 x 300 positions 9.2 us against 7.2, 4 x 5 tokens over 4,000 19.0 against 17.5)
    const long long wanted = (plan.chunks + least - 1) / least;
    plan.blocks = (int)(wanted < resident ? wanted : resident);
    const long long workers = (long long)plan.blocks * KV4_WARPS, run = plan.chunks / workers > least ? plan.chunks / workers : least;
    const uint32_t group = (uint32_t)(num_heads / num_kv_heads);
    plan.cut = {n_seqs, num_heads, num_kv_heads, window, least, (int)most, max_q_len, row_tiles, (int)group, (uint32_t)((0x100000000ull + group - 1) / group)};
    // Runs, or clusters?  Counted in rounds, a chunk for every warp: a cluster's warps take as many as the longest item has chunks for them, and again
    // for every wave of clusters that the GPU takes at once; runs take the mean, but their partial results pass through memory to a second launch.
    // us, runs / clusters, heads of 128: 1 x 300 positions, 8 key heads (1 round / 1) 7.6 / 5.8; 1 x 8,000 (1 / 4) 12.3 / 10.0, 1 x 16,000 (2 / 8) 14.4 /
    // 15.5; 8 x 4,000 (4 / 4) 19.6 / 14.0; 64 x 300 (3 / 2 waves of 2) 18.3 / 13.6; 32 key heads 64 x 1,000 (28 / 7 waves of 4) 85 / 79, 64 x 150 (5 / 7 waves
    // of 1) 23.5 / 33.9.  Of ragged sequences a cluster waits for the longest: lengths that fall evenly from the longest to nothing 8 x 2,000, 32 key
    // heads (8 rounds) 19.4 / 19.8, 8 x 4,000 (16 rounds) 28.7 / 35.5, all as long as the longest 24.7 / 20.5 and 41.0 / 37.4; so at most 8 rounds.
    const int variant = 2 * (plan.tiles_of_8 - 1) + (plan.chunk == 16);
    // How many blocks: twice as many where each warp has more than one and a half chunks to lose (1 x 300 positions, 8 key heads of 128, one block 5.5, two
    // 5.8; 8 x 1,000, two 9.7, four 8.1), as long as they fit.  Where clusters of eight just fill the GPU a model's step gains or loses a little against four,
    // as its other kernels leave them room: a layer, 8 x 2,200, 4 key heads of 64 36.8 / 34.6; 4 x 2,200, 8 of 128 38.6 / 39.6; 1 x 3,000, 32 of 128
    // 40.5 / 42.0 (runs 36.9, 41.8, 44.2).
    plan.cluster = 1;
    while (plan.cluster < 8 && 2 * chunks > 3 * KV4_WARPS * plan.cluster && plan.items <= most_clusters(variant, 2 * plan.cluster)) plan.cluster *= 2;
    const long long rounds = (chunks + KV4_WARPS * plan.cluster - 1) / (KV4_WARPS * plan.cluster), at_once = most_clusters(variant, plan.cluster);
    const long long waves = at_once > 0 ? (plan.items + at_once - 1) / at_once : 1 << 30;
    const long long of_runs = (plan.chunks + workers - 1) / workers;
    if ((n_seqs > 1 && rounds > 8) || (waves == 1 ? rounds > of_runs + 3 : 4 * waves * (rounds + 1) > 5 * of_runs + 20)) plan.cluster = 0;
    plan.parts = chunks > 1 ? (chunks + run - 1) / run + 1 : 1;
    plan.floats = plan.parts > 1 && !plan.cluster ? 2 * workers * 8 * plan.tiles_of_8 * (FPAD + 2) : 0;
    return plan;
}

template <int NT, int CK>
static int kv4_launch(const Kv4Plan& plan, const void* q, const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale,
                      const int* block_table, int table_width, const int* cu_q, const int* ctx_after, void* out, float* scratch, int block_size,
                      float scale, cudaStream_t stream) {
    // a chunk's block is chunk / (block_size / CK): the upper half of a product, exact while chunks x chunks a block stay below 2^32
    const uint32_t chunks_magic = block_size == CK ? 0u : (uint32_t)((0x100000000ull + block_size / CK - 1) / (block_size / CK));
    const int workers = plan.blocks * KV4_WARPS;
    float* partial_ml = plan.floats ? scratch + (size_t)2 * workers * 8 * NT * FPAD : nullptr;
    auto start = [&](auto kernel, unsigned blocks, int smem) {
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(blocks);
        config.blockDim = dim3(KV4_WARPS * 32);
        config.dynamicSmemBytes = smem;
        config.stream = stream;
        cudaLaunchAttribute attributes[2];
        attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
        attributes[1].id = cudaLaunchAttributeClusterDimension;
        attributes[1].val.clusterDim.x = plan.cluster > 1 ? plan.cluster : 1;
        attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
        config.attrs = attributes;
        config.numAttrs = plan.cluster > 1 ? 2 : 1;
        const cudaError_t status = cudaLaunchKernelEx(&config, kernel, (const __nv_bfloat16*)q, (const uint8_t*)k_codes, (const uint8_t*)v_codes,
                                                      (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_table, table_width, cu_q, ctx_after,
                                                      (__nv_bfloat16*)out, (float4*)scratch, (float2*)partial_ml, plan.cut, block_size, scale,
                                                      chunks_magic, KV4_ONES, plan.cluster);
        return status == cudaSuccess ? 0 : fail("skv_attention_kv4", cudaGetErrorString(status));
    };
    if (plan.cluster) {
        if (int code = reserve_shared_once<kv4_attention_kernel<NT, CK, true>>("skv_attention_kv4", KV4_SMEM<NT, CK, true>)) return code;
        return start(kv4_attention_kernel<NT, CK, true>, (unsigned)(plan.items * plan.cluster), KV4_SMEM<NT, CK, true>);
    }
    if (int code = reserve_shared_once<kv4_attention_kernel<NT, CK, false>>("skv_attention_kv4", RING_OF<CK>)) return code;
    if (int code = start(kv4_attention_kernel<NT, CK, false>, plan.blocks, RING_OF<CK>)) return code;
    if (plan.floats == 0) return 0;
    const bool spread = plan.parts > 9 && plan.items * OTILE4 * NT <= 2 * sm_count();
    auto merge = spread ? kv4_merge_kernel<NT, CK, true> : kv4_merge_kernel<NT, CK, false>;
    return launch_pdl("skv_attention_kv4(merge)", merge, dim3((unsigned)plan.items, spread ? OTILE4 * NT : (OTILE4 * NT + KV4_WARPS - 1) / KV4_WARPS), dim3(KV4_WARPS * 32), 0, stream,
                      (const float4*)scratch, (const float4*)partial_ml, cu_q, ctx_after, (__nv_bfloat16*)out, plan.cut, workers);
}

}  // namespace skv

using namespace skv;

// Floats of scratch that a call of these sizes needs (0: none).
SKV_EXPORT long long skv_attention_kv4_scratch(int n_seqs, int max_q_len, int table_width, int num_heads, int num_kv_heads, int block_size,
                                               int window) {
    // (sizes that skv_attention_kv4 does nothing for, or refuses)
    if (n_seqs <= 0 || max_q_len <= 0 || table_width <= 0 || num_kv_heads <= 0 || num_heads <= 0 || num_heads % num_kv_heads != 0 || block_size <= 0 ||
        block_size % 16 != 0 || window < 0)
        return 0;
    return kv4_plan(n_seqs, max_q_len, table_width, num_heads, num_kv_heads, block_size, window, sm_count()).floats;
}

// Sequence s owns rows cu_q[s] .. cu_q[s+1]-1 of q and out ([tokens][heads][head_dim]), at most max_q_len; ctx_after[s] positions are cached, its own
// included, at most table_width blocks of them.
SKV_EXPORT int skv_attention_kv4(const void* q, const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale,
                                 const int* block_table, int table_width, const int* cu_q, const int* ctx_after, void* out, float* scratch,
                                 long long scratch_floats, int n_seqs, int max_q_len, int num_heads, int num_kv_heads, int head_dim,
                                 int block_size, float scale, int window, cudaStream_t stream) {
    if (n_seqs <= 0 || max_q_len <= 0 || table_width <= 0) return 0;
    if (n_seqs > KV4_SEQS) return fail("skv_attention_kv4", "at most 1,024 sequences in a call");
    if (head_dim != FHD) return fail("skv_attention_kv4", "this library was built for another head size");
    if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
        return fail("skv_attention_kv4", "heads must be a positive multiple of kv heads");
    if (block_size <= 0 || block_size % 16 != 0) return fail("skv_attention_kv4", "block_size must be a positive multiple of 16");
    if (window < 0) return fail("skv_attention_kv4", "a window must not be negative");
    if ((unsigned long long)num_kv_heads * block_size * FHD > 0x80000000ull) return fail("skv_attention_kv4", "a cache block is too large (2 GB at most)");
    if ((unsigned long long)table_width * (block_size / 16) * (block_size / 16) >= 0x100000000ull || (unsigned long long)table_width * block_size > 0x7fffff00ull)
        return fail("skv_attention_kv4", "the block table spans too many positions for blocks of this size");
    if (((uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scale | (uintptr_t)v_scale | (uintptr_t)out | (uintptr_t)scratch) & 15)
        return fail("skv_attention_kv4", "operands must be 16-byte aligned");
    if ((long long)n_seqs * max_q_len * num_heads > 0x3fffffffLL || (long long)(max_q_len + 16) * num_heads * (num_heads / num_kv_heads) > 0xffffffffLL) return fail("skv_attention_kv4", "too many rows in one step");
    const Kv4Plan plan = kv4_plan(n_seqs, max_q_len, table_width, num_heads, num_kv_heads, block_size, window, sm_count());
    if (plan.chunks > 0x7fffffffLL) return fail("skv_attention_kv4", "too many rows and positions in one step");
    if (plan.floats && (!scratch || scratch_floats < plan.floats)) return fail("skv_attention_kv4", "scratch is too small");
    auto launch = plan.tiles_of_8 == 2 ? (plan.chunk == 32 ? kv4_launch<2, 32> : kv4_launch<2, 16>) : plan.chunk == 32 ? kv4_launch<1, 32> : kv4_launch<1, 16>;
    return launch(plan, q, k_codes, v_codes, k_scale, v_scale, block_table, table_width, cu_q, ctx_after, out, scratch, block_size, scale, stream);
}

#else

SKV_EXPORT long long skv_attention_kv4_scratch(int, int, int, int, int, int, int) { return 0; }

SKV_EXPORT int skv_attention_kv4(const void*, const void*, const void*, const void*, const void*, const int*, int, const int*, const int*,
                                 void*, float*, long long, int, int, int, int, int, int, float, int, cudaStream_t) {
    return skv::fail("skv_attention_kv4", "a 4-bit cache is built for bfloat16");
}

#endif
