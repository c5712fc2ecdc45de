// Causal grouped-query attention of one or a few new tokens a sequence over a paged cache held in 4 bits (kv4.cuh).
//
// The mathematics is that of attention_decode.cu: scores (q.k) * scale over the sequence's visible positions, a softmax whose maximum
// and sum run along with one pass over the keys, and the weighted sum of values, in float.  The products take half precision,
// in which what the cache holds is exact: a query is brought to a largest magnitude between 1 and 2 by a power of two (its 8
// bits fit a half's 11), and the probabilities keep 11 bits.
//
// A block has up to 8 NT rows (a row: a query head of one new token; the heads that share a key head lie side by side), a warp 16 keys
// at a time.  Both products are turned so that the keys are the rows of mma.sync m16n8k16: S^T = K Q^T, O^T = V^T P^T.  Eight rows
// then fill an instruction, and a lane has eight keys' or values' numbers for each instead of four.  Which number of
// a head is which index of the sum is free as long as both operands agree: lane t of four has a quarter of a key's numbers, one after
// the other, so it reads its codes in one piece and one scale byte serves sixteen of them.  For the second product a lane has
// a run of numbers of four keys; the bytes of two keys are put side by side ahead of the unpacking, which then yields the pairs of keys
// that the instruction wants.  P goes from one product to the other by movmatrix.
#include "head_size.cuh"

#include "kv4.cuh"

#if SKV_DTYPE == SKV_BF16

namespace skv {

constexpr int FHD = SKV_HEAD_DIM;
constexpr int FPAD = (FHD + 63) / 64 * 64;        // a lane has whole groups of 16 of a key, and whole words of a value
constexpr int KWORDS = FPAD / 32, VWORDS4 = FPAD / 64;      // words of eight codes a lane reads per key, per value
constexpr int KSTEP4 = FPAD / 16, OTILE4 = FPAD / 16;       // k16 steps of K Q^T; m16 tiles of V^T P^T
// Scale bytes of a lane's words of a value: one where they lie in one group, one for two words or one each.
constexpr int VGROUPS = FPAD == 192 ? 3 : FPAD == 256 ? 2 : 1, VWORDS_OF_GROUP = VWORDS4 / VGROUPS;
constexpr int KV4_WARPS = 8;

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

// Probabilities are taken against a maximum that is raised when a score exceeds it by 2^8, and carry a factor 2^7: they stay
// below 2^15 (a half ends at 65,504), and one 2^-21 of the largest still has all its 11 bits.
constexpr float KV4_MARGIN = 8.0f, KV4_LIFT = 7.0f;

// The weight of a part whose maximum is m next to a common maximum: one that saw no finite score has sums of zero, or NaN if a
// NaN was among them, which must not get lost.
__device__ __forceinline__ float part_weight(float m, float top) { return m == -INFINITY ? 1.0f : kv4_exp2(m - top); }

template <int NT>
__global__ void __launch_bounds__(KV4_WARPS * 32)
kv4_attention_kernel(const __nv_bfloat16* __restrict__ q, const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes,
                     const uint8_t* __restrict__ k_scale, const uint8_t* __restrict__ v_scale, const int* __restrict__ block_table,
                     int table_width, const int* __restrict__ cu_q, const int* __restrict__ ctx_after, __nv_bfloat16* __restrict__ out,
                     float* __restrict__ partial_o, float* __restrict__ partial_ml, int num_heads, int num_kv_heads, int block_size,
                     float scale, int window, int splits, int row_tiles) {
    extern __shared__ float merge4[];                 // [warps][8 NT][FHD + 2]
    constexpr int ROWS = 8 * NT, PITCH = FHD + 2;
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int seq = blockIdx.x, kv_head = blockIdx.y / row_tiles, row0 = (blockIdx.y - kv_head * row_tiles) * ROWS, split = blockIdx.z;
    const int group = num_heads / num_kv_heads;
    const int q_begin = cu_q[seq], q_len = cu_q[seq + 1] - q_begin, rows = q_len * group;
    if (row0 >= rows) return;
    const int ctx = ctx_after[seq], before = ctx - q_len;
    const int last_query = min(rows, row0 + ROWS) - 1;
    const int end = before + last_query / group + 1;                        // keys that any row of the block sees: lo .. end - 1
    const int lo = window > 0 ? max(0, before + row0 / group - window + 1) : 0;
    const int first_group = lo >> 4, end_group = (end + 15) >> 4, per_split = (end_group - first_group + splits - 1) / splits;
    const int my_first = first_group + split * per_split, my_end = min(end_group, my_first + per_split);
    const int* table = block_table + (size_t)seq * table_width;

    // Queries: lane (g, t) has a quarter of row g of each tile of eight; word j's codes p and p + 4 meet numbers 8j + p and 8j + p + 4.
    uint32_t qb[NT][KSTEP4][2];
    float factor[NT][2];                              // of rows 2t and 2t + 1: scale * log2 e * the power of two taken off the query
    int position[NT][2];                              // and where they sit (-1: no such row)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = row0 + 8 * n + g;
        const __nv_bfloat16* at = q + ((size_t)(q_begin + min(r, rows - 1) / group) * num_heads + kv_head * group + min(r, rows - 1) % group) * FHD;
        uint4 raw[KWORDS];
        float most = 0.0f;
        bool finite = true;
#pragma unroll
        for (int j = 0; j < KWORDS; ++j) {
            const int d = t * (FPAD / 4) + 8 * j;
            raw[j] = r < rows && d < FHD ? *(const uint4*)(at + d) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = (&raw[j].x)[e];
                const float a = __uint_as_float(w << 16), b = __uint_as_float(w & 0xffff0000u);
                most = fmaxf(most, fmaxf(fabsf(a), fabsf(b)));
                finite = finite && isfinite(a) && isfinite(b);
            }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        finite = (__ballot_sync(0xffffffffu, finite) >> (lane & 28) & 15u) == 15u;
        // most = 2^power (1 + ...); what is not finite stays so in a half
        const int power = most > 0.0f && finite ? min(max((int)(__float_as_uint(most) >> 23) - 127, -100), 126) : 0;
        const float down = __uint_as_float((uint32_t)(127 - power) << 23);
#pragma unroll
        for (int j = 0; j < KWORDS; ++j) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t w = (&raw[j].x)[e];
                x[2 * e] = __uint_as_float(w << 16) * down;
                x[2 * e + 1] = __uint_as_float(w & 0xffff0000u) * down;
            }
            qb[n][2 * j][0] = pack_half(x[0], x[4]); qb[n][2 * j][1] = pack_half(x[1], x[5]);
            qb[n][2 * j + 1][0] = pack_half(x[2], x[6]); qb[n][2 * j + 1][1] = pack_half(x[3], x[7]);
        }
        const float up = scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + power) << 23);
        factor[n][0] = __shfl_sync(0xffffffffu, up, 8 * t);
        factor[n][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int of = row0 + 8 * n + 2 * t + c;
            position[n][c] = of < rows ? before + of / group : -1;
        }
    }

    float o[OTILE4][NT][4];
#pragma unroll
    for (int j = 0; j < OTILE4; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[j][n][0] = o[j][n][1] = o[j][n][2] = o[j][n][3] = 0.0f;
    float most[NT][2], sum[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) { most[n][0] = most[n][1] = -INFINITY; sum[n][0] = sum[n][1] = 0.0f; }

    for (int at = my_first + warp; at < my_end; at += KV4_WARPS) {
        const int j0 = at << 4;
        const size_t row = ((size_t)table[j0 / block_size] * num_kv_heads + kv_head) * block_size + j0 % block_size;
        const int live = min(16, ctx - j0);           // keys behind them hold what earlier users of the block left

        // codes and scales of keys g and g + 8, of values 2t, 2t + 1, 2t + 8 and 2t + 9
        uint32_t kw[2][KWORDS], ks[2][KWORDS / 2], vw[4][VWORDS4], vs[4][VGROUPS];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int key = g + 8 * i;
#pragma unroll
            for (int j = 0; j < KWORDS; j += 2) {
                const int d = t * (FPAD / 4) + 8 * j;
                const bool there = d < FHD && key < live;
                const uint2 w = there ? *(const uint2*)(k_codes + (row + key) * (FHD / 2) + d / 2) : make_uint2(0u, 0u);
                kw[i][j] = w.x; kw[i][j + 1] = w.y;
                ks[i][j / 2] = there ? k_scale[(row + key) * (FHD / 16) + d / 16] : 0u;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int key = 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
            for (int j = 0; j < VWORDS4; ++j) {
                const int d = g * (FPAD / 8) + 8 * j;
                const bool there = d < FHD && key < live;
                vw[i][j] = there ? *(const uint32_t*)(v_codes + (row + key) * (FHD / 2) + d / 2) : 0u;
                if (j % VWORDS_OF_GROUP == 0) vs[i][j / VWORDS_OF_GROUP] = there ? v_scale[(row + key) * (FHD / 16) + d / 16] : 0u;
            }
        }

        // S^T: keys g, g + 8 by rows 2t, 2t + 1
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
#pragma unroll
        for (int j = 0; j < KWORDS; ++j) {
            uint32_t a[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t h = ks[i][j / 2] * 0x00800080u, off = kv4_offset(h);
                kv4_spread(kw[i][j], a[i]);
#pragma unroll
                for (int p = 0; p < 4; ++p) a[i][p] = kv4_value(a[i][p], h, off);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                mma_f16_16816(s[n], a[0][0], a[1][0], a[0][1], a[1][1], qb[n][2 * j][0], qb[n][2 * j][1]);
                mma_f16_16816(s[n], a[0][2], a[1][2], a[0][3], a[1][3], qb[n][2 * j + 1][0], qb[n][2 * j + 1][1]);
            }
        }
        bool raise = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = j0 + g + 8 * (c >> 1), pos = position[n][c & 1];
                const bool seen = key <= pos && (window == 0 || key > pos - window);
                s[n][c] = seen ? s[n][c] * factor[n][c & 1] : -INFINITY;
                raise = raise || s[n][c] > most[n][c & 1] + KV4_MARGIN;
            }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float by[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = fmaxf(s[n][c], s[n][c + 2]);
#pragma unroll
                    for (int o2 = 4; o2 < 32; o2 *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o2));
                    m = fmaxf(m, most[n][c]);
                    by[c] = m == most[n][c] ? 1.0f : kv4_exp2(most[n][c] - m);       // (0 if nothing was seen before)
                    most[n][c] = m;
                    sum[n][c] *= by[c];
                }
#pragma unroll
                for (int j = 0; j < OTILE4; ++j) { o[j][n][0] *= by[0]; o[j][n][1] *= by[1]; o[j][n][2] *= by[0]; o[j][n][3] *= by[1]; }
            }
        }
        uint32_t pb[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float p[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float m = most[n][c & 1];
                p[c] = kv4_exp2(s[n][c] - (m == -INFINITY ? 0.0f : m) + KV4_LIFT);
                sum[n][c & 1] += p[c];
            }
            pb[n][0] = turn_8x8(pack_half(p[0], p[1]));
            pb[n][1] = turn_8x8(pack_half(p[2], p[3]));
        }
        // A NaN among the values reaches the rows that see its key alone: times a masked key's zero it would reach all.
        uint32_t spoiled = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < VGROUPS; ++j)
                if (vs[i][j] > KV4_LARGEST) { spoiled |= 1u << (4 * j + i); vs[i][j] = 0u; }
        // O^T += V^T P^T
#pragma unroll
        for (int j = 0; j < VWORDS4; ++j) {
            const int of = j / VWORDS_OF_GROUP;
            const uint32_t h01 = (vs[0][of] | vs[1][of] << 16) << 7, h89 = (vs[2][of] | vs[3][of] << 16) << 7;
            const uint32_t off01 = kv4_offset(h01), off89 = kv4_offset(h89);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t x[4], y[4];
                kv4_spread(__byte_perm(vw[0][j], vw[1][j], half ? 0x7632 : 0x5410), x);
                kv4_spread(__byte_perm(vw[2][j], vw[3][j], half ? 0x7632 : 0x5410), y);
#pragma unroll
                for (int p = 0; p < 4; ++p) { x[p] = kv4_value(x[p], h01, off01); y[p] = kv4_value(y[p], h89, off89); }
#pragma unroll
                for (int p = 0; p < 4; p += 2)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma_f16_16816(o[4 * j + 2 * half + p / 2][n], x[p], x[p + 1], y[p], y[p + 1], pb[n][0], pb[n][1]);
            }
        }
        if (__any_sync(0xffffffffu, spoiled != 0u)) {
            // how many NaN a row sees in a group of numbers: a product of ones
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float sees[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = j0 + g + 8 * (c >> 1), pos = position[n][c & 1];
                    sees[c] = key <= pos && (window == 0 || key > pos - window) ? 1.0f : 0.0f;
                }
                const uint32_t b0 = turn_8x8(pack_half(sees[0], sees[1])), b1 = turn_8x8(pack_half(sees[2], sees[3]));
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
    // merge the warps
    float* mine = merge4 + (size_t)warp * ROWS * PITCH;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int o2 = 4; o2 < 32; o2 *= 2) sum[n][c] += __shfl_xor_sync(0xffffffffu, sum[n][c], o2);
            float* to = mine + (8 * n + 2 * t + c) * PITCH;
#pragma unroll
            for (int j = 0; j < OTILE4; ++j) {
                const int d = g * (FPAD / 8) + 2 * j;
                if (d < FHD) *(float2*)(to + d) = make_float2(o[j][n][c], o[j][n][c + 2]);
            }
            if (g == 0) { to[FHD] = most[n][c]; to[FHD + 1] = sum[n][c]; }
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < ROWS * FHD; idx += blockDim.x) {
        const int r = idx / FHD, d = idx - r * FHD;
        if (row0 + r >= rows) break;
        float m = -INFINITY;
        for (int w = 0; w < KV4_WARPS; ++w) m = fmaxf(m, merge4[((size_t)w * ROWS + r) * PITCH + FHD]);
        float total = 0.0f, l = 0.0f;
        for (int w = 0; w < KV4_WARPS; ++w) {
            const float* from = merge4 + ((size_t)w * ROWS + r) * PITCH;
            const float weight = part_weight(from[FHD], m);
            total += weight * from[d];
            l += weight * from[FHD + 1];
        }
        const size_t item = (size_t)(q_begin + (row0 + r) / group) * num_heads + kv_head * group + (row0 + r) % group;
        if (splits == 1) {
            out[item * FHD + d] = __float2bfloat16_rn(total / l);
        } else {
            partial_o[(item * splits + split) * FHD + d] = total;
            if (d == 0) { partial_ml[2 * (item * splits + split)] = m; partial_ml[2 * (item * splits + split) + 1] = l; }
        }
    }
}

constexpr int KV4_COMBINE_THREADS = (FHD + 31) / 32 * 32;

__global__ void __launch_bounds__(KV4_COMBINE_THREADS)
kv4_combine_kernel(const float* __restrict__ partial_o, const float* __restrict__ partial_ml, const int* __restrict__ cu_q,
                   __nv_bfloat16* __restrict__ out, int n_seqs, int num_heads, int splits) {
    pdl_launch_dependents();
    pdl_wait();
    const size_t item = blockIdx.x;
    const int d = threadIdx.x;
    if (d >= FHD || blockIdx.x >= cu_q[n_seqs] * num_heads) return;     // (rows behind the last sequence stay as they are)
    const float* ml = partial_ml + 2 * item * splits;
    float m = -INFINITY, total = 0.0f, l = 0.0f;
    for (int s = 0; s < splits; ++s) m = fmaxf(m, ml[2 * s]);
    for (int s = 0; s < splits; ++s) {
        const float weight = part_weight(ml[2 * s], m);
        total += weight * partial_o[(item * splits + s) * FHD + d];
        l += weight * ml[2 * s + 1];
    }
    out[item * FHD + d] = __float2bfloat16_rn(total / l);
}

static int kv4_row_tiles(int max_q_len, int group) { return max_q_len * group > 8 ? (max_q_len * group + 15) / 16 : 1; }

// Pieces of each context: enough blocks to fill the GPU twice over, at least 128 keys a piece.  By sizes alone.
static int kv4_splits(int n_seqs, int max_q_len, int table_width, int num_heads, int num_kv_heads, int block_size, int window, int sms) {
    const long long most = (long long)table_width * block_size, keys = window > 0 && window + max_q_len < most ? window + max_q_len : most;
    const long long blocks = (long long)n_seqs * num_kv_heads * kv4_row_tiles(max_q_len, num_heads / num_kv_heads);
    const long long by_length = keys / 128, by_count = (2 * sms + blocks - 1) / blocks;
    long long splits = by_length < by_count ? by_length : by_count;
    return (int)(splits < 1 ? 1 : splits > 64 ? 64 : splits);
}

template <int NT>
static int kv4_launch(const void* q, const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const int* block_table,
                      int table_width, const int* cu_q, const int* ctx_after, void* out, float* scratch, int n_seqs, int n_tokens, int num_heads,
                      int num_kv_heads, int block_size, float scale, int window, int splits, int row_tiles, cudaStream_t stream) {
    const size_t smem = (size_t)KV4_WARPS * 8 * NT * (FHD + 2) * sizeof(float);
    if (int code = reserve_shared_once<kv4_attention_kernel<NT>>("skv_attention_kv4", smem)) return code;
    float* partial_o = scratch;
    float* partial_ml = scratch ? scratch + (size_t)n_tokens * num_heads * splits * FHD : nullptr;
    if (int code = launch_pdl("skv_attention_kv4", kv4_attention_kernel<NT>, dim3(n_seqs, num_kv_heads * row_tiles, splits), dim3(KV4_WARPS * 32), smem,
                              stream, (const __nv_bfloat16*)q, (const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint8_t*)k_scale,
                              (const uint8_t*)v_scale, block_table, table_width, cu_q, ctx_after, (__nv_bfloat16*)out, partial_o, partial_ml, num_heads,
                              num_kv_heads, block_size, scale, window, splits, row_tiles))
        return code;
    if (splits == 1) return 0;
    return launch_pdl("skv_attention_kv4(combine)", kv4_combine_kernel, dim3(n_tokens * num_heads), dim3(KV4_COMBINE_THREADS), 0, stream,
                      (const float*)partial_o, (const float*)partial_ml, cu_q, (__nv_bfloat16*)out, n_seqs, num_heads, splits);
}

}  // namespace skv

using namespace skv;

// Floats of scratch that a call of these sizes needs (0: none).
SKV_EXPORT long long skv_attention_kv4_scratch(int n_seqs, int n_tokens, int max_q_len, int table_width, int num_heads, int num_kv_heads,
                                               int block_size, int window) {
    if (n_seqs <= 0 || max_q_len <= 0 || num_kv_heads <= 0 || num_heads < num_kv_heads) return 0;
    const int splits = kv4_splits(n_seqs, max_q_len, table_width, num_heads, num_kv_heads, block_size, window, sm_count());
    return splits > 1 ? (long long)n_tokens * num_heads * splits * (FHD + 2) : 0;
}

// Sequence s owns rows cu_q[s] .. cu_q[s+1]-1 of q and out ([tokens][heads][head_dim]); ctx_after[s] positions are cached, its own included.
SKV_EXPORT int skv_attention_kv4(const void* q, const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale,
                                 const int* block_table, int table_width, const int* cu_q, const int* ctx_after, void* out, float* scratch,
                                 long long scratch_floats, int n_seqs, int n_tokens, int max_q_len, int num_heads, int num_kv_heads,
                                 int head_dim, int block_size, float scale, int window, cudaStream_t stream) {
    if (n_seqs <= 0 || n_tokens <= 0 || max_q_len <= 0) return 0;
    if (head_dim != FHD) return fail("skv_attention_kv4", "this library was built for another head size");
    if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
        return fail("skv_attention_kv4", "heads must be a positive multiple of kv heads");
    if (block_size <= 0 || block_size % 16 != 0) return fail("skv_attention_kv4", "block_size must be a positive multiple of 16");
    if (window < 0) return fail("skv_attention_kv4", "a window must not be negative");
    if (((uintptr_t)q | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)out) & 15)
        return fail("skv_attention_kv4", "operands must be 16-byte aligned");
    const int row_tiles = kv4_row_tiles(max_q_len, num_heads / num_kv_heads);
    if ((long long)num_kv_heads * row_tiles > 65535) return fail("skv_attention_kv4", "too many rows in one step (kv heads x tiles of 16 rows: 65,535 at most)");
    if ((long long)n_tokens * num_heads > 0x7fffffffLL) return fail("skv_attention_kv4", "too many rows in one step");
    const int splits = kv4_splits(n_seqs, max_q_len, table_width, num_heads, num_kv_heads, block_size, window, sm_count());
    if (splits > 1 && (!scratch || scratch_floats < (long long)n_tokens * num_heads * splits * (FHD + 2)))
        return fail("skv_attention_kv4", "scratch is too small");
    auto launch = max_q_len * (num_heads / num_kv_heads) > 8 ? kv4_launch<2> : kv4_launch<1>;
    return launch(q, k_codes, v_codes, k_scale, v_scale, block_table, table_width, cu_q, ctx_after, out, scratch, n_seqs, n_tokens, num_heads,
                  num_kv_heads, block_size, scale, window, splits, row_tiles, stream);
}

#else

SKV_EXPORT long long skv_attention_kv4_scratch(int, int, int, int, int, int, int, int) { return 0; }

SKV_EXPORT int skv_attention_kv4(const void*, const void*, const void*, const void*, const void*, const int*, int, const int*, const int*,
                                 void*, float*, long long, int, int, int, int, int, int, int, float, int, cudaStream_t) {
    return skv::fail("skv_attention_kv4", "a 4-bit cache is built for bfloat16");
}

#endif
