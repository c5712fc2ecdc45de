// Appending to a paged cache whose keys and values are held in 4 bits (kv4.cuh), and reading it back.
//
// The reference keeps its cache in full precision and appends a token with two device-to-device copies
// (src/models/transformer_block.cpp:484-509); it has no counterpart of these kernels.
#include "kv4.cuh"

#if SKV_DTYPE == SKV_BF16

namespace skv {

// A thread has four neighbouring numbers of a head of the float32 row [q | k | v]; four lanes have a group of 16.  Queries and keys are
// rotated (number i with number i + head_dim / 2; products and sum rounded one by one, so that a code never depends on how an
// expression was compiled), queries rounded to bfloat16, keys and values to codes.
constexpr int APPEND_THREADS = 256;

__global__ void __launch_bounds__(APPEND_THREADS)
kv4_append_kernel(const float* __restrict__ qkv, const float* __restrict__ cos_sin, const int* __restrict__ positions,
                  const int* __restrict__ token_seq, const int* __restrict__ block_table, int table_width,
                  __nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ v_codes,
                  uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v_scale, int num_heads, int num_kv_heads, int head_dim,
                  int block_size, int write_kv) {
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, quads = head_dim >> 2, half = head_dim >> 1;
    const int item = blockIdx.y * APPEND_THREADS + threadIdx.x;
    const int head = item / quads, d = (item - head * quads) << 2;
    const int all_heads = num_heads + (write_kv ? 2 * num_kv_heads : 0);
    if (head >= all_heads) return;                     // (whole groups: a head is a multiple of four quads)
    const int pos = positions[t];
    const float* x = qkv + (size_t)t * (num_heads + 2 * num_kv_heads) * head_dim + (size_t)head * head_dim;
    const float4 own = *(const float4*)(x + d);
    float v[4] = {own.x, own.y, own.z, own.w};
    if (cos_sin && head < num_heads + num_kv_heads) {
        const bool low = d < half;
        const float4 other = *(const float4*)(x + (low ? d + half : d - half));
        const float4* at = (const float4*)(cos_sin + (size_t)pos * head_dim + 2 * (low ? d : d - half));
        const float4 a = at[0], b = at[1];             // (cos, sin) of four pairs
        const float w[4] = {other.x, other.y, other.z, other.w}, c[4] = {a.x, a.z, b.x, b.z}, s[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = low ? __fsub_rn(__fmul_rn(v[i], c[i]), __fmul_rn(w[i], s[i])) : __fadd_rn(__fmul_rn(w[i], s[i]), __fmul_rn(v[i], c[i]));
    }
    if (head < num_heads) {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
        *(uint2*)(q_out + ((size_t)t * num_heads + head) * head_dim + d) = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&hi);
        return;
    }
    const bool value = head >= num_heads + num_kv_heads;
    const int kv_head = head - num_heads - (value ? num_kv_heads : 0);
    const int block = block_table[(size_t)token_seq[t] * table_width + pos / block_size];
    const size_t row = ((size_t)block * num_kv_heads + kv_head) * block_size + pos % block_size;
    const unsigned int mates = 0xFu << (threadIdx.x & 28);
    float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
    bool finite = isfinite(v[0]) && isfinite(v[1]) && isfinite(v[2]) && isfinite(v[3]);
    most = fmaxf(most, __shfl_xor_sync(mates, most, 1));
    most = fmaxf(most, __shfl_xor_sync(mates, most, 2));
    finite = __all_sync(mates, finite);
    const uint32_t byte = finite ? kv4_scale_byte(most) : KV4_NOT_FINITE;
    const float inverse = finite && byte ? __frcp_rn(kv4_scale(byte)) : 0.0f;
    uint32_t codes = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) codes |= kv4_code(finite ? v[i] : 0.0f, inverse) << (4 * i);
    *(unsigned short*)((value ? v_codes : k_codes) + row * (head_dim >> 1) + (d >> 1)) = (unsigned short)codes;
    if ((threadIdx.x & 3) == 0) (value ? v_scale : k_scale)[row * (head_dim >> 4) + (d >> 4)] = (uint8_t)byte;
}

// Blocks of the cache as the bfloat16 numbers they stand for.  Block i of sequence s is its logical block first + i, where `first` holds
// the oldest of the last `keep` positions (0: all of them); rows behind the sequence's end are zero.  out_table[s][b] is where logical
// block b went (0 for those before the first, which nobody may read).
constexpr int UNPACK_THREADS = 256;

__global__ void __launch_bounds__(UNPACK_THREADS)
kv4_unpack_kernel(const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ k_scale,
                  const uint8_t* __restrict__ v_scale, const int* __restrict__ block_table, int table_width,
                  const int* __restrict__ ctx_after, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                  int* __restrict__ out_table, int out_width, int num_kv_heads, int head_dim, int block_size, int keep) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.x / out_width, i = blockIdx.x - seq * out_width, kv_head = blockIdx.y;
    const int ctx = ctx_after[seq];
    const int first = keep > 0 ? max(0, ctx - keep) / block_size : 0, logical = first + i;
    if (kv_head == 0) {
        if (threadIdx.x == 0 && logical < table_width) out_table[(size_t)seq * table_width + logical] = blockIdx.x;
        if (i == 0)
            for (int b = threadIdx.x; b < table_width; b += UNPACK_THREADS)
                if (b < first || b >= first + out_width) out_table[(size_t)seq * table_width + b] = 0;
    }
    const int rows = min(block_size, ctx - logical * block_size);          // live rows of this block (none: not positive)
    const int block = logical < table_width && rows > 0 ? block_table[(size_t)seq * table_width + logical] : 0;
    const size_t from = ((size_t)block * num_kv_heads + kv_head) * block_size;
    const size_t to = ((size_t)blockIdx.x * num_kv_heads + kv_head) * block_size;
    const int words = head_dim >> 3;                                      // of eight numbers
    for (int idx = threadIdx.x; idx < 2 * block_size * words; idx += UNPACK_THREADS) {
        const bool value = idx >= block_size * words;
        const int at = idx - (value ? block_size * words : 0), row = at / words, w = at - row * words;
        uint4 out = make_uint4(0u, 0u, 0u, 0u);
        if (row < rows) {
            const uint32_t word = *(const uint32_t*)((value ? v_codes : k_codes) + (from + row) * (head_dim >> 1) + 4 * w);
            const float s = kv4_scale((value ? v_scale : k_scale)[(from + row) * (head_dim >> 4) + (w >> 1)]);
            uint32_t packed[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 pair = __floats2bfloat162_rn((float)((int)(word >> (8 * e) & 15u) - 8) * s,
                                                                  (float)((int)(word >> (8 * e + 4) & 15u) - 8) * s);
                packed[e] = *(const uint32_t*)&pair;
            }
            out = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        }
        *(uint4*)((value ? v_out : k_out) + (to + row) * head_dim + 8 * w) = out;
    }
}

}  // namespace skv

using namespace skv;

// Codes uint8 [blocks][kv_heads][block_size][head_dim / 2], scales uint8 [blocks][kv_heads][block_size][head_dim / 16].
SKV_EXPORT int skv_append_kv4(const float* qkv, const float* cos_sin, const int* positions, const int* token_seq,
                              const int* block_table, int table_width, void* q_out, void* k_codes, void* v_codes, void* k_scale,
                              void* v_scale, int n_tokens, int num_heads, int num_kv_heads, int head_dim, int block_size, int write_kv,
                              cudaStream_t stream) {
    if (n_tokens <= 0) return 0;
    if (head_dim <= 0 || head_dim % KV4_GROUP != 0) return fail("skv_append_kv4", "the head size must be a positive multiple of 16");
    if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0)
        return fail("skv_append_kv4", "heads must be a positive multiple of kv heads");
    if (block_size <= 0 || block_size % 16 != 0) return fail("skv_append_kv4", "block_size must be a positive multiple of 16");
    if (((uintptr_t)qkv | (uintptr_t)cos_sin | (uintptr_t)q_out) & 15) return fail("skv_append_kv4", "operands must be 16-byte aligned");
    const long long items = (long long)(num_heads + (write_kv ? 2 * num_kv_heads : 0)) * (head_dim / 4);
    const long long pieces = (items + APPEND_THREADS - 1) / APPEND_THREADS;
    if (pieces > 65535) return fail("skv_append_kv4", "a row of queries, keys and values is too long");
    return launch_pdl("skv_append_kv4", kv4_append_kernel, dim3(n_tokens, (unsigned)pieces), dim3(APPEND_THREADS), 0, stream, qkv, cos_sin,
                      positions, token_seq, block_table, table_width, (__nv_bfloat16*)q_out, (uint8_t*)k_codes, (uint8_t*)v_codes,
                      (uint8_t*)k_scale, (uint8_t*)v_scale, num_heads, num_kv_heads, head_dim, block_size, write_kv);
}

SKV_EXPORT int skv_unpack_kv4(const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const int* block_table,
                              int table_width, const int* ctx_after, void* k_out, void* v_out, int* out_table, int n_seqs, int out_width,
                              int num_kv_heads, int head_dim, int block_size, int keep, cudaStream_t stream) {
    if (n_seqs <= 0 || out_width <= 0) return 0;
    if (head_dim <= 0 || head_dim % KV4_GROUP != 0) return fail("skv_unpack_kv4", "the head size must be a positive multiple of 16");
    if (block_size <= 0 || block_size % 16 != 0) return fail("skv_unpack_kv4", "block_size must be a positive multiple of 16");
    if (num_kv_heads <= 0 || num_kv_heads > 65535) return fail("skv_unpack_kv4", "between 1 and 65,535 kv heads are needed");
    if (keep < 0) return fail("skv_unpack_kv4", "the positions to keep must not be negative");
    if ((long long)n_seqs * out_width > 0x7fffffffLL) return fail("skv_unpack_kv4", "too many blocks");
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15)
        return fail("skv_unpack_kv4", "operands must be 16-byte aligned");
    return launch_pdl("skv_unpack_kv4", kv4_unpack_kernel, dim3((unsigned)(n_seqs * out_width), (unsigned)num_kv_heads), dim3(UNPACK_THREADS), 0,
                      stream, (const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_table,
                      table_width, ctx_after, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, out_table, out_width, num_kv_heads, head_dim,
                      block_size, keep);
}

SKV_EXPORT int skv_has_kv4() { return 1; }

#else

SKV_EXPORT int skv_append_kv4(const float*, const float*, const int*, const int*, const int*, int, void*, void*, void*, void*, void*, int,
                              int, int, int, int, int, cudaStream_t) {
    return skv::fail("skv_append_kv4", "a 4-bit cache is built for bfloat16");
}

SKV_EXPORT int skv_unpack_kv4(const void*, const void*, const void*, const void*, const int*, int, const int*, void*, void*, int*, int, int,
                              int, int, int, int, cudaStream_t) {
    return skv::fail("skv_unpack_kv4", "a 4-bit cache is built for bfloat16");
}

SKV_EXPORT int skv_has_kv4() { return 0; }

#endif
