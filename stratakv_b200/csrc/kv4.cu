// Appending to a paged cache whose keys and values are held in 4 bits (kv4.cuh), and reading it back.
//
// The reference keeps its cache in full precision and appends a token with two device-to-device copies
// (src/models/transformer_block.cpp:484-509); it has no counterpart of these kernels.
#include "kv4.cuh"

#if SKV_DTYPE == SKV_BF16

namespace skv {

// Queries and keys of the float32 rows [q | k | v] are rotated (number i with number i + head_dim / 2; products and sum rounded one by one, so that a
// code never depends on how an expression was compiled), queries rounded to bfloat16, keys and values to codes.  Bound by the rows it
// reads once there are enough of them.
constexpr int APPEND_THREADS = 256;

// Codes and scale byte of a group of 16 whose numbers four neighbouring lanes have, four each.
__device__ __forceinline__ void kv4_store_group(const float (&v)[4], uint8_t* codes, uint8_t* scale, unsigned int mates) {
    // magnitudes are ordered as their bits are, infinities and NaN above the rest
    uint32_t bits = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) bits = max(bits, __float_as_uint(v[i]) & 0x7fffffffu);
    bits = max(bits, __shfl_xor_sync(mates, bits, 1));
    bits = max(bits, __shfl_xor_sync(mates, bits, 2));
    const bool finite = bits < 0x7f800000u;
    const uint32_t byte = finite ? kv4_scale_byte(__uint_as_float(bits)) : KV4_NOT_FINITE;
    const float inverse = finite && byte ? __frcp_rn(kv4_scale(byte)) : 0.0f;
    uint32_t packed = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) packed |= kv4_code(v[i], inverse) << (4 * i);
    if (!finite) packed = 0x8888u;
    *(unsigned short*)codes = (unsigned short)packed;
    if ((threadIdx.x & 3) == 0) *scale = (uint8_t)byte;
}
__device__ __forceinline__ void kv4_store_query(const float (&v)[4], __nv_bfloat16* to) {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
    *(uint2*)to = make_uint2(*(const uint32_t*)&lo, *(const uint32_t*)&hi);
}
__device__ __forceinline__ float turned_low(float x, float y, float c, float s) { return __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s)); }
__device__ __forceinline__ float turned_high(float x, float y, float c, float s) { return __fadd_rn(__fmul_rn(x, s), __fmul_rn(y, c)); }

// Head sizes that are multiples of 32, whose halves are whole groups: a thread has four neighbouring numbers and the four half a head further.  (Three such
// pairs a thread, 71 registers: 2,048 tokens of 32 + 2 x 8 heads of 128, read back, 30.7 us against 21.8.)
__global__ void __launch_bounds__(APPEND_THREADS, 8)
kv4_append_kernel(const float* __restrict__ qkv, const float* __restrict__ cos_sin, const int* __restrict__ positions,
                  const int* __restrict__ token_seq, const int* __restrict__ block_table, int table_width,
                  __nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ v_codes,
                  uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v_scale, int num_heads, int num_kv_heads, int head_dim,
                  int block_size, int write_kv, uint32_t quads_magic) {
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, half = head_dim >> 1, quads = half >> 2;
    const int item = blockIdx.y * APPEND_THREADS + threadIdx.x;
    const int head = (int)__umulhi((uint32_t)item, quads_magic), d = (item - head * quads) << 2;          // item / quads
    if (head >= num_heads + (write_kv ? 2 * num_kv_heads : 0)) return;     // (whole groups: half a head is a multiple of four quads)
    const float* row = qkv + (size_t)t * (num_heads + 2 * num_kv_heads) * head_dim + (size_t)head * head_dim + d;
    const float4 x = *(const float4*)row, y = *(const float4*)(row + half);
    const int pos = positions[t];
    float low[4] = {x.x, x.y, x.z, x.w}, high[4] = {y.x, y.y, y.z, y.w};
    if (cos_sin && head < num_heads + num_kv_heads) {
        const float4* at = (const float4*)(cos_sin + (size_t)pos * head_dim + 2 * d);       // (cos, sin) of four pairs
        const float4 a = at[0], b = at[1];
        const float c[4] = {a.x, a.z, b.x, b.z}, s[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float l = low[i], h = high[i];
            low[i] = turned_low(l, h, c[i], s[i]);
            high[i] = turned_high(l, h, c[i], s[i]);
        }
    }
    if (head < num_heads) {
        __nv_bfloat16* to = q_out + ((size_t)t * num_heads + head) * head_dim + d;
        kv4_store_query(low, to);
        kv4_store_query(high, to + half);
        return;
    }
    const bool value = head >= num_heads + num_kv_heads;
    const int kv_head = head - num_heads - (value ? num_kv_heads : 0);
    const int block = block_table[(size_t)token_seq[t] * table_width + pos / block_size];
    const size_t at = ((size_t)block * num_kv_heads + kv_head) * block_size + pos % block_size;
    uint8_t* codes = (value ? v_codes : k_codes) + at * half + (d >> 1);
    uint8_t* scale = (value ? v_scale : k_scale) + at * (head_dim >> 4) + (d >> 4);
    const unsigned int mates = 0xFu << (threadIdx.x & 28);
    kv4_store_group(low, codes, scale, mates);
    kv4_store_group(high, codes + (half >> 1), scale + (half >> 4), mates);
}

// Other head sizes: a thread has four neighbouring numbers, and reads those half a head away for its rotation.
__global__ void __launch_bounds__(APPEND_THREADS)
kv4_append_odd_kernel(const float* __restrict__ qkv, const float* __restrict__ cos_sin, const int* __restrict__ positions,
                      const int* __restrict__ token_seq, const int* __restrict__ block_table, int table_width,
                      __nv_bfloat16* __restrict__ q_out, uint8_t* __restrict__ k_codes, uint8_t* __restrict__ v_codes,
                      uint8_t* __restrict__ k_scale, uint8_t* __restrict__ v_scale, int num_heads, int num_kv_heads, int head_dim,
                      int block_size, int write_kv, uint32_t quads_magic) {
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, quads = head_dim >> 2, half = head_dim >> 1;
    const int item = blockIdx.y * APPEND_THREADS + threadIdx.x;
    const int head = (int)__umulhi((uint32_t)item, quads_magic), d = (item - head * quads) << 2;
    if (head >= num_heads + (write_kv ? 2 * num_kv_heads : 0)) return;     // (whole groups: a head is a multiple of four quads)
    const int pos = positions[t];
    const float* x = qkv + (size_t)t * (num_heads + 2 * num_kv_heads) * head_dim + (size_t)head * head_dim;
    const float4 own = *(const float4*)(x + d);
    float v[4] = {own.x, own.y, own.z, own.w};
    if (cos_sin && head < num_heads + num_kv_heads) {
        const bool low = d < half;
        const float4 other = *(const float4*)(x + (low ? d + half : d - half));
        const float4* at = (const float4*)(cos_sin + (size_t)pos * head_dim + 2 * (low ? d : d - half));
        const float4 a = at[0], b = at[1];
        const float w[4] = {other.x, other.y, other.z, other.w}, c[4] = {a.x, a.z, b.x, b.z}, s[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = low ? turned_low(v[i], w[i], c[i], s[i]) : turned_high(w[i], v[i], c[i], s[i]);
    }
    if (head < num_heads) {
        kv4_store_query(v, q_out + ((size_t)t * num_heads + head) * head_dim + d);
        return;
    }
    const bool value = head >= num_heads + num_kv_heads;
    const int kv_head = head - num_heads - (value ? num_kv_heads : 0);
    const int block = block_table[(size_t)token_seq[t] * table_width + pos / block_size];
    const size_t row = ((size_t)block * num_kv_heads + kv_head) * block_size + pos % block_size;
    kv4_store_group(v, (value ? v_codes : k_codes) + row * half + (d >> 1), (value ? v_scale : k_scale) + row * (head_dim >> 4) + (d >> 4),
                    0xFu << (threadIdx.x & 28));
}

// Blocks of the cache as the bfloat16 numbers they stand for.  Block i of sequence s is its logical block first + i, where `first` holds
// the oldest of the last `keep` positions (0: all of them); rows behind the sequence's end are zero.  out_table[s][b] is where logical
// block b went (0 for one that went nowhere: that is the first sequence's).
// SEEN: what a sequence's own new tokens see through a window, for a kernel that reads whole tiles of `tile` positions: `first` is the block where the
// tile of the oldest such position begins, and rows ahead of that position are zero as those behind the end are.  What left the window may have been given
// back and be another sequence's by now, and a tile multiplies its values with probabilities of zero, which make a NaN of a NaN; for the same reason an entry that went nowhere
// names the first of its own sequence.
constexpr int UNPACK_THREADS = 256, UNPACK_ITEMS = 4;          // words of eight codes that a thread has on their way at once

template <bool SEEN>
__global__ void __launch_bounds__(UNPACK_THREADS, SEEN ? 8 : 0)
kv4_unpack_kernel(const uint8_t* __restrict__ k_codes, const uint8_t* __restrict__ v_codes, const uint8_t* __restrict__ k_scale,
                  const uint8_t* __restrict__ v_scale, const int* __restrict__ block_table, int table_width,
                  const int* __restrict__ ctx_after, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                  int* __restrict__ out_table, int out_width, int num_kv_heads, int head_dim, int block_size, int keep, const int* __restrict__ cu_q,
                  int most_new, int window, int tile) {
    pdl_launch_dependents();
    pdl_wait();
    const int seq = blockIdx.x / out_width, i = blockIdx.x - seq * out_width, kv_head = blockIdx.y;
    // (for attention a length beyond the table is cut)
    const int ctx = SEEN ? (int)min((long long)ctx_after[seq], (long long)table_width * block_size) : ctx_after[seq];
    int first = 0, oldest = 0;
    if (!SEEN) {
        if (keep > 0) first = max(0, ctx - keep) / block_size;
    } else if (window > 0) {
        const int q_len = max(0, min(cu_q[seq + 1] - cu_q[seq], most_new));
        oldest = (int)max(0ll, (long long)ctx - q_len - window + 1);
        first = oldest / tile * tile / block_size;
    }
    const int logical = first + i;
    if (kv_head == 0 && blockIdx.z == 0) {
        if (threadIdx.x == 0 && logical < table_width) out_table[(size_t)seq * table_width + logical] = blockIdx.x;
        if (i == 0)
            for (int b = threadIdx.x; b < table_width; b += UNPACK_THREADS)
                if (b < first || b >= first + out_width) out_table[(size_t)seq * table_width + b] = SEEN ? seq * out_width : 0;
    }
    const int begin = SEEN ? max(0, oldest - logical * block_size) : 0, rows = min(block_size, ctx - logical * block_size) - begin;     // live rows of this block (none: not positive)
    const int block = logical < table_width && rows > 0 ? block_table[(size_t)seq * table_width + logical] : 0;
    const size_t from = ((size_t)block * num_kv_heads + kv_head) * block_size;
    const size_t to = ((size_t)blockIdx.x * num_kv_heads + kv_head) * block_size;
    const int words = head_dim >> 3, of_one = block_size * words;          // words of eight numbers
    constexpr int ITEMS = UNPACK_ITEMS;
    for (int first_item = threadIdx.x + blockIdx.z * ITEMS * UNPACK_THREADS; first_item < 2 * of_one;
         first_item += gridDim.z * ITEMS * UNPACK_THREADS) {
        uint32_t word[ITEMS], byte[ITEMS];
        size_t target[ITEMS];
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) {
            const int idx = first_item + u * UNPACK_THREADS;
            const bool value = idx >= of_one;
            const int at = idx - (value ? of_one : 0), row = at / words, w = at - row * words;
            const bool live = idx < 2 * of_one && (SEEN ? (uint32_t)(row - begin) < (uint32_t)max(0, rows) : row < rows);
            word[u] = live ? *(const uint32_t*)((value ? v_codes : k_codes) + (from + row) * (head_dim >> 1) + 4 * w) : 0u;
            byte[u] = live ? (value ? v_scale : k_scale)[(from + row) * (head_dim >> 4) + (w >> 1)] : 0u;
            target[u] = (to + row) * head_dim + 8 * w;
        }
#pragma unroll
        for (int u = 0; u < ITEMS; ++u) {
            const int idx = first_item + u * UNPACK_THREADS;
            if (idx >= 2 * of_one) break;
            const float s = kv4_scale(byte[u]);                            // (0 where no row is live, and so is all that it scales)
            uint32_t packed[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const __nv_bfloat162 pair = __floats2bfloat162_rn((float)((int)(word[u] >> (8 * e) & 15u) - 8) * s,
                                                                  (float)((int)(word[u] >> (8 * e + 4) & 15u) - 8) * s);
                packed[e] = byte[u] ? *(const uint32_t*)&pair : 0u;        // (no negative zero)
            }
            *(uint4*)((idx >= of_one ? v_out : k_out) + target[u]) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
        }
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
    if (((uintptr_t)qkv | (uintptr_t)cos_sin | (uintptr_t)q_out | (uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_scale | (uintptr_t)v_scale) & 15)
        return fail("skv_append_kv4", "operands must be 16-byte aligned");
    // twice four numbers a thread, or four
    const bool paired = head_dim % 32 == 0;
    const long long items = (long long)(num_heads + (write_kv ? 2 * num_kv_heads : 0)) * (head_dim / (paired ? 8 : 4));
    const long long pieces = (items + APPEND_THREADS - 1) / APPEND_THREADS;
    if (pieces > 65535) return fail("skv_append_kv4", "a row of queries, keys and values is too long");
    // item / quads as the upper half of a product: exact while items x quads stay below 2^32
    const uint32_t quads = head_dim / (paired ? 8 : 4), quads_magic = (uint32_t)((0x100000000ull + quads - 1) / quads);
    if ((items + APPEND_THREADS) * quads >= 0x100000000ll) return fail("skv_append_kv4", "a row of queries, keys and values is too long");
    auto kernel = paired ? kv4_append_kernel : kv4_append_odd_kernel;
    return launch_pdl("skv_append_kv4", kernel, dim3(n_tokens, (unsigned)pieces), dim3(APPEND_THREADS), 0, stream, qkv, cos_sin, positions, token_seq,
                      block_table, table_width, (__nv_bfloat16*)q_out, (uint8_t*)k_codes, (uint8_t*)v_codes, (uint8_t*)k_scale, (uint8_t*)v_scale,
                      num_heads, num_kv_heads, head_dim, block_size, write_kv, quads_magic);
}

static int unpack_kv4(const char* name, const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const int* block_table,
                      int table_width, const int* ctx_after, void* k_out, void* v_out, int* out_table, int n_seqs, int out_width, int num_kv_heads,
                      int head_dim, int block_size, int keep, const int* cu_q, int most_new, int window, int tile, cudaStream_t stream) {
    if (n_seqs <= 0 || out_width <= 0) return 0;
    if (head_dim <= 0 || head_dim % KV4_GROUP != 0) return fail(name, "the head size must be a positive multiple of 16");
    if (block_size <= 0 || block_size % 16 != 0) return fail(name, "block_size must be a positive multiple of 16");
    if (num_kv_heads <= 0 || num_kv_heads > 65535) return fail(name, "between 1 and 65,535 kv heads are needed");
    if (keep < 0) return fail(name, "the positions to keep must not be negative");
    if ((long long)n_seqs * out_width > 0x7fffffffLL) return fail(name, "too many blocks");
    if (((uintptr_t)k_codes | (uintptr_t)v_codes | (uintptr_t)k_out | (uintptr_t)v_out) & 15)
        return fail(name, "operands must be 16-byte aligned");
    const long long items = 2ll * block_size * (head_dim / 8);
    if (items > 0x40000000ll) return fail(name, "a cache block is too large");
    const long long wanted = (items + UNPACK_ITEMS * UNPACK_THREADS - 1) / (UNPACK_ITEMS * UNPACK_THREADS), parts = wanted < 64 ? wanted : 64;
    return launch_pdl(name, cu_q ? kv4_unpack_kernel<true> : kv4_unpack_kernel<false>, dim3((unsigned)(n_seqs * out_width), (unsigned)num_kv_heads, (unsigned)parts), dim3(UNPACK_THREADS), 0,
                      stream, (const uint8_t*)k_codes, (const uint8_t*)v_codes, (const uint8_t*)k_scale, (const uint8_t*)v_scale, block_table,
                      table_width, ctx_after, (__nv_bfloat16*)k_out, (__nv_bfloat16*)v_out, out_table, out_width, num_kv_heads, head_dim,
                      block_size, keep, cu_q, most_new, window, tile);
}

SKV_EXPORT int skv_unpack_kv4(const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const int* block_table,
                              int table_width, const int* ctx_after, void* k_out, void* v_out, int* out_table, int n_seqs, int out_width,
                              int num_kv_heads, int head_dim, int block_size, int keep, cudaStream_t stream) {
    return unpack_kv4("skv_unpack_kv4", k_codes, v_codes, k_scale, v_scale, block_table, table_width, ctx_after, k_out, v_out, out_table, n_seqs, out_width,
                      num_kv_heads, head_dim, block_size, keep, nullptr, 0, 0, 1, stream);
}

// What the new tokens cu_q[s] .. cu_q[s + 1] - 1 of a sequence (at most most_new of them) see through a window (0: none), for a reader of tiles of `tile` positions.
SKV_EXPORT int skv_unpack_kv4_seen(const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, const int* block_table,
                                   int table_width, const int* ctx_after, void* k_out, void* v_out, int* out_table, int n_seqs, int out_width,
                                   int num_kv_heads, int head_dim, int block_size, const int* cu_q, int most_new, int window, int tile,
                                   cudaStream_t stream) {
    if (n_seqs > 0 && out_width > 0 && (!cu_q || most_new < 0 || window < 0 || tile <= 0))
        return fail("skv_unpack_kv4_seen", "the tokens' offsets and a positive tile are needed, most_new and window must not be negative");
    return unpack_kv4("skv_unpack_kv4_seen", k_codes, v_codes, k_scale, v_scale, block_table, table_width, ctx_after, k_out, v_out, out_table, n_seqs,
                      out_width, num_kv_heads, head_dim, block_size, 0, cu_q, most_new, window, tile, stream);
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

SKV_EXPORT int skv_unpack_kv4_seen(const void*, const void*, const void*, const void*, const int*, int, const int*, void*, void*, int*, int, int, int,
                                   int, int, const int*, int, int, int, cudaStream_t) {
    return skv::fail("skv_unpack_kv4_seen", "a 4-bit cache is built for bfloat16");
}

SKV_EXPORT int skv_has_kv4() { return 0; }

#endif
