// mx.hip — microscaled 4-bit (MXFP4): rows to and from f32, MUL_MAT, MUL_MAT_ID, and the experts' bias rows (ADD_ID).
//
// A block is 32 values: a byte e and 16 bytes of codes, value j in the low nibble of byte j, value 16 + j in the high nibble.  A value is E2M1(code) 2^(e - 127), E2M1 = 0, 1/2, 1, 3/2, 2, 3, 4,
// 6 with the sign in bit 3; e = 255 makes the whole block NaN.
//
// Products.  The matrix cores take two operands of 4 .. 8 bits per value and a power of two per 32 of them, and multiply by both powers themselves (v_mfma_scale_f32_*_f8f6f4): a weight block goes
// in as it lies in memory.  The activations are quantised to the same form, a block of 32 as whole numbers q of -255 .. 255 times 2^s (the counterpart of the Q8_0 / Q8_K activations of the other
// block formats; half a step is at most 2^-8 of the block's largest value, Q8_0's 1 / 254).  |q| = 16 h + l, and each of h, l <= 15 is one E2M3 value (6 bits: the codes 0 .. 15 stand for code / 8):
// two instructions a tile, at twice the rate of 8-bit operands, and their products are exact.  Only the f32 sums round.
#include "common.h"
#include "dev_util.h"
#include "kernels.h"

namespace mi355x {

typedef int mx_i4 __attribute__((ext_vector_type(4)));
typedef int mx_i2 __attribute__((ext_vector_type(2)));
typedef int mx_i8 __attribute__((ext_vector_type(8)));
typedef float mx_f4 __attribute__((ext_vector_type(4)));
typedef float mx_f16 __attribute__((ext_vector_type(16)));
typedef mx_i4 __attribute__((aligned(4))) mx_i4_a4;
typedef uint32_t __attribute__((aligned(1))) mx_u32_a1;
typedef mx_f4 __attribute__((aligned(4))) mx_f4_a4;

static constexpr int MX_BLOCK = 17;  // bytes
static constexpr int MX_FP4 = 4, MX_FP6 = 2;  // operand formats of the matrix instructions: E2M1, E2M3

// ------------------------------------------------------------------------------------------------ rows
// Four lanes share a block: lane i of them has the values 4i .. 4i + 3 (v[0]) and 16 + 4i .. 16 + 4i + 3 (v[1]), whose codes are the bytes 4i .. 4i + 3.
// the bits of the block's largest magnitude (an infinity's or NaN's bits are larger than any number's)
__device__ __forceinline__ uint32_t mx_top(const mx_f4 (&v)[2]) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = max(m, __float_as_uint(v[k >> 2][k & 3]) & 0x7FFFFFFFu);
    m = max(m, (uint32_t) dpp_i32<MI_DPP_QUAD_XOR1>((int) m));
    return max(m, (uint32_t) dpp_i32<MI_DPP_QUAD_XOR2>((int) m));
}
__device__ __forceinline__ void mx_load8(const char * at, const int i, mx_f4 (&v)[2]) {
    v[0] = *(const mx_f4_a4 *) (at + 16 * i);
    v[1] = *(const mx_f4_a4 *) (at + 64 + 16 * i);
}
// the nearest code of v 2^x, a tie to the lower one (of two magnitudes the smaller, of two zeros +0).  From 1 on a code is exponent and first bit of the mantissa, rounded down in a tie
__device__ __forceinline__ uint32_t mx_code(const float v, const int x) {
    const float m = __builtin_amdgcn_ldexpf(fabsf(v), x);
    const uint32_t high = min(((__float_as_uint(m) + 0x1FFFFFu) >> 22) - 0xFCu, 7u), low = (uint32_t) (m > 0.25f) + (uint32_t) (m > 0.75f), c = m >= 1.0f ? high : low;
    return c ? c | ((__float_as_uint(v) >> 31) << 3) : 0u;
}
// -> the block's scale byte; the lane's four bytes of codes
__device__ __forceinline__ int mx_quantise8(const mx_f4 (&v)[2], uint32_t & codes) {
    const uint32_t top = mx_top(v);
    const int e = top >= 0x7F800000u ? 255 : max((int) (top >> 23) - 2, 0);  // floor(log2) - 2 + 127 (a subnormal's is below every scale)
    codes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) codes |= (mx_code(v[0][k], 127 - e) | mx_code(v[1][k], 127 - e) << 4) << (8 * k);
    if (e == 255) codes = 0;
    return e;
}
// 2^(e - 127) as f32 (e = 0: subnormal), NaN for 255
__device__ __forceinline__ float mx_scale(const int e) { return e == 255 ? __uint_as_float(0x7FC00000u) : e == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t) e << 23); }
__device__ __forceinline__ float mx_value(const uint32_t code, const float scale) {
    // magnitudes 0 .. 7 doubled: 0 1 2 3 4 6 8 12, a nibble each
    const float m = 0.5f * (float) ((0xC8643210u >> (4 * (code & 7))) & 15u);
    return ((code & 8) ? -m : m) * scale;
}
__device__ __forceinline__ void mx_put8(char * at, const int i, const uint32_t c, const float s) {
    mx_f4 v[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[0][k] = mx_value((c >> (8 * k)) & 15, s);
        v[1][k] = mx_value((c >> (8 * k + 4)) & 15, s);
    }
    *(mx_f4_a4 *) (at + 16 * i) = v[0];
    *(mx_f4_a4 *) (at + 64 + 16 * i) = v[1];
}
// Row blockIdx.x, 64 blocks of it.  f32 rows -> blocks; idx: SET_ROWS, the rows' places (one outside the destination is skipped); without: row i to row i
template <bool IDX> __global__ void __launch_bounds__(256) k_mx_store(const tdesc a, const tdesc idx, const tdesc d) {
    const uint32_t row = blockIdx.x, n1 = (uint32_t) a.ne[1], n2 = (uint32_t) a.ne[2], r23 = row / n1, i1 = row - r23 * n1, i3 = r23 / n2, i2 = r23 - i3 * n2;
    const int blk = (int) (blockIdx.y * 64 + (threadIdx.x >> 2)), i = threadIdx.x & 3;
    if (blk >= a.ne[0] / 32) return;  // (four lanes leave together)
    int64_t to = i1;
    if (IDX) {
        to = *(const int64_t *) (idx.data + i1 * idx.nb[0] + (i2 % (uint32_t) idx.ne[1]) * idx.nb[1] + (i3 % (uint32_t) idx.ne[2]) * idx.nb[2]);
        if (to < 0 || to >= d.ne[1]) return;
    }
    mx_f4 v[2];
    mx_load8(a.data + i1 * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3] + (int64_t) blk * 128, i, v);
    uint32_t codes;
    const int e = mx_quantise8(v, codes);
    uint8_t * out = (uint8_t *) d.data + to * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3] + (int64_t) blk * MX_BLOCK;
    if (i == 0) out[0] = (uint8_t) e;
    *(mx_u32_a1 *) (out + 1 + 4 * i) = codes;
}
// blocks -> f32 rows; idx: GET_ROWS, the rows taken (one outside the source is skipped)
template <bool IDX> __global__ void __launch_bounds__(256) k_mx_read(const tdesc a, const tdesc idx, const tdesc d) {
    const uint32_t row = blockIdx.x, n1 = (uint32_t) d.ne[1], n2 = (uint32_t) d.ne[2], r23 = row / n1, i1 = row - r23 * n1, i3 = r23 / n2, i2 = r23 - i3 * n2;
    const int blk = (int) (blockIdx.y * 64 + (threadIdx.x >> 2)), i = threadIdx.x & 3;
    if (blk >= a.ne[0] / 32) return;
    int64_t from = i1;
    if (IDX) {
        from = *(const int32_t *) (idx.data + i1 * idx.nb[0] + i2 * idx.nb[1] + i3 * idx.nb[2]);
        if (from < 0 || from >= a.ne[1]) return;
    }
    const uint8_t * in = (const uint8_t *) a.data + from * a.nb[1] + i2 * a.nb[2] + i3 * a.nb[3] + (int64_t) blk * MX_BLOCK;
    mx_put8(d.data + i1 * d.nb[1] + i2 * d.nb[2] + i3 * d.nb[3] + (int64_t) blk * 128, i, *(const mx_u32_a1 *) (in + 1 + 4 * i), mx_scale(in[0]));
}
// Dense tensors (CPY): a workgroup has 256 blocks, whose 4352 bytes cross LDS so that they are read and written 16 bytes at a time.  Bytes bound it: 14336 x 4096 values there and back, 532 MB, 113 us, 4.7
// TB/s, a large copy's rate (byte by byte as above: 151 us)
static constexpr int MX_CPY = 256;
__global__ void __launch_bounds__(256) k_mx_store_dense(const char * __restrict__ x, uint8_t * __restrict__ out, const int64_t blocks) {
    __shared__ __align__(16) uint8_t s[MX_CPY * MX_BLOCK];
    const int64_t b0 = (int64_t) blockIdx.x * MX_CPY;
    const int n = (int) min((int64_t) MX_CPY, blocks - b0), tid = threadIdx.x, i = tid & 3;
    mx_f4 v[4][2];
#pragma unroll
    for (int k = 0; k < 4; ++k) mx_load8(x + (b0 + min(64 * k + (tid >> 2), n - 1)) * 128, i, v[k]);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int blk = 64 * k + (tid >> 2);
        uint32_t codes;
        const int e = mx_quantise8(v[k], codes);
        if (i == 0) s[blk * MX_BLOCK] = (uint8_t) e;
        *(mx_u32_a1 *) (s + blk * MX_BLOCK + 1 + 4 * i) = codes;
    }
    __syncthreads();
    uint8_t * to = out + b0 * MX_BLOCK;
    const int bytes = n * MX_BLOCK;
    for (int at = tid; at < bytes / 16; at += 256) ((mx_i4 *) to)[at] = ((const mx_i4 *) s)[at];
    for (int at = (bytes & ~15) + tid; at < bytes; at += 256) to[at] = s[at];
}
__global__ void __launch_bounds__(256) k_mx_read_dense(const uint8_t * __restrict__ in, char * __restrict__ out, const int64_t blocks) {
    __shared__ __align__(16) uint8_t s[MX_CPY * MX_BLOCK];
    const int64_t b0 = (int64_t) blockIdx.x * MX_CPY;
    const int n = (int) min((int64_t) MX_CPY, blocks - b0), tid = threadIdx.x, i = tid & 3, bytes = n * MX_BLOCK;
    const uint8_t * from = in + b0 * MX_BLOCK;
    for (int at = tid; at < bytes / 16; at += 256) ((mx_i4 *) s)[at] = ((const mx_i4 *) from)[at];
    for (int at = (bytes & ~15) + tid; at < bytes; at += 256) s[at] = from[at];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int blk = 64 * k + (tid >> 2);
        if (blk < n) mx_put8(out + (b0 + blk) * 128, i, *(const mx_u32_a1 *) (s + blk * MX_BLOCK + 1 + 4 * i), mx_scale(s[blk * MX_BLOCK]));
    }
}
// the launches' sizes: rows, 64 blocks of a row each (a launch has less than 2^32 threads in x)
static dim3 mx_rows_grid(const tdesc & t) { return dim3((unsigned) (t.ne[1] * t.ne[2] * t.ne[3]), (unsigned) ((t.ne[0] / 32 + 63) / 64)); }
bool mx_rows_ok(const tdesc & f32) { return f32.ne[1] * f32.ne[2] * f32.ne[3] < ((int64_t) 1 << 24) && f32.ne[0] / 32 <= 64 * 65535; }
void launch_mx_store(hipStream_t s, const tdesc & a, const tdesc * idx, const tdesc & d) {
    const int64_t n = (a.ne[0] / 32) * a.ne[1] * a.ne[2] * a.ne[3];
    if (n <= 0) return;
    if (idx) hipLaunchKernelGGL(k_mx_store<true>, mx_rows_grid(a), dim3(256), 0, s, a, *idx, d);
    else if (((uintptr_t) d.data & 15) == 0) hipLaunchKernelGGL(k_mx_store_dense, dim3((unsigned) ((n + MX_CPY - 1) / MX_CPY)), dim3(256), 0, s, a.data, (uint8_t *) d.data, n);
    else hipLaunchKernelGGL(k_mx_store<false>, mx_rows_grid(a), dim3(256), 0, s, a, a, d);
}
void launch_mx_read(hipStream_t s, const tdesc & a, const tdesc * idx, const tdesc & d) {
    const int64_t n = (a.ne[0] / 32) * d.ne[1] * d.ne[2] * d.ne[3];
    if (n <= 0) return;
    if (idx) hipLaunchKernelGGL(k_mx_read<true>, mx_rows_grid(d), dim3(256), 0, s, a, *idx, d);
    else if (((uintptr_t) a.data & 15) == 0) hipLaunchKernelGGL(k_mx_read_dense, dim3((unsigned) ((n + MX_CPY - 1) / MX_CPY)), dim3(256), 0, s, (const uint8_t *) a.data, d.data, n);
    else hipLaunchKernelGGL(k_mx_read<false>, mx_rows_grid(d), dim3(256), 0, s, a, a, d);
}

// ------------------------------------------------------------------------------------------------ activations
// The quantised columns lie in groups of 32, a group in steps of 128 values (four blocks), as the lanes of a product fetch them: for each block the 16 first bytes of h of the 32 columns, those of l, the
// 8 last bytes of h, those of l (24 bytes are 32 codes of 6 bits), and behind the four blocks 4 scale bytes a column.  A block's codes stand in the order of the weights' nibbles: value j at place 2j,
// value 16 + j at place 2j + 1.  The scale byte is h's exponent, s + 7 + 127; l's is 4 less.  Blocks behind the last one of a row are zeros (a product takes the row's last block once more for them: whatever it holds, its own product is in the sum already).
static constexpr int MX_ACT_BLK = 32 * 48, MX_ACT_STEP = 4 * MX_ACT_BLK + 32 * 4;
static inline int64_t mx_steps(int64_t K) { return (K + 127) / 128; }
size_t mx_act_bytes(int64_t K, int64_t cols) { return (size_t) ((cols + 31) / 32) * (size_t) (mx_steps(K) * MX_ACT_STEP); }

// Columns of MUL_MAT_ID sorted by expert, every expert's first column in a group of its own: list[p] the column (u + n_used t) at place p or -1, owner[g] the expert of group g, tiles[4 t]: up to
// MX_TILE groups of one expert as (expert, first group, groups); total[0] and total[1]: groups and tiles in use
struct mx_lists {
    int32_t * total, * tiles, * owner, * list;
};
static constexpr int MX_TILE = 4;
// ids outside the experts are in no list: their columns are left as they are
static int64_t mx_id_groups(int64_t n_expert, int64_t cols) { return cols / 32 + std::min(n_expert, cols); }  // (at most: an expert's last group may hold one column)
static int64_t mx_id_tiles(int64_t n_expert, int64_t cols) { return cols / (32 * MX_TILE) + std::min(n_expert, cols); }
static mx_lists mx_lists_at(void * ws, int64_t groups) {  // (no more tiles than groups)
    mx_lists l;
    l.total = (int32_t *) ws;
    l.tiles = l.total + 4;
    l.owner = l.tiles + 4 * groups;
    l.list = l.owner + ((groups + 3) & ~(int64_t) 3);
    return l;
}
static size_t mx_lists_bytes(int64_t groups) { return ((size_t) (4 + 4 * groups + ((groups + 3) & ~(int64_t) 3) + groups * 32) * 4 + 255) & ~(size_t) 255; }
size_t mx_id_act_bytes(int64_t K, int64_t n_expert, int64_t cols) {
    const int64_t g = mx_id_groups(n_expert, cols);
    return mx_lists_bytes(g) + mx_act_bytes(K, 32 * g);
}
static constexpr int MX_MAX_EXPERTS = 1024;
// One workgroup an expert: every workgroup counts all experts' columns (whole numbers in LDS: no order to depend on), takes the groups and tiles in front of its own, and lists its columns in ascending
// order.  A round is MX_IDS ids a thread, requested at once (4000 ids of 32 experts: 15.7 us with one id a thread and round on 256 threads).
static constexpr int MX_IDS = 4;
__global__ void __launch_bounds__(1024) k_mx_group(const tdesc ids, const int n_expert, const mx_lists l) {
    __shared__ int cnt[MX_MAX_EXPERTS], s_before[16], s_tiles[16], s_hits[MX_IDS * 16];
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t n_used = (uint32_t) ids.ne[0], n = n_used * (uint32_t) ids.ne[1];
    int32_t id[MX_IDS];
    auto fetch = [&](const uint32_t i0) {
#pragma unroll
        for (int k = 0; k < MX_IDS; ++k) {
            const uint32_t i = i0 + (uint32_t) (k * 1024 + tid), t = i / n_used;
            id[k] = i < n ? *(const int32_t *) (ids.data + (int64_t) (i - t * n_used) * ids.nb[0] + (int64_t) t * ids.nb[1]) : -1;
        }
    };
    fetch(0);
    if (tid < n_expert) cnt[tid] = 0;
    __syncthreads();
    for (uint32_t i0 = 0; i0 < n; i0 += MX_IDS * 1024) {
        if (i0) fetch(i0);
#pragma unroll
        for (int k = 0; k < MX_IDS; ++k)
            if (id[k] >= 0 && id[k] < n_expert) atomicAdd(&cnt[id[k]], 1);
    }
    __syncthreads();
    int before = 0, before_t = 0;
    if (tid < e) {
        before = (cnt[tid] + 31) / 32;
        before_t = (before + MX_TILE - 1) / MX_TILE;
    }
    for (int o = 32; o > 0; o >>= 1) {
        before += __shfl_xor(before, o, 64);
        before_t += __shfl_xor(before_t, o, 64);
    }
    if (lane == 0) {
        s_before[wave] = before;
        s_tiles[wave] = before_t;
    }
    __syncthreads();
    int g0 = 0, t0 = 0;
    for (int w = 0; w < 16; ++w) {
        g0 += s_before[w];
        t0 += s_tiles[w];
    }
    const int mine = cnt[e], groups = (mine + 31) / 32, tiles = (groups + MX_TILE - 1) / MX_TILE;
    for (int i = tid; i < tiles; i += 1024) {
        int32_t * t = l.tiles + 4 * (t0 + i);
        t[0] = e;
        t[1] = g0 + MX_TILE * i;
        t[2] = min(MX_TILE, groups - MX_TILE * i);
    }
    for (int i = tid; i < groups; i += 1024) l.owner[g0 + i] = e;
    for (int i = mine + tid; i < groups * 32; i += 1024) l.list[g0 * 32 + i] = -1;
    if (e == n_expert - 1 && tid == 0) {
        l.total[0] = g0 + groups;
        l.total[1] = t0 + tiles;
    }
    if (mine == 0) return;
    int placed = g0 * 32;
    for (uint32_t i0 = 0; i0 < n; i0 += MX_IDS * 1024) {
        if (n > MX_IDS * 1024) fetch(i0);  // (else they are still at hand)
        uint64_t hit[MX_IDS];
#pragma unroll
        for (int k = 0; k < MX_IDS; ++k) hit[k] = __ballot(id[k] == e);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < MX_IDS; ++k)
            if (lane == 0) s_hits[k * 16 + wave] = __popcll(hit[k]);
        __syncthreads();
        int sum = s_hits[lane];  // (64 counts in the order of the columns: an inclusive sum over them)
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(sum, o, 64);
            if (lane >= o) sum += v;
        }
#pragma unroll
        for (int k = 0; k < MX_IDS; ++k) {
            const int at = __shfl(sum, k * 16 + wave, 64) - __popcll(hit[k]);
            if (id[k] == e) l.list[placed + at + __popcll(hit[k] & ((1ull << lane) - 1ull))] = (int32_t) (i0 + (uint32_t) (k * 1024 + tid));
        }
        placed += __shfl(sum, 63, 64);
    }
}

// whole numbers and step of a block: q = v f rounded, f = 2^-s, s the exponent of the block's largest magnitude (its bits: top), rounded to 8 significant bits, - 7; -> the scale byte of h
__device__ __forceinline__ uint32_t mx_step(const uint32_t top, float & f) {
    const int s = min(max((int) ((top + 0x8000u) >> 23) - 134, -120), 120);
    f = top >= 0x7F800000u ? 0.0f : __uint_as_float((uint32_t) (127 - s) << 23);
    return top >= 0x7F800000u ? 255u : (uint32_t) (s + 134);
}
// one value's digits: 6 bits of h, of l
__device__ __forceinline__ void mx_digits(const float v, const float f, uint32_t & h, uint32_t & l) {
    const float q = rintf(v * f);
    const uint32_t m = min((uint32_t) fabsf(q), 255u), sign = (__float_as_uint(q) >> 26) & 32u;
    h = (m >> 4) | sign;
    l = (m & 15) | sign;
}
// Four lanes a block: lane i has the values 4i .. 4i + 3 (v[0]) and 16 + 4i .. 16 + 4i + 3 (v[1]), places 8i .. 8i + 7, 48 bits of h and of l; a pair of lanes has three dwords of each, put(d, ..) is given
// dword d of the block's six.  -> the scale byte
template <class Put> __device__ __forceinline__ uint32_t mx_act_quad(const mx_f4 (&v)[2], const int i, Put && put) {
    float f;
    const uint32_t e = mx_step(mx_top(v), f);
    uint64_t h = 0, l = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {  // place k: value k / 2 of the first four or of the second
        uint32_t a, b;
        mx_digits(v[k & 1][k >> 1], f, a, b);
        h |= (uint64_t) a << (6 * k);
        l |= (uint64_t) b << (6 * k);
    }
    if (e == 255u) h = l = 0;  // (0 f is NaN for an infinity: the digits do not matter beside this scale, but they are numbers)
    // an even lane's six bytes and its neighbour's: dwords 0, 1 (its last two bytes and the neighbour's first two), 2 (the neighbour's other four)
    const uint32_t hn = (uint32_t) dpp_i32<MI_DPP_QUAD_XOR1>((int) (uint32_t) h), ln = (uint32_t) dpp_i32<MI_DPP_QUAD_XOR1>((int) (uint32_t) l);
    const int d = 3 * (i >> 1);
    if (i & 1) put(d + 2, (uint32_t) (h >> 16), (uint32_t) (l >> 16));
    else {
        put(d, (uint32_t) h, (uint32_t) l);
        put(d + 1, (uint32_t) (h >> 32) | hn << 16, (uint32_t) (l >> 32) | ln << 16);
    }
    return e;
}
// One workgroup a group of columns and a step of 128 values.  The 6272 bytes are put together in LDS and leave in 16-byte pieces.  ID: column c of the list is row (c % n_used) % b.ne[1] of token c / n_used
template <bool ID> __global__ void __launch_bounds__(256) k_mx_act(const tdesc b, const int64_t n_cols, const mx_lists l, const int n_used, uint8_t * __restrict__ act, const int steps) {
    __shared__ __align__(16) uint8_t s[MX_ACT_STEP];
    const int step = blockIdx.x, group = blockIdx.y, tid = threadIdx.x;
    int listed[2];
    if (ID) {  // (requested together; behind the groups in use the list's room holds anything)
        listed[0] = l.list[group * 32 + (tid >> 4)];
        listed[1] = l.list[group * 32 + 16 + (tid >> 4)];
        if (group >= l.total[0]) return;
    }
    const int i = tid & 3, blk = (tid >> 2) & 3;
    const int64_t k0 = (int64_t) step * 128 + blk * 32;
    mx_f4 v[2][2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        int c = group * 32 + r * 16 + (tid >> 4);
        const char * col;
        if (ID) {
            c = listed[r];
            col = b.data + ((c % n_used) % (int) b.ne[1]) * b.nb[1] + (int64_t) (c / n_used) * b.nb[2];
        } else {
            const uint32_t n1 = (uint32_t) b.ne[1], n2 = (uint32_t) b.ne[2], c2 = (uint32_t) c / n1, c3 = c2 / n2;
            col = b.data + (int64_t) ((uint32_t) c - c2 * n1) * b.nb[1] + (int64_t) (c2 - c3 * n2) * b.nb[2] + (int64_t) c3 * b.nb[3];
            if (c >= n_cols) c = -1;
        }
        v[r][0] = v[r][1] = mx_f4{0, 0, 0, 0};
        if (c >= 0 && k0 < b.ne[0]) {
            v[r][0] = *(const mx_f4_a4 *) (col + (k0 + 4 * i) * 4);
            v[r][1] = *(const mx_f4_a4 *) (col + (k0 + 16 + 4 * i) * 4);
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int cg = r * 16 + (tid >> 4);
        uint8_t * o = s + blk * MX_ACT_BLK;
        const uint32_t e = mx_act_quad(v[r], i, [&](const int d, const uint32_t h, const uint32_t lo) {
            *(uint32_t *) (o + (d < 4 ? cg * 16 + 4 * d : 1024 + cg * 8 + 4 * (d - 4))) = h;
            *(uint32_t *) (o + (d < 4 ? 512 + cg * 16 + 4 * d : 1280 + cg * 8 + 4 * (d - 4))) = lo;
        });
        if (i == 0) s[4 * MX_ACT_BLK + cg * 4 + blk] = (uint8_t) e;
    }
    __syncthreads();
    uint8_t * out = act + ((int64_t) group * steps + step) * MX_ACT_STEP;
    for (int at = tid; at < MX_ACT_STEP / 16; at += 256) ((mx_i4 *) out)[at] = ((const mx_i4 *) s)[at];
}
void launch_mx_act(hipStream_t s, const tdesc & b, void * act) {
    const int64_t cols = b.ne[1] * b.ne[2] * b.ne[3], steps = mx_steps(b.ne[0]);
    hipLaunchKernelGGL(k_mx_act<false>, dim3((unsigned) steps, (unsigned) ((cols + 31) / 32)), dim3(256), 0, s, b, cols, mx_lists{}, 1, (uint8_t *) act, (int) steps);
}
void launch_mx_group(hipStream_t s, const tdesc & ids, int64_t n_expert, void * ws) {
    hipLaunchKernelGGL(k_mx_group, dim3((unsigned) n_expert), dim3(1024), 0, s, ids, (int) n_expert, mx_lists_at(ws, mx_id_groups(n_expert, ids.ne[0] * ids.ne[1])));
}
void launch_mx_id_act(hipStream_t s, const tdesc & b, const tdesc & ids, int64_t n_expert, void * ws) {
    const int64_t cols = ids.ne[0] * ids.ne[1], steps = mx_steps(b.ne[0]), g = mx_id_groups(n_expert, cols);
    hipLaunchKernelGGL(k_mx_act<true>, dim3((unsigned) steps, (unsigned) g), dim3(256), 0, s, b, cols, mx_lists_at(ws, g), (int) ids.ne[0], (uint8_t *) ws + mx_lists_bytes(g), (int) steps);
}

// ------------------------------------------------------------------------------------------------ products
struct mx_mm {
    const uint8_t * w;
    int64_t nb1, nb2;     // bytes between rows, between experts
    int n_rows, blocks;   // rows of the (an expert's) matrix; blocks of a row
    const uint8_t * act;
    int steps;            // of 128 values
    int64_t cols;         // columns of the product
    int n_expert;
    float * dst;          // column c at dst + c ldd
    int64_t ldd;
    const float * bias;   // + bias[expert] (nb_bias bytes apart), or null
    int64_t nb_bias;
    mx_lists l;
};
__device__ __forceinline__ mx_i8 mx_op4(const mx_i4 a) { return mx_i8{a.x, a.y, a.z, a.w, 0, 0, 0, 0}; }
__device__ __forceinline__ mx_i8 mx_op6(const mx_i4 a, const mx_i2 b) { return mx_i8{a.x, a.y, a.z, a.w, b.x, b.y, 0, 0}; }

// Weights.  A row is a run of 17-byte blocks; a lane takes four blocks (a step's 128 values, 68 bytes) of one row at a time.  Loads at odd addresses cost four times those at whole dwords, so the 68
// bytes come as 17 dwords and the codes are moved into place (GB/s over rows of 2176 bytes: 16 bytes at 17 b + 1 and a byte at 17 b 2335, the dwords around a block 4750, 17 dwords a lane 6960,
// aligned 16-byte loads of something else 7500).  A scale byte stays where it is, byte j of its dword: the instruction picks it.
// DW: rows of whole steps at whole dwords (K a multiple of 128); otherwise block by block, the dwords around each (none of them without a byte of the block).
template <bool DW> struct mx_raw;
template <> struct mx_raw<true> {
    mx_i4 v[4];
    int d;
    __device__ __forceinline__ void load(const uint8_t * row, const int step, const int) {
        const uint8_t * p = row + (int64_t) step * (4 * MX_BLOCK);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = *(const mx_i4_a4 *) (p + 16 * i);
        d = *(const int *) (p + 64);
    }
    __device__ __forceinline__ void place(const int j, mx_i4 & a, int & s) const {  // block j's codes; a dword whose byte j is its scale
        const int q[17] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w, v[2].x, v[2].y, v[2].z, v[2].w, v[3].x, v[3].y, v[3].z, v[3].w, d};
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = j == 3 ? q[i + 13] : (int) __builtin_amdgcn_alignbyte(q[4 * j + i + 1], q[4 * j + i], j + 1);
        s = q[4 * j];
    }
};
// a block's codes out of the five dwords around it, sh the first one's bytes in front of the block
__device__ __forceinline__ mx_i4 mx_window(const mx_i4 v, const int d, const uint32_t sh) {
    const uint32_t sel = 0x04030201u + 0x01010101u * sh;
    return mx_i4{(int) __builtin_amdgcn_perm((uint32_t) v.y, (uint32_t) v.x, sel), (int) __builtin_amdgcn_perm((uint32_t) v.z, (uint32_t) v.y, sel),
                 (int) __builtin_amdgcn_perm((uint32_t) v.w, (uint32_t) v.z, sel), (int) __builtin_amdgcn_perm((uint32_t) d, (uint32_t) v.w, sel)};
}
template <> struct mx_raw<false> {
    mx_i4 v[4];
    int d[4];
    uint32_t sh[4];
    __device__ __forceinline__ void load(const uint8_t * row, const int step, const int blocks) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uintptr_t p = (uintptr_t) row + (uintptr_t) (min(step * 4 + j, blocks - 1) * MX_BLOCK);
            const uint8_t * q = (const uint8_t *) (p & ~(uintptr_t) 3);
            sh[j] = (uint32_t) p & 3u;
            v[j] = *(const mx_i4_a4 *) q;
            d[j] = *(const int *) (q + 16);
        }
    }
    __device__ __forceinline__ void place(const int j, mx_i4 & a, int & s) const {
        a = mx_window(v[j], d[j], sh[j]);
        s = (int) ((((uint32_t) v[j].x >> (8 * sh[j])) & 255u) << (8 * j));
    }
};
// acc += one block: the codes A by the digits H, L; the scales are the bytes J of S, of SH and SL
#define MX_MFMA(N, ACC, A, S, J, H, L, SH, SL)                                                                                 \
    ACC = __builtin_amdgcn_mfma_scale_f32_##N##_f8f6f4(mx_op4(A), H, ACC, MX_FP4, MX_FP6, J, S, J, (int) (SH));              \
    ACC = __builtin_amdgcn_mfma_scale_f32_##N##_f8f6f4(mx_op4(A), L, ACC, MX_FP4, MX_FP6, J, S, J, (int) (SL));

// ---- one to a few columns: 16 rows a workgroup, its waves take four steps of 128 values in turn.  The workgroup quantises its columns itself, behind the requests of its first weights (both are
// there before the first product: requests complete in order).  A lane of
// v_mfma_scale_f32_16x16x128: row (column) lane % 16, step lane / 16 of the four.  The weights' bytes bound it, behind the launch (us, with the 4 that a graph of one small launch takes: one column of 14336 x 4096,
// 31 MB, 9.9; of 4096 x 4096 4.8; a token's 4 experts of 2048 x 4096, 18 MB, 6.9).  ONE: a wave has one turn, and no registers for the weights of a second (half as many, twice the waves: 8.7 us)
// ID: blockIdx.y is a column (u + n_used t) of at most 64; the first column of an expert takes all of its expert, the others' workgroups end at once.
static constexpr int MX_VEC_REC = 48;     // LDS bytes of a block of one column: 24 of h, 24 of l
template <bool ID, bool DW, bool ONE> __global__ void __launch_bounds__(512, ONE ? 4 : 2) k_mx_vec(const mx_mm p, const tdesc b, const tdesc ids, const int chunk) {
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ int s_cols[64];
    __shared__ int64_t s_at[64];  // where the workgroup's columns start in b
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, r16 = lane & 15, q = lane >> 4;
    const int row0 = (int) blockIdx.x * 16, all = (p.steps + 3) / 4 * 16;  // blocks of a column, with those behind its last that the last turn takes (zeros)
    int e = 0, n = (int) p.cols;
    if (ID) {
        const int n_used = (int) ids.ne[0], slot = blockIdx.y;
        const int id = lane < n ? *(const int32_t *) (ids.data + (int64_t) (lane % n_used) * ids.nb[0] + (int64_t) (lane / n_used) * ids.nb[1]) : -1;
        e = __builtin_amdgcn_readlane(id, slot);
        if (e < 0 || e >= p.n_expert) return;
        const uint64_t mine = __ballot(id == e);
        if (mine & ((1ull << slot) - 1ull)) return;
        n = __popcll(mine);
        if (wave == 0 && id == e) {
            const int at = __popcll(mine & ((1ull << lane) - 1ull));
            s_cols[at] = lane;
            s_at[at] = ((lane % n_used) % (int) b.ne[1]) * b.nb[1] + (int64_t) (lane / n_used) * b.nb[2];
        }
    } else if ((int) threadIdx.x < n) {
        const uint32_t c = threadIdx.x, n1 = (uint32_t) b.ne[1], n2 = (uint32_t) b.ne[2], c23 = c / n1, c3 = c23 / n2;
        s_at[c] = (int64_t) (c - c23 * n1) * b.nb[1] + (int64_t) (c23 - c3 * n2) * b.nb[2] + (int64_t) c3 * b.nb[3];
    }
    const uint8_t * w = p.w + (int64_t) e * p.nb2 + (int64_t) min(row0 + r16, p.n_rows - 1) * p.nb1;
    uint8_t * s_rec = lds, * s_scale = lds + (size_t) chunk * all * MX_VEC_REC;  // [block][column of the chunk]; [step][column][block] scale bytes
    float * s_part = (float *) (lds + (size_t) chunk * all * (MX_VEC_REC + 1));  // [wave][column][row]
    const float * bias = p.bias ? (const float *) ((const char *) p.bias + (int64_t) e * p.nb_bias) : nullptr;
    for (int c0 = 0; c0 < n; c0 += chunk) {
        const int m = min(chunk, n - c0);
        mx_raw<DW> f0, f1;
        const int last = p.steps - 1, stride = 4 * waves;
        int step = wave * 4 + q;  // (behind the last step: its weights again, and digits of zero)
        f0.load(w, min(step, last), p.blocks);
        if (!ONE && wave * 4 + stride < p.steps) f1.load(w, min(step + stride, last), p.blocks);
        __syncthreads();  // (the columns' places; the last chunk's partial sums and digits are read)
        const int i = threadIdx.x & 3, per = (int) blockDim.x >> 2;  // four lanes a block
        for (int at0 = threadIdx.x >> 2; at0 < m * all; at0 += 2 * per) {
            mx_f4 v[2][2];
            int blk[2], c[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int at = min(at0 + k * per, m * all - 1);
                c[k] = m == 1 ? 0 : at / all;
                blk[k] = at - c[k] * all;
                mx_load8(b.data + s_at[c0 + c[k]] + min(blk[k], p.blocks - 1) * 128, i, v[k]);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (at0 + k * per >= m * all) break;
                if (blk[k] >= p.blocks) v[k][0] = v[k][1] = mx_f4{0, 0, 0, 0};
                uint32_t * rec = (uint32_t *) (s_rec + (blk[k] * chunk + c[k]) * MX_VEC_REC);
                const uint32_t e = mx_act_quad(v[k], i, [&](const int d, const uint32_t h, const uint32_t l) {
                    rec[d] = h;
                    rec[6 + d] = l;
                });
                if (i == 0) s_scale[((blk[k] >> 2) * chunk + c[k]) * 4 + (blk[k] & 3)] = (uint8_t) e;
            }
        }
        __syncthreads();
        mx_f4 acc = {0, 0, 0, 0};
        auto add = [&](const int st, const mx_raw<DW> & f) {
            const int c = min(r16, m - 1);  // (a lane without a column: the last one's digits, for sums that nobody reads)
            const uint32_t sx = *(const uint32_t *) (s_scale + (st * chunk + c) * 4), sl = sx - 0x04040404u;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t * rec = s_rec + ((st * 4 + j) * chunk + c) * MX_VEC_REC;
                const mx_i4 h0 = *(const mx_i4 *) rec, l1 = *(const mx_i4 *) (rec + 32);
                const mx_i2 h1 = *(const mx_i2 *) (rec + 16), l0 = *(const mx_i2 *) (rec + 24);
                const mx_i8 h = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, 0, 0}, l = {l0.x, l0.y, l1.x, l1.y, l1.z, l1.w, 0, 0};
                mx_i4 a;
                int sw;
                f.place(j, a, sw);
                if (j == 0) { MX_MFMA(16x16x128, acc, a, sw, 0, h, l, sx, sl) }
                if (j == 1) { MX_MFMA(16x16x128, acc, a, sw, 1, h, l, sx, sl) }
                if (j == 2) { MX_MFMA(16x16x128, acc, a, sw, 2, h, l, sx, sl) }
                if (j == 3) { MX_MFMA(16x16x128, acc, a, sw, 3, h, l, sx, sl) }
                if (j & 1) __builtin_amdgcn_sched_barrier(0);  // (two blocks' digits at a time: fewer registers)
            }
        };
        if (ONE && wave * 4 < p.steps) add(step, f0);
        for (int s0 = wave * 4; !ONE && s0 < p.steps; s0 += 2 * stride, step += 2 * stride) {  // (s0: the wave's, for all its lanes)
            add(step, f0);
            if (s0 + 2 * stride < p.steps) f0.load(w, min(step + 2 * stride, last), p.blocks);
            if (s0 + stride < p.steps) add(step + stride, f1);
            if (s0 + 3 * stride < p.steps) f1.load(w, min(step + 3 * stride, last), p.blocks);
        }
        if (r16 < m) *(mx_f4 *) (s_part + ((wave * chunk + r16) * 16 + 4 * q)) = acc;
        __syncthreads();
        if ((int) threadIdx.x < 16 * m) {
            const int row = threadIdx.x & 15, c = threadIdx.x >> 4;
            float v = 0.0f;
            for (int k = 0; k < waves; ++k) v += s_part[(k * chunk + c) * 16 + row];
            if (row0 + row < p.n_rows) p.dst[(int64_t) (ID ? s_cols[c0 + c] : c0 + c) * p.ldd + row0 + row] = bias ? v + bias[row0 + row] : v;
        }
    }
}

// ---- a few groups of columns: 32 rows by one group a workgroup, its waves take two steps in turn, everything straight from memory; the waves' sums are added in LDS in their order.  (Two groups a
// workgroup would read the weights once for both; their digits do not fit in registers beside the weights of two turns: 64 columns of 4096 x 4096 22.4 us, 12.2 like this)
template <bool ID, bool DW> __global__ void __launch_bounds__(512) k_mx_few(const mx_mm p) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, r32 = lane & 31, half = lane >> 5;
    const int group = blockIdx.y, row0 = (int) blockIdx.x * 32;
    int e = 0;
    if (ID) {
        if (group >= p.l.total[0]) return;
        e = p.l.owner[group];
    }
    const uint8_t * w = p.w + (int64_t) e * p.nb2 + (int64_t) min(row0 + r32, p.n_rows - 1) * p.nb1;
    const uint8_t * x = p.act + (int64_t) group * p.steps * MX_ACT_STEP;
    const bool live = ID ? p.l.list[group * 32 + r32] >= 0 : (int64_t) group * 32 + r32 < p.cols;  // the lane's column
    mx_f16 acc;
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
    const int last = p.steps - 1, stride = 2 * waves;
    mx_raw<DW> f0, f1;  // the weights of two turns
    mx_i8 h[4], l[4];
    uint32_t sx;
    auto fetch_x = [&](const int step) {
        sx = 0x7F7F7F7Fu;
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = l[j] = mx_i8{0, 0, 0, 0, 0, 0, 0, 0};
        if (live && step <= last) {
            const uint8_t * xs = x + (int64_t) step * MX_ACT_STEP;
            sx = *(const uint32_t *) (xs + 4 * MX_ACT_BLK + r32 * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t * xb = xs + j * MX_ACT_BLK;
                h[j] = mx_op6(*(const mx_i4 *) (xb + r32 * 16), *(const mx_i2 *) (xb + 1024 + r32 * 8));
                l[j] = mx_op6(*(const mx_i4 *) (xb + 512 + r32 * 16), *(const mx_i2 *) (xb + 1280 + r32 * 8));
            }
        }
    };
    int step = wave * 2 + half;
    f0.load(w, min(step, last), p.blocks);
    f1.load(w, min(step + stride, last), p.blocks);
    fetch_x(step);
    auto turn = [&](mx_raw<DW> & f) {
        mx_i4 a[4];
        int sw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) f.place(j, a[j], sw[j]);
        f.load(w, min(step + 2 * stride, last), p.blocks);
        step += stride;
        const uint32_t sl = sx - 0x04040404u;
        MX_MFMA(32x32x64, acc, a[0], sw[0], 0, h[0], l[0], sx, sl)
        MX_MFMA(32x32x64, acc, a[1], sw[1], 1, h[1], l[1], sx, sl)
        MX_MFMA(32x32x64, acc, a[2], sw[2], 2, h[2], l[2], sx, sl)
        MX_MFMA(32x32x64, acc, a[3], sw[3], 3, h[3], l[3], sx, sl)
        fetch_x(step);
    };
    for (int s0 = wave * 2; s0 < p.steps; s0 += stride) {  // (s0: the wave's, for both halves)
        turn(f0);
        if ((s0 += stride) < p.steps) turn(f1);
    }
    // [wave][column][row], the rows of a column 36 apart (of 32: no two quarters of a wave on the same banks)
    float * part_sums = (float *) lds;
#pragma unroll
    for (int i = 0; i < 4; ++i) *(mx_f4 *) (part_sums + (wave * 32 + r32) * 36 + 8 * i + 4 * half) = mx_f4{acc[4 * i], acc[4 * i + 1], acc[4 * i + 2], acc[4 * i + 3]};
    __syncthreads();
    const float * bias = p.bias ? (const float *) ((const char *) p.bias + (int64_t) e * p.nb_bias) : nullptr;
    for (int at = threadIdx.x; at < 32 * 32; at += blockDim.x) {
        const int row = at & 31, cg = at >> 5;
        int64_t c = (int64_t) group * 32 + cg;
        if (ID) c = p.l.list[c];
        else if (c >= p.cols) c = -1;
        if (c < 0 || row0 + row >= p.n_rows) continue;
        float v = 0.0f;
        for (int k = 0; k < waves; ++k) v += part_sums[(k * 32 + cg) * 36 + row];
        p.dst[c * p.ldd + row0 + row] = bias ? v + bias[row0 + row] : v;
    }
}

// Consecutive workgroups go to the eight dies in turn: each die has a run of tiles, four column tiles of a row tile after the other, then the next row tile's; the tiles that a die works on at a time
// so share their digits and their weights in its L2
// (block of blocks, both counted from a multiple of 8)
__device__ __forceinline__ bool mx_tile_of(const mx_mm & p, const int block, const int blocks, const int row_tiles, int & rt, int & tile) {
    const int n_tiles = (int) ((p.cols + 127) / 128), at = (block & 7) * (blocks >> 3) + (block >> 3);
    const int band = at / (row_tiles * 4), in = at - band * row_tiles * 4, width = min(4, n_tiles - 4 * band);
    if (width <= 0) return false;
    rt = in / width;
    tile = 4 * band + in - rt * width;
    return rt < row_tiles;
}
// MUL_MAT_ID: a tile of columns and all of its row tiles to one die, whose L2 then serves its digits; the tiles go to the dies in turn (us, row tiles to the dies in turn | tiles: 2048 tokens of 128 experts,
// 8 each, of 1536 x 2048 187 | 183, 600 of 32, 4 each, of 1024 x 1024 29.2 | 27.5, 1000 of 4096 x 2048 104 | 98, of 2048 x 4096 105 | 106)
__device__ __forceinline__ void mx_id_tile_of(const int row_tiles, int & rt, int & tile) {
    const int at = (int) (blockIdx.x >> 3);
    rt = at % row_tiles;
    tile = at / row_tiles * 8 + (int) (blockIdx.x & 7);
}
// A wave's 32 RT rows by 32 columns to their places, by way of LDS of its own (mx_store_floats): a column's rows lie side by side there and leave in runs of 128 RT bytes, where a lane's own four would
// go out 16 bytes here and there (1000 tokens of 32 experts, rows with a bias, four bytes at a time: 172 us).  The stores leave the result where its reader finds it: past the caches the product alone is up to
// 5 % faster and the product with its reader slower (us, like this | past them: 512 columns of 4096 x 14336 42.4 | 42.2, and an addition to them 68 | 78, a feed-forward block 156 | 160; 300 tokens of 32
// experts of 2048 x 4096, 4 each, 50 | 48, and their rows weighted 62 | 65)
template <int RT> constexpr int mx_store_floats() { return 32 * (32 * RT + 4); }
template <bool ID, int RT> __device__ __forceinline__ void mx_store_tile(const mx_mm & p, const mx_f16 (&acc)[RT], const int group, const int row0, const int e, const int lane, float * lds) {
    constexpr int ROWS = 32 * RT, RUN = ROWS / 4, COLS = 64 / RUN;  // lanes of a column, columns at a time
    const int r32 = lane & 31, half = lane >> 5, row = row0 + lane % RUN * 4;
    int64_t c = (int64_t) group * 32 + r32;
    if (ID) c = p.l.list[c];
    else if (c >= p.cols) c = -1;
    const float * bias = p.bias ? (const float *) ((const char *) p.bias + (int64_t) e * p.nb_bias) : nullptr;
    mx_f4 bv = {0, 0, 0, 0};
    if (bias)
#pragma unroll
        for (int k = 0; k < 4; ++k) bv[k] = bias[min(row + k, p.n_rows - 1)];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) *(mx_f4 *) (lds + r32 * (ROWS + 4) + 32 * t + 8 * i + 4 * half) = mx_f4{acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]};
    __builtin_amdgcn_wave_barrier();
    const bool whole = ((((uintptr_t) p.dst) | (uintptr_t) (p.ldd * 4)) & 15) == 0;
#pragma unroll 4
    for (int c0 = 0; c0 < 32; c0 += COLS) {
        const int cg = c0 + lane / RUN, to = __shfl((int) c, cg, 64);
        mx_f4 v = *(const mx_f4 *) (lds + cg * (ROWS + 4) + lane % RUN * 4);
        if (bias) v += bv;
        if (to < 0) continue;
        float * d = p.dst + to * p.ldd + row;
        if (whole && row + 4 <= p.n_rows) *(mx_f4 *) d = v;
        else
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (row + k < p.n_rows) d[k] = v[k];
    }
}

// ---- many columns: 32 RT rows by four groups of columns a workgroup.  A wave has one group and all rows: its digits come straight from memory (no other wave reads them), the weights through LDS,
// where their blocks are aligned ([block of the step][row] 16 bytes, and 4 scale bytes a row).  In a step of 128 values: the next step's digits are requested, the next step's weights (requested a step
// ago) stored, the weights after those requested — one such item behind each product.  (Requested in a bunch in front of the products they hold up all four waves at once.)  RT = 4 with two workgroups a
// CU beats RT = 8 (us: 1024 / 2048 columns of 2080 x 14336 54 / 97 | 59 / 114, of 4064 x 14336 91 / 168 | 93 / 182)
#define MX_MFMA1(A, B, C, BYTE, SA, SB) __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, C, MX_FP4, MX_FP6, BYTE, SA, BYTE, (int) (SB))
template <bool ID, int RT, bool DW> __global__ void __launch_bounds__(256, 2) k_mx_tile(const mx_mm p, const int row_tiles) {
    constexpr int ROWS = 32 * RT, PLANE = ROWS * 16 + 64;  // (64: the four planes that a quad of lanes writes to lie on different banks)
    constexpr int STAGE = 4 * PLANE + ROWS * 4, OUT = 4 * 4 * mx_store_floats<RT>();
    __shared__ __align__(16) uint8_t lds[2 * STAGE > OUT ? 2 * STAGE : OUT];  // two stages: the planes, their scales
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r32 = lane & 31, half = lane >> 5;
    int rt, tile;
    if (ID) {
        mx_id_tile_of(row_tiles, rt, tile);
    } else {
        if (!mx_tile_of(p, blockIdx.x, gridDim.x, row_tiles, rt, tile)) return;
    }
    const int row0 = rt * ROWS;
    int e = 0, group = tile * 4 + wave, groups = (int) ((p.cols + 31) / 32);
    if (ID) {
        if (tile >= p.l.total[1]) return;
        const int32_t * t = p.l.tiles + 4 * tile;
        e = t[0];
        group = t[1] + wave;
        groups = t[1] + t[2];
    }
    const bool live = group < groups;
    // weights: four lanes a row, its 68 bytes of a step as 64 in a row and one dword; lane q's block starts at byte q of its first dword
    const int q = tid & 3, lrow = tid >> 2;
    const uint8_t * w0 = p.w + (int64_t) e * p.nb2 + (int64_t) row0 * p.nb1;
    const uint32_t odd = DW ? 0u : (uint32_t) (uintptr_t) w0 & 3u;
    w0 -= odd;
    uint32_t wl[RT / 2];
#pragma unroll
    for (int i = 0; i < RT / 2; ++i) wl[i] = (uint32_t) (min(row0 + lrow + 64 * i, p.n_rows - 1) - row0) * (uint32_t) p.nb1 + (DW ? 16u * q : odd);
    mx_i4 wr[RT / 2];
    int wd[RT / 2];
    uint32_t wsh[RT / 2];
    auto fetch_w = [&](const int i, const int step) {
        if (DW) {
            const uint8_t * a = w0 + (int64_t) step * (4 * MX_BLOCK);
            wr[i] = *(const mx_i4_a4 *) (a + wl[i]);
            wd[i] = *(const int *) (a + 64 - 16 * q + wl[i]);
        } else {
            const uint32_t a = wl[i] + (uint32_t) (min(step * 4 + q, p.blocks - 1) * MX_BLOCK);
            wsh[i] = a & 3u;
            wr[i] = *(const mx_i4_a4 *) (w0 + (a & ~3u));
            wd[i] = *(const int *) (w0 + (a & ~3u) + 16);
        }
    };
    auto store_w = [&](const int i, const int buf) {
        const uint32_t sh = DW ? (uint32_t) q : wsh[i];
        const int next = __builtin_amdgcn_update_dpp(0, wr[i].x, 0xF9, 0xF, 0xF, true);  // (the first dword of the quad's next lane: quad_perm 1, 2, 3, 3)
        const int d = !DW || q == 3 ? wd[i] : next;
        *(mx_i4 *) (lds + buf * STAGE + q * PLANE + (lrow + 64 * i) * 16) = mx_window(wr[i], d, sh);
        lds[buf * STAGE + 4 * PLANE + (lrow + 64 * i) * 4 + q] = (uint8_t) ((uint32_t) wr[i].x >> (8 * sh));
    };
    const uint8_t * x = p.act + (int64_t) (live ? group : groups - 1) * p.steps * MX_ACT_STEP;
    const uint32_t x16 = (uint32_t) (half * MX_ACT_BLK + r32 * 16), x8 = (uint32_t) (half * MX_ACT_BLK + r32 * 8);
    mx_i4 h4[2], l4[2], hn4[2], ln4[2];  // the digits of this step and of the next
    mx_i2 h2[2], l2[2], hn2[2], ln2[2];
    uint32_t sx, sxn;
    auto fetch_x = [&](const int n, const int step) {  // the n-th of nine loads
        const uint8_t * xs = x + (int64_t) step * MX_ACT_STEP;
        if (n == 0) sxn = *(const uint32_t *) (xs + 4 * MX_ACT_BLK + r32 * 4);
        const int j = (n - 1) >> 2, what = (n - 1) & 3;
        const uint8_t * xb = xs + 2 * j * MX_ACT_BLK;
        if (n > 0 && what == 0) hn4[j] = *(const mx_i4 *) (xb + x16);
        if (n > 0 && what == 1) hn2[j] = *(const mx_i2 *) (xb + 1024 + x8);
        if (n > 0 && what == 2) ln4[j] = *(const mx_i4 *) (xb + 512 + x16);
        if (n > 0 && what == 3) ln2[j] = *(const mx_i2 *) (xb + 1280 + x8);
    };
    auto take_x = [&]() {
        sx = sxn;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            h4[j] = hn4[j];
            h2[j] = hn2[j];
            l4[j] = ln4[j];
            l2[j] = ln2[j];
        }
    };
    mx_f16 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    const int last = p.steps - 1;
    // the two blocks of a half in turn: an accumulator's next product comes RT instructions later, and the next block's weights are read meanwhile
    auto multiply = [&](const int buf, const int step) {
        constexpr int ITEMS = 9 + 3 * (RT / 2), PER = (ITEMS + 4 * RT - 1) / (4 * RT);
        const int next = min(step + 1, last), after = min(step + 2, last);  // (behind the last step: loads that nobody uses)
        const uint32_t sh = sx >> (8 * half), sl = sh - 0x00040004u;
        auto item = [&](const int n) {
            if (n < 9) fetch_x(n, next);
            else if (n < ITEMS && (n - 9) % 3 == 0) store_w((n - 9) / 3, buf ^ 1);
            else if (n < ITEMS && (n - 9) % 3 == 1) fetch_w((n - 9) / 3, after);
        };
        mx_i4 a[2][RT];
        int sw[2][RT];
        auto read = [&](const int j) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                a[j][t] = *(const mx_i4 *) (lds + buf * STAGE + (2 * j + half) * PLANE + (32 * t + r32) * 16);
                sw[j][t] = (int) (*(const uint32_t *) (lds + buf * STAGE + 4 * PLANE + (32 * t + r32) * 4) >> (8 * half));
            }
        };
        read(0);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (j == 0) read(1);
            const mx_i8 hx = mx_op6(h4[j], h2[j]), lx = mx_op6(l4[j], l2[j]);
#pragma unroll
            for (int u = 0; u < 2 * RT; ++u) {
                const int t = u % RT;
                const mx_i8 wx = mx_op4(a[j][t]);
                if (j == 0) acc[t] = u < RT ? MX_MFMA1(wx, hx, acc[t], 0, sw[j][t], sh) : MX_MFMA1(wx, lx, acc[t], 0, sw[j][t], sl);
                else acc[t] = u < RT ? MX_MFMA1(wx, hx, acc[t], 2, sw[j][t], sh) : MX_MFMA1(wx, lx, acc[t], 2, sw[j][t], sl);
#pragma unroll
                for (int k = 0; k < PER; ++k) item((j * 2 * RT + u) * PER + k);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < RT / 2; ++i) fetch_w(i, 0);
#pragma unroll
    for (int n = 0; n < 9; ++n) fetch_x(n, 0);
#pragma unroll
    for (int i = 0; i < RT / 2; ++i) {
        store_w(i, 0);
        fetch_w(i, min(1, last));
    }
    take_x();
    __syncthreads();
    if (!live) {  // a wave without columns: its share of the weights alone, with the barriers of the others
        for (int step = 0, buf = 0; step < p.steps; ++step, buf ^= 1) {
#pragma unroll
            for (int i = 0; i < RT / 2; ++i) {
                store_w(i, buf ^ 1);
                fetch_w(i, min(step + 2, last));
            }
            __syncthreads();
        }
        return;
    }
    for (int step = 0, buf = 0; step < p.steps; ++step, buf ^= 1) {
        multiply(buf, step);
        take_x();
        __syncthreads();
    }
    // (behind the loop's last barrier: nobody reads the stages any more)
    mx_store_tile<ID, RT>(p, acc, group, row0, e, lane, (float *) lds + wave * mx_store_floats<RT>());
}
// ---- many columns of rows that are whole 16-byte pieces (K a multiple of 512: 272 bytes): as k_mx_tile, but the weights go to LDS by DMA as they lie in memory, 512 values a stage and row by row, and a
// lane moves its codes into place behind its LDS read.  Eight waves: a group of columns has two, which take the even and the odd quarters of a row's stage (68 bytes, four blocks each) and add up at the
// end; the second wave of a SIMD issues while the first one's product runs (one wave alone, eight blocks a stage: 512 columns 46 us).  512 / 1900 columns of 4096 x 14336: 43 / 150 us, 2.8 / 3.0 10^15
// operations a second of the 7.9 that the instruction reaches alone: 3.6 us a stage, of which the matrix pipe works 51 % (2.25 GHz).  Without the DMA a stage takes 2.9 us, without the digits' loads 3.4,
// without both 2.7: 170 KB a stage and CU on the one path from L2 (its address unit works 64 % of the time).  What left the time as it was: rows in LDS 144 bytes apart, without a bank conflict (whole
// rows: half of LDS's cycles), and a product of another tile between the two of a tile.  In a quarter that starts at a unit of 8 bytes (the odd ones: at its
// second half) block i starts at byte i of a unit, and needs the two units behind it: one 16-byte read a block (the unit between two blocks is kept) and up to four byte shifts.
// lane i's 16 bytes at base + off to LDS[lds + 16 i]; base and lds of the wave.  ("memory": the stage's one barrier waits for it by counting the requests behind it, none of which may move in front)
__device__ __forceinline__ void mx_dma16(const uint8_t * base, const uint32_t off, const uint32_t lds) {
    uint32_t keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0" : "=&s"(keep) : "v"(off), "s"(base), "s"(lds) : "memory");
}
template <int RT> constexpr int mx_wide_pieces() { return (32 * RT * 17 + 511) / 512; }  // DMA instructions a wave and stage
template <int RT> struct mx_wide_args {
    const uint8_t * w;    // the tile's first row
    uint32_t first, last; // byte offsets of the lane's pieces of a stage (17 a row, in the order of LDS): its first and its last; the n-th between them is 30 rows and 2 pieces behind the one before,
    int piece;            // one row and no 17 pieces where that leaves the row (piece: of the first)
    uint32_t jump, wrap;
    const uint8_t * x;    // the group's digits
    int stages, wave, lane;
    bool idle;            // a wave without columns
};
// one wave's share of a tile: quarter 2 half + ODD of every stage
template <int RT, int ODD> __device__ __forceinline__ void mx_wide_sum(const mx_wide_args<RT> & p, uint8_t * lds, mx_f16 (&acc)[RT]) {
    constexpr int SET = 1, SETS = RT / SET, PIECES = mx_wide_pieces<RT>(), STAGE = PIECES * 8192, GROUPS = 4 * SETS, SLOTS = 2 * SET;
    const int r32 = p.lane & 31, half = p.lane >> 5;
    const uint32_t lds0 = (uint32_t) (uintptr_t) lds;
    uint32_t first = p.first;
    auto dma = [&](const int n, const int stage, const int buf) {
        const uint32_t off = n == PIECES - 1 ? p.last : first + (uint32_t) n * p.jump + (p.piece >= 17 - 2 * n ? p.wrap : 0u);
        mx_dma16(p.w + (int64_t) stage * 272, off, lds0 + (uint32_t) (buf * STAGE + n * 8192 + p.wave * 1024));
    };
    const uint32_t q = (uint32_t) (half * 2 + ODD) * MX_ACT_STEP, x16 = q + (uint32_t) r32 * 16, x8 = q + (uint32_t) r32 * 8, x4 = q + (uint32_t) r32 * 4;
    const __amdgpu_buffer_rsrc_t digits = __builtin_amdgcn_make_buffer_rsrc((void *) p.x, 0, p.stages * (4 * MX_ACT_STEP), 0x00020000);
    mx_i4 h4[4], l4[4];
    mx_i2 h2[4], l2[4];
    uint32_t sx, sxn;  // the scale bytes of this stage's four blocks and of the next's
    auto fetch_x = [&](const int i, const int what, const int stage) {
        const int at = stage * (4 * MX_ACT_STEP), blk = at + i * MX_ACT_BLK;
        if (what == 0) h4[i] = __builtin_bit_cast(mx_i4, __builtin_amdgcn_raw_buffer_load_b128(digits, (int) x16, blk, 0));
        if (what == 1) h2[i] = __builtin_bit_cast(mx_i2, __builtin_amdgcn_raw_buffer_load_b64(digits, (int) x8, blk + 1024, 0));
        if (what == 2) l4[i] = __builtin_bit_cast(mx_i4, __builtin_amdgcn_raw_buffer_load_b128(digits, (int) x16, blk + 512, 0));
        if (what == 3) l2[i] = __builtin_bit_cast(mx_i2, __builtin_amdgcn_raw_buffer_load_b64(digits, (int) x8, blk + 1280, 0));
        if (what == 3 && i == 0) sxn = (uint32_t) __builtin_amdgcn_raw_buffer_load_b32(digits, (int) x4, at + 4 * MX_ACT_BLK, 0);
    };
    // The stream of groups (a block, SET tiles), GROUPS a stage: group g is multiplied, the codes of g + 1 are moved into place, those of g + 2 read, and what a product's time leaves room for stands
    // behind it.  The one barrier of a stage lies ahead of its last two groups, which already read the next stage: all of this stage's reads are done by then, and the DMA of the next one, in
    // the stage's second quarter, has landed.
    const uint8_t * own = lds + r32 * 272 + half * 136 + ODD * 64;
    mx_i2 kept[RT];       // the unit between a tile's last block and its next
    mx_i4 a[2][SET];      // the two units behind it
    mx_i8 wx[2][SET];     // codes in place
    int sw[2][SET];
    auto read = [&](const int g, const int u, const uint8_t * at) {
        typedef mx_i4 __attribute__((aligned(8))) mx_i4_a8;
        const int t = (g % SETS) * SET + u;
        if (g < SETS) kept[t] = *(const mx_i2 *) (at + t * (32 * 272));
        a[g & 1][u] = *(const mx_i4_a8 *) (at + t * (32 * 272) + 16 * (g / SETS) + 8);
    };
    auto place = [&](const int g, const int u) {
        const int i = g / SETS, t = (g % SETS) * SET + u, k = (i + 1) / 4 + ODD, sh8 = (i + 1) % 4;
        const mx_i4 v = a[g & 1][u];
        const int d[6] = {kept[t].x, kept[t].y, v.x, v.y, v.z, v.w};
        mx_i4 c;
#pragma unroll
        for (int z = 0; z < 4; ++z) c[z] = sh8 ? (int) __builtin_amdgcn_alignbyte(d[k + z + (sh8 ? 1 : 0)], d[k + z], sh8) : d[k + z];
        wx[g & 1][u] = mx_op4(c);
        sw[g & 1][u] = d[ODD];
        kept[t] = mx_i2{v.z, v.w};
    };
#pragma unroll
    for (int n = 0; n < PIECES; ++n) dma(n, 0, 0);
    if (p.idle) {  // its share of the weights alone, with the barriers of the others (1000 tokens of 32 experts: 116 us with products of a neighbour's digits, 107)
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        for (int stage = 0, buf = 0; stage < p.stages; ++stage, buf ^= 1) {
#pragma unroll
            for (int n = 0; n < PIECES; ++n) dma(n, min(stage + 1, p.stages - 1), buf ^ 1);
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            fetch_x(i, k, 0);
            __builtin_amdgcn_sched_barrier(0);  // (in the order of the loop's: the compiler's counts of what is under way then hold for both)
        }
    sx = sxn;
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int u = 0; u < SET; ++u) {
            read(g, u, own);
            if (g == 0) place(0, u);
        }
    for (int stage = 0, buf = 0; stage < p.stages; ++stage, buf ^= 1) {
        const int next = min(stage + 1, p.stages - 1);  // (behind the last stage: loads that nobody uses)
        const uint8_t * at = own + buf * STAGE, * at_next = own + (buf ^ 1) * STAGE;
        asm volatile("" : "+v"(first));  // (the pieces' offsets are made where they are used: kept for the whole loop they leave no room for the digits)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const int i = g / SETS, t0 = (g % SETS) * SET;
            const mx_i8 hx = mx_op6(h4[i], h2[i]), lx = mx_op6(l4[i], l2[i]);
            const uint32_t sh = sx, sl = sh - 0x04040404u;
            // (at least as many requests of digits lie behind the last DMA: those of block 1 and, with four tiles and eight, 2)
            if (g == GROUPS - 2) {
                if (RT == 8) asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                else asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            }
#pragma unroll
            for (int u = 0; u < SLOTS; ++u) {
                const int t = u % SET;
                const mx_i8 dx = u < SET ? hx : lx;
                const uint32_t sd = u < SET ? sh : sl;
                if (i == 0) acc[t0 + t] = MX_MFMA1(wx[g & 1][t], dx, acc[t0 + t], 0, sw[g & 1][t], sd);
                if (i == 1) acc[t0 + t] = MX_MFMA1(wx[g & 1][t], dx, acc[t0 + t], 1, sw[g & 1][t], sd);
                if (i == 2) acc[t0 + t] = MX_MFMA1(wx[g & 1][t], dx, acc[t0 + t], 2, sw[g & 1][t], sd);
                if (i == 3) acc[t0 + t] = MX_MFMA1(wx[g & 1][t], dx, acc[t0 + t], 3, sw[g & 1][t], sd);
                if (u < SET) read((g + 2) % GROUPS, u, g + 2 < GROUPS ? at : at_next);
                else place((g + 1) % GROUPS, u - SET);
                // requests, the n-th slot of block i: the last block's digits in block 0, then the digits of block i - 1 of the next stage, and behind those of block 0 the next stage's
                // weights (together with the last block's digits they hold up both: 2048 columns of 4096 x 16384 190 us, 185 like this)
                constexpr int PER = 8 / RT;
#pragma unroll
                for (int k = 0; k < PER; ++k) {
                    const int n = ((g % SETS) * SLOTS + u) * PER + k;
                    if (i == 0 && n < 4) fetch_x(3, n, stage);
                    if (i >= 1 && n < 4) fetch_x(i - 1, n, next);
                    if (i == 1 && n >= 4 && n - 4 < PIECES) dma(n - 4, next, buf ^ 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        sx = sxn;
    }
}
// where the workgroups of low tiles begin behind `head` row tiles
__host__ __device__ static inline int mx_tail_at(const int head, const int64_t cols) { return (int) ((head * ((cols + 127) / 128) + 7) / 8 * 8); }
template <bool ID, int RT> __device__ __forceinline__ void mx_wide_tile(const mx_mm & p, const int row0, const int tile, uint8_t * lds) {
    constexpr int ROWS = 32 * RT, PIECES = mx_wide_pieces<RT>();
    static_assert(PIECES <= 9, "a lane's pieces leave their row once");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int e = 0, group = tile * 4 + (wave & 3), groups = (int) ((p.cols + 31) / 32);
    if (ID) {
        if (tile >= p.l.total[1]) return;
        const int32_t * t = p.l.tiles + 4 * tile;
        e = t[0];
        group = t[1] + (wave & 3);
        groups = t[1] + t[2];
    }
    mx_wide_args<RT> q;
    q.w = p.w + (int64_t) e * p.nb2 + (int64_t) row0 * p.nb1;
    auto offset = [&](const int c) { return (uint32_t) (c / 17) * (uint32_t) p.nb1 + (uint32_t) (c % 17) * 16u; };
    q.first = offset(tid);
    q.last = offset(min((PIECES - 1) * 512 + tid, ROWS * 17 - 1));
    q.piece = tid % 17;
    q.jump = 30u * (uint32_t) p.nb1 + 32u;
    q.wrap = (uint32_t) p.nb1 - 272u;
    q.x = p.act + (int64_t) min(group, groups - 1) * p.steps * MX_ACT_STEP;
    q.stages = p.steps / 4;
    q.idle = group >= groups;
    q.wave = wave;
    q.lane = lane;
    mx_f16 acc[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    if (wave < 4) mx_wide_sum<RT, 0>(q, lds, acc);
    else mx_wide_sum<RT, 1>(q, lds, acc);
    // the two waves of a group: each passes one half of the tiles to the other and ends with the sum of the other half
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // (no DMA under way, no stage read any more)
    mx_f16 sum[RT / 2];
    mx_f4 * give = (mx_f4 *) lds + (wave * (RT / 2) * 4) * 64 + lane, * take = (mx_f4 *) lds + ((wave ^ 4) * (RT / 2) * 4) * 64 + lane;
#pragma unroll
    for (int t = 0; t < RT / 2; ++t) {
        sum[t] = wave < 4 ? acc[t] : acc[RT / 2 + t];
        const mx_f16 other = wave < 4 ? acc[RT / 2 + t] : acc[t];
#pragma unroll
        for (int i = 0; i < 4; ++i) give[(t * 4 + i) * 64] = mx_f4{other[4 * i], other[4 * i + 1], other[4 * i + 2], other[4 * i + 3]};
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < RT / 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const mx_f4 v = take[(t * 4 + i) * 64];
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[t][4 * i + k] += v[k];
        }
    __syncthreads();
    if (group < groups) mx_store_tile<ID, RT / 2>(p, sum, group, row0 + (wave < 4 ? 0 : ROWS / 2), e, lane, (float *) lds + wave * mx_store_floats<RT / 2>());
}
// (RT = 2: two workgroups a CU, 10 tokens of 32 experts of 2048 x 4096 44 us, one 57.)  The last tile has some of the rows of the one before it, with the same result.  Behind the first `head` row tiles of
// RT = 8 the rows are in tiles of `low` = 128 or 64 rows, in the launch's last workgroups (row_tiles: their number, or head where there are none)
template <bool ID, int RT> __global__ void __launch_bounds__(512, RT == 2 ? 4 : 2) k_mx_wide(const mx_mm p, const int row_tiles, const int head, const int low) {
    extern __shared__ __align__(16) uint8_t lds[];  // two stages of [row] 272 bytes
    int rt, tile;
    if (ID) {
        mx_id_tile_of(row_tiles, rt, tile);
        mx_wide_tile<ID, RT>(p, min(rt * 32 * RT, p.n_rows - 32 * RT), tile, lds);
        return;
    }
    const int first = RT == 8 ? mx_tail_at(head, p.cols) : (int) gridDim.x;
    if ((int) blockIdx.x < first) {
        if (mx_tile_of(p, blockIdx.x, first, RT == 8 ? head : row_tiles, rt, tile)) mx_wide_tile<ID, RT>(p, min(rt * 32 * RT, p.n_rows - 32 * RT), tile, lds);
    } else if (RT == 8) {
        if (!mx_tile_of(p, (int) blockIdx.x - first, (int) gridDim.x - first, row_tiles, rt, tile)) return;
        const int row0 = min(head * 256 + rt * low, p.n_rows - low);
        if (low == 128) mx_wide_tile<ID, 4>(p, row0, tile, lds);
        else mx_wide_tile<ID, 2>(p, row0, tile, lds);
    }
}
static mx_mm mx_args(const tdesc & w, const tdesc & d, int64_t cols) {
    mx_mm p{};
    p.w = (const uint8_t *) w.data;
    p.nb1 = w.nb[1];
    p.nb2 = w.nb[2];
    p.n_rows = (int) w.ne[1];
    p.n_expert = (int) w.ne[2];
    p.blocks = (int) (w.ne[0] / 32);
    p.steps = (int) mx_steps(w.ne[0]);
    p.dst = (float *) d.data;
    p.ldd = w.ne[1];
    p.cols = cols;
    return p;
}
// k_mx_vec: columns quantised at a time (0: a column does not fit); waves: one turn where eight make it one, and eight where the workgroups alone do not fill the GPU (us, four waves | eight: a column of
// 4096 x 4096, 256 workgroups, 5.2 | 4.5, of 2048 x 5632, 352 workgroups, one turn in both, 4.0 | 4.5, of 2048 x 32000 8.5 | 12.0, of 4096 x 14336 11.1 | 9.8; 5 columns of 2080 x 1001 7.7 | 6.2)
static constexpr size_t MX_VEC_LDS = 60 << 10;
static int mx_vec_waves(int64_t K, int64_t N, int64_t slots) { return (int) std::min<int64_t>(8, std::max<int64_t>((N + 15) / 16 * slots <= 256 ? 8 : 4, (mx_steps(K) + 3) / 4)); }
static size_t mx_vec_lds(int64_t K, int64_t cols) { return (size_t) cols * (size_t) ((mx_steps(K) + 3) / 4 * 16 * (MX_VEC_REC + 1)) + (size_t) (8 * cols * 16 * 4); }
static int mx_vec_chunk(int64_t K, int64_t cols) {
    int64_t c = std::min<int64_t>(16, cols);
    while (c > 0 && mx_vec_lds(K, c) > MX_VEC_LDS) --c;
    return (int) c;
}
// Every workgroup quantises its columns: a launch less (two with MUL_MAT_ID), for work that grows with columns and rows.  us, k_mx_vec | the faster of the others: 2 / 3 columns of 4096 x 14336 11.5 / 14.2 |
// 13.7, 2 of 14336 x 4096 12.9 | 20.1, 4 / 8 of 4096 x 4096 6.5 / 9.4 | 11.7, 8 / 12 of 2048 x 5632 8.9 / 11.2 | 9.0, 6 / 8 of 2080 x 5000 9.8 / 12.0 | 10.6, 16 of 1024 x 1024 6.2 | 7.9; expert columns,
// 16 / 24 of 32 experts of 2048 x 4096 23.0 / 29.1 | 25.7 / 26.1, of 4096 x 4096 32.8 / 41.4 | 35.6 / 38.8, 64 of 1024 x 1024 9.7 | 14.2, of 128 experts of 2048 x 768 18.5 | 21.7
bool mx_vec_takes(int64_t K, int64_t N, int64_t cols) {
    return (cols == 1 || (cols <= 16 && cols * K * N <= 150000000 && cols * K <= 4096 * mx_vec_waves(K, N, 1))) && mx_vec_chunk(K, cols) >= cols;
}
bool mx_id_vec_takes(int64_t K, int64_t N, int64_t cols) { return (cols <= 16 || (cols <= 64 && cols * K * N <= 110000000)) && mx_vec_chunk(K, cols) >= 1; }
// rows of whole steps, every one at a whole dword
static bool mx_dwords(const mx_mm & p) { return p.blocks % 4 == 0 && p.nb1 % 4 == 0 && p.nb2 % 4 == 0 && ((uintptr_t) p.w & 3) == 0; }
// ... of whole 16-byte pieces
static bool mx_pieces(const mx_mm & p) { return p.blocks % 16 == 0 && p.nb1 % 16 == 0 && p.nb2 % 16 == 0 && ((uintptr_t) p.w & 15) == 0 && p.nb1 <= (1 << 22); }

static void mx_launch_vec(hipStream_t s, const mx_mm & p, const tdesc & b, const tdesc * ids) {
    const int64_t K = b.ne[0];
    const int chunk = mx_vec_chunk(K, p.cols);
    const dim3 block((unsigned) (64 * mx_vec_waves(K, p.n_rows, ids ? p.cols : 1)));
    const unsigned rows = (unsigned) ((p.n_rows + 15) / 16);
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(rows, ids ? (unsigned) p.cols : 1u), block, mx_vec_lds(K, chunk), s, p, b, ids ? *ids : b, chunk); };
    const bool dw = mx_dwords(p), one = p.steps <= (int) block.x / 64 * 4;
    if (ids) one ? (dw ? go(k_mx_vec<true, true, true>) : go(k_mx_vec<true, false, true>)) : dw ? go(k_mx_vec<true, true, false>) : go(k_mx_vec<true, false, false>);
    else one ? (dw ? go(k_mx_vec<false, true, true>) : go(k_mx_vec<false, false, true>)) : dw ? go(k_mx_vec<false, true, false>) : go(k_mx_vec<false, false, false>);
}
// Costs of a product by k_mx_few and in tiles of 32 rt rows, in quarters of a us at 4096 values a row: 256 workgroups at a time, a tile's by its groups of columns.  What they compare, us, k_mx_few | tiles of 64
// rows: 32 columns of 4096 x 14336 18.9 | 14.4, of 4096 x 32000 30.5 | 19.0, of 14336 x 8192 23.5 | 28.3, 64 of 4096 x 4096 12.2 | 14.4, 128 18.0 | 19.8, 256 29.8 | 21.3; 4 / 18 columns an expert, 32 experts
// of 2048 x 4096 49 / 87 | 35 / 59.  (k_mx_tile's tiles of 64 rows take longer, which these costs leave out: 256 columns of 4224 x 2080 24.3 | 29.6.)  Tiles of 64 | 128 | 256 rows: 256 columns of
// 4096 x 14336 32.5 | 28.6 | 34.8, 384 46.1 | 48.5 | 38.7
static int64_t mx_few_cost(int64_t N, int64_t groups) { return ((N + 31) / 32 * groups + 255) / 256 * 22; }
static int64_t mx_tile_cost(int rt, int64_t N, int64_t tiles, int64_t groups) {
    const int64_t rounds = ((N + 32 * rt - 1) / (32 * rt) * tiles + 255) / 256, g = std::min<int64_t>(groups, 4);
    return rounds * (rt == 2 ? 20 + 9 * g : rt == 4 ? 47 + 11 * g : 70 + 17 * g);
}
// A product in tiles of 256 rows whose last round of 256 workgroups is far from full: that round's rows in lower tiles where it ends earlier by the costs above.  -> the cost; low: their height (0: none), head:
// the row tiles in front of them.  us, without | with: 640 columns of 4096 x 14336 75.6 | 61.5, 768 75.7 | 67.4, 1900 (840 tiles, or 765 and 150 of
// 128 rows) 158 | 153, 2048 of 4096 x 5632 79.4 | 70.7, 2200 of 14336 x 4096 216 | 190
static int64_t mx_tail(int64_t N, int64_t tiles, int & head, int & low) {
    const int64_t all = (N + 255) / 256, whole = all * tiles / 256, full = std::min(all, whole * 256 / tiles), idle = whole * 256 - full * tiles, c8 = mx_tile_cost(8, N, tiles, 4);
    head = (int) all;
    low = 0;
    if (whole == 0 || full == all) return c8;
    auto cost = [&](int rt) { return whole * mx_tile_cost(8, 1, 1, 4) + (std::max<int64_t>(0, (N - 256 * full + 32 * rt - 1) / (32 * rt) * tiles - idle) + 255) / 256 * mx_tile_cost(rt, 1, 1, 4); };
    const int64_t c4 = cost(4), c2 = cost(2);
    if (c8 <= std::min(c4, c2)) return c8;
    head = (int) full;
    low = c2 < c4 ? 64 : 128;
    return std::min(c4, c2);
}
template <bool ID, int RT> static void mx_launch_tile_of(hipStream_t s, const mx_mm & p, int64_t col_tiles) {
    const int row_tiles = (p.n_rows + 32 * RT - 1) / (32 * RT);
    const dim3 grid((unsigned) (ID ? (col_tiles + 7) / 8 * 8 * row_tiles : (row_tiles * col_tiles + 7) / 8 * 8));
    if (mx_pieces(p) && p.n_rows >= 32 * RT) {
        constexpr size_t lds = std::max<size_t>(2 * mx_wide_pieces<RT>() * 8192, 8 * 4 * mx_store_floats<RT / 2>());
        static std::atomic<uint32_t> done{0};
        if (ensure_dyn_lds((const void *) k_mx_wide<ID, RT>, lds, done)) {
            int head = row_tiles, low = 0;
            if (!ID && RT == 8) mx_tail(p.n_rows, col_tiles, head, low);
            const int tail = low ? (p.n_rows - 256 * head + low - 1) / low : 0;
            if (low) hipLaunchKernelGGL((k_mx_wide<ID, RT>), dim3((unsigned) (mx_tail_at(head, p.cols) + (tail * col_tiles + 7) / 8 * 8)), dim3(512), lds, s, p, tail, head, low);
            else hipLaunchKernelGGL((k_mx_wide<ID, RT>), grid, dim3(512), lds, s, p, row_tiles, head, 0);
            return;
        }
    }
    if constexpr (RT < 8) {
        if (mx_dwords(p)) hipLaunchKernelGGL((k_mx_tile<ID, RT, true>), grid, dim3(256), 0, s, p, row_tiles);
        else hipLaunchKernelGGL((k_mx_tile<ID, RT, false>), grid, dim3(256), 0, s, p, row_tiles);
    } else mx_launch_tile_of<ID, 4>(s, p, col_tiles);
}
template <bool ID> static void mx_launch_tile(hipStream_t s, const mx_mm & p, int64_t tiles, int rt) {
    if (rt == 8) mx_launch_tile_of<ID, 8>(s, p, tiles);
    else if (rt == 4) mx_launch_tile_of<ID, 4>(s, p, tiles);
    else mx_launch_tile_of<ID, 2>(s, p, tiles);
}
// Rows of a tile, in units of 32, among the heights that there is a kernel for: of rows in whole pieces 64, 128 and 256 where the matrix has as many (k_mx_wide, the costs above); of others 64 and 128
// (k_mx_tile): 128 from 512 tiles of 64 on, two a CU, or 2200 of experts with few columns each (`each`).  us, tiles of 64 | 128 rows: 384 / 1024 / 2048 columns of 2080 x 14336 29.4 / 62.7 / 124 |
// 27.4 / 53.6 / 98, 512 / 1024 / 2048 of 4064 x 4096 31.9 / 39.7 / 69 | 35.0 / 36.5 / 55, 1024 of 4224 x 2080 34.2 | 36.5; 2, 15 / 62 columns an expert, 32 experts of 2080 x 2080 25.5, 38.4 / 53.2 |
// 27.5, 39.6 / 49.9, of 1056 x 4096 25.9, 34.8 / 46.2 | 29.2, 34.1 / 46.0, 15 of 128 experts of 2080 x 2080 123 | 113
static int mx_tile_rows(const mx_mm & p, int64_t tiles, int64_t groups, int64_t each, bool tail) {
    const int64_t N = p.n_rows;
    if (!mx_pieces(p)) return N > 64 && (N + 63) / 64 * tiles >= (each >= 48 ? 512 : 2200) ? 4 : 2;
    int head, low;
    const int64_t never = INT64_MAX, c2 = mx_tile_cost(2, N, tiles, groups), c4 = N >= 128 ? mx_tile_cost(4, N, tiles, groups) : never;
    const int64_t c8 = N < 256 ? never : tail && groups >= 4 ? mx_tail(N, tiles, head, low) : mx_tile_cost(8, N, tiles, groups);
    return c8 <= c4 && c8 <= c2 ? 8 : c4 <= c2 ? 4 : 2;
}
// Four waves where the rows and groups alone fill the GPU, eight where they do not (us for 8 / 32 columns, four waves | eight: 4096 rows of 14336 19.7 / 22.0 | 20.2 / 22.1, 14336 of 4096 17.5 / 18.9 |
// 20.3 / 21.4; 10 / 125 tokens of 32 experts of 4096 x 2048 37.6 / 75.8 | 47.6 / 93.3)
template <bool ID> static void mx_launch_few(hipStream_t s, const mx_mm & p, int64_t groups) {
    const int waves = (p.n_rows + 31) / 32 * groups < 256 ? 8 : 4;
    const dim3 grid((unsigned) ((p.n_rows + 31) / 32), (unsigned) groups), block((unsigned) (64 * waves));
    const size_t lds = (size_t) waves * 32 * 36 * 4;
    if (mx_dwords(p)) hipLaunchKernelGGL((k_mx_few<ID, true>), grid, block, lds, s, p);
    else hipLaunchKernelGGL((k_mx_few<ID, false>), grid, block, lds, s, p);
}
// the tiles' rows in units of 32, or 0: k_mx_few
static int mx_form(const mx_mm & p) {
    const int64_t groups = (p.cols + 31) / 32, tiles = (p.cols + 127) / 128;
    return mx_few_cost(p.n_rows, groups) < mx_tile_cost(2, p.n_rows, tiles, groups) ? 0 : mx_tile_rows(p, tiles, groups, p.cols, mx_pieces(p));
}
// With fewer than 64 columns an expert the weights' way from memory counts for more than the products: of rows in whole pieces tiles of 256 rows where there are two rounds of them, of 64 (two workgroups a CU)
// elsewhere.  us, 64 | 256 rows, 10 / 28 columns an expert: 32 experts of 2048 x 4096 48 / 71 | 46 / 57, of 1024 x 1024 16.8 / 20.4 | 21.1 / 23.8, 128 of 2048 x 768 40 / 53 | 48 / 57
static int mx_id_form(const mx_mm & p) {
    const int64_t g = mx_id_groups(p.n_expert, p.cols), tiles = mx_id_tiles(p.n_expert, p.cols), each = p.cols / p.n_expert;
    if (mx_few_cost(p.n_rows, g) < mx_tile_cost(2, p.n_rows, tiles, each / 32 + 1)) return 0;
    if (each >= 64 || !mx_pieces(p)) return mx_tile_rows(p, tiles, 4, each, false);
    return each >= 16 && p.n_rows / 256 * tiles >= 512 ? 8 : 2;
}
int mx_tile_rows_of(int64_t K, int64_t N, int64_t n_expert, int64_t cols) {
    mx_mm p{};
    p.blocks = (int) (K / 32);
    p.nb1 = K / 32 * MX_BLOCK;
    p.nb2 = p.nb1 * N;
    p.n_rows = (int) N;
    p.n_expert = (int) n_expert;
    p.cols = cols;
    if (n_expert ? mx_id_vec_takes(K, N, cols) : mx_vec_takes(K, N, cols)) return 0;
    return 32 * (n_expert ? mx_id_form(p) : mx_form(p));
}
// act: null where mx_vec_takes
void launch_mx_mul_mat(hipStream_t s, const tdesc & w, const tdesc & b, const tdesc & d, const void * act) {
    mx_mm p = mx_args(w, d, b.ne[1] * b.ne[2] * b.ne[3]);
    p.act = (const uint8_t *) act;
    if (p.n_rows == 0 || p.cols == 0) return;
    if (!act) return mx_launch_vec(s, p, b, nullptr);
    if (const int rt = mx_form(p)) mx_launch_tile<false>(s, p, (p.cols + 127) / 128, rt);
    else mx_launch_few<false>(s, p, (p.cols + 31) / 32);
}
void launch_mx_mul_mat_id(hipStream_t s, const tdesc & w, const tdesc & b, const tdesc & ids, const tdesc & d, const void * ws, const float * bias, int64_t nb_bias) {
    const int64_t cols = ids.ne[0] * ids.ne[1], g = mx_id_groups(w.ne[2], cols);
    mx_mm p = mx_args(w, d, cols);
    p.bias = bias;
    p.nb_bias = nb_bias;
    if (p.n_rows == 0 || g == 0) return;
    if (!ws) return mx_launch_vec(s, p, b, &ids);
    p.act = (const uint8_t *) ws + mx_lists_bytes(g);
    p.l = mx_lists_at((void *) ws, g);
    if (const int rt = mx_id_form(p)) mx_launch_tile<true>(s, p, mx_id_tiles(w.ne[2], cols), rt);
    else mx_launch_few<true>(s, p, g);
}
// Which operands the products take (type and shape; the rows of both are dense, whole blocks).  The kernels hold offsets inside a tile of 256 rows and inside a group's digits in 32 bits, and a launch less than
// 2^32 threads in x
static constexpr int64_t MX_MAX_ROW = 1 << 23;  // bytes between rows
static bool mx_grid_ok(int64_t N, int64_t tiles) { return N < (1 << 26) && (N + 63) / 64 * (tiles + 7) < (1 << 22); }
bool mx_product_ok(const tdesc & w, const tdesc & b) {
    const int64_t cols = b.ne[1] * b.ne[2] * b.ne[3];
    return w.ne[0] % 32 == 0 && w.ne[0] > 0 && w.nb[0] == MX_BLOCK && w.ne[0] / 32 * MX_BLOCK <= MX_MAX_ROW && (int64_t) w.nb[1] <= MX_MAX_ROW && b.nb[0] == 4 && b.nb[1] % 4 == 0 && b.nb[2] % 4 == 0 &&
           b.nb[3] % 4 == 0 && (cols + 31) / 32 <= 65535 && mx_grid_ok(w.ne[1], (cols + 127) / 128);
}
bool mx_id_ok(const tdesc & w, const tdesc & ids) {
    const int64_t cols = ids.ne[0] * ids.ne[1];
    return w.ne[2] > 0 && w.ne[2] <= MX_MAX_EXPERTS && ids.nb[0] % 4 == 0 && ids.nb[1] % 4 == 0 && ids.ne[0] > 0 && ids.ne[2] == 1 && ids.ne[3] == 1 && cols < ((int64_t) 1 << 30) &&
           mx_id_groups(w.ne[2], cols) <= 65535 && mx_grid_ok(w.ne[1], mx_id_tiles(w.ne[2], cols));
}

// ------------------------------------------------------------------------------------------------ ADD_ID
// a [N, n_used, T] + the row of b [N, n_expert] that ids [n_used, T] names (an id outside them: a's row alone).  Bytes bound it behind the launch: 1000 tokens of 4 rows of 4096 32 us, 4.1 TB/s
__global__ void __launch_bounds__(256) k_add_id(const tdesc a, const tdesc b, const tdesc ids, const tdesc d) {
    const int64_t u = blockIdx.y, t = blockIdx.z, n = (int64_t) blockIdx.x * 256 + threadIdx.x;
    if (n >= a.ne[0]) return;
    const int32_t e = *(const int32_t *) (ids.data + u * ids.nb[0] + t * ids.nb[1]);
    float v = *(const float *) (a.data + n * 4 + u * a.nb[1] + t * a.nb[2]);
    if (e >= 0 && e < b.ne[1]) v += *(const float *) (b.data + n * 4 + (int64_t) e * b.nb[1]);
    *(float *) (d.data + n * 4 + u * d.nb[1] + t * d.nb[2]) = v;
}
void launch_add_id(hipStream_t s, const tdesc & a, const tdesc & b, const tdesc & ids, const tdesc & d) {
    if (a.ne[0] * a.ne[1] * a.ne[2] == 0) return;
    hipLaunchKernelGGL(k_add_id, dim3((unsigned) ((a.ne[0] + 255) / 256), (unsigned) a.ne[1], (unsigned) a.ne[2]), dim3(256), 0, s, a, b, ids, d);
}

MI_TU_TOUCH(mx)

}  // namespace mi355x
