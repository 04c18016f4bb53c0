// Grouped-query attention of the newest token(s) over a KV cache held in 4 bits (u4.cuh).
//
// The reference has no cache; the definition is its attention (src/demo.cu:28-70) over the values
// K^ = z + s c, V^ = z + s c of the cache, for query rows that see the keys up to their own position.
//
// Mathematics.  With codes c in 0..15 and a (scale s, offset z) for each 64 elements of a key (group g of the row):
//     S = scale * sum_g [ s_g sum_d q_d (c_d - 8) + (z_g + 8 s_g) sum_d q_d ]
//     O = sum_k P_k V^_k  with  V^_k = s_kg (c_kd - 8) + (z_kg + 8 s_kg)
//       = 2^E sum_k [P_k s_kg 2^-E] (c_kd - 8)  +  sum_k P_k (z_kg + 8 s_kg)
// The sums over d and over k with c run on the tensor core: c - 8 is a whole number, exact in both 16-bit types, q is
// the caller's 16-bit q, and the bracket is rounded to fp16, the one rounding on the way to O (2^-11 of a term, half
// a step; 2^E follows the scales of a warp's tile up and down, so that no bracket leaves fp16; beside one whose scale is 2^18 times its
// own a key of the same tile gets fp16's last digits, 2^-26 of the largest scale at most).  Everything else is held in 32 bits.
//
// What bounds it.  With a few query rows a key (T * group) HBM does: 4.5 bits an element.  The codes must be unpacked
// between memory and tensor core, and the registers are where that costs no second trip through shared memory;
// tcgen05.mma takes no operand from registers, and unpacked keys in shared memory would be 4 times the bytes that
// came in, written and read back.  So the products are mma.sync m16n8k16 with the unpacked codes as the register operand A:
// keys are the rows of S^T = K Q^T, head elements the rows of O^T = V^T P^T, and a query row takes one of 8 columns.
//
// Work split.  All (sequence, KV head, row block) items are laid out one after the other in tiles of 64 or 32 keys, and
// the resulting line is cut into equal parts, one for each warp of the GPU, whatever the lengths of the sequences: a warp may
// finish one item, do several and begin the next.  A warp streams its tiles through a ring of its own and meets the others
// only once, at the end, where the CTA merges what its warps have of the same item.  Items that lie in several CTAs go
// through the workspace and a second small kernel.  Short jobs are done in one launch instead: a cluster of up to 8 CTAs an
// item, which merges through distributed shared memory (plan.cluster says when).
//
// Measured (f16, 4 query heads a KV head, D = 128, a call in a graph): B=32 Hkv=8 Skv=16384 127 us, 4.8 TB/s (loads alone 104; unpacking K and V
// takes the rest: instructions that wait for one another with two warps a scheduler, slots 50 % used); B=16 Skv=4096 21.5; B=1 Skv=2048
// 7.4; 16 query rows B=32 Skv=16384 198.
#include <atomic>
#include <cmath>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "fast_div.h"
#include "host_common.h"
#include "ptx.cuh"
#include "u4.cuh"

namespace fa {
namespace {

constexpr int kWarps = 8;
constexpr int kMaxCluster = 8;                 // portable cluster size
// Keys of a tile.  The longer one has a third fewer instructions a key besides the products and twice the independent ones
// to fill a product's latency with (B=32 Hkv=8 Skv=16384: 149 us with 32, 126 with 64); with two columns of 8 rows there are
// enough of those, and no registers.
constexpr int tile_keys(int nt) { return nt == 1 ? 64 : 32; }
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kClusterTiles = 1;               // see make_plan
constexpr int kManyRows = 96, kManyRowsF16 = 128, kManyKeys = 512;    // see many_rows
constexpr size_t kCopyBytes = 256u << 20;      // of K and V in fp16 (and their remainders) at a time
constexpr float kScaleRange = 0x1p-12f;        // V's scales may fall this far below what 2^E allows before E follows them
constexpr float kGrow = 8.0f;                  // a running max may be exceeded by this much (in powers of two) before it is raised

struct U4Args {
    CUtensorMap tk, tv;                        // codes: (bytes of a row, rows of a block, KV heads, blocks), boxes of a tile's rows or a page's
    const uint16_t* q;
    const __half2 *kp, *vp;
    uint16_t* o;
    float* lse;
    float* scratch;                            // head records of the warps, then two records a CTA
    int* status;
    int2* meta;                                // per CTA: item that begins in it and goes on (or -1), one past the last CTA of that item
    long long p_block_stride, p_head_stride, p_row_stride;    // pairs
    CacheMap map;
    const int* seq_lens;
    int batch, hq, hkv, group, n_tok, rows, row_blocks, kv_len;
    int cluster;                               // CTAs of an item's cluster; 0: the line
    int box_shift;                             // rows of a TMA box: a tile's, or a page's
    FastDiv by_group, by_row_blocks, by_hkv, by_cluster;
    float scale_log2;
};

// Output row of query row r of a (sequence, KV head): token r / group, head r % group of the group.
__device__ __forceinline__ long long out_row(const U4Args& a, int b, int h, int r) {
    const int tok = a.by_group.quot(r);
    return ((long long)b * a.n_tok + tok) * a.hq + (long long)h * a.group + (r - tok * a.group);
}

// Shapes of an instance: D, row columns of 8.
template <int D, int NT>
struct Shape {
    static constexpr int G = D / kU4Group;                     // groups of a row
    static constexpr int Keys = tile_keys(NT), J = Keys / 16;  // of a tile, and its 16-key steps
    static constexpr int RowBytes = D / 2;
    static constexpr int Stages = 3;
    static constexpr int CodeBytes = Keys * RowBytes;
    static constexpr int StageBytes = 2 * CodeBytes;
    static constexpr int FactorBytes = Keys * G * 16;         // of a tile: for each key K's (scale, offset) and V's, unpacked
    static constexpr int WarpBytes = Stages * StageBytes + FactorBytes;
    static constexpr int Rows = 8 * NT;
    // the rings, aligned, and a cluster's rows: from each of its CTAs up to Rows / size of them (rounded up), O [D], max, sum
    static constexpr int SmemBytes = 1024 + kWarps * WarpBytes + (Rows + kMaxCluster - 1) * (D + 4) * 4;
    static constexpr int Record = Rows * (D + 2);              // floats: O [row][D], then m [row], l [row]
    static_assert(Record * 4 <= WarpBytes, "a record fits the ring it replaces");
};

// Two at a time: d = a b - c, a += b.
__device__ __forceinline__ void fma2(float (&d)[2], const float* a, const float (&b)[2], const float (&c)[2]) {
    asm("{\n\t.reg .b64 x, y, z, r;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 r, x, y, z;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "=f"(d[0]), "=f"(d[1]) : "f"(a[0]), "f"(a[1]), "f"(b[0]), "f"(b[1]), "f"(-c[0]), "f"(-c[1]));
}
__device__ __forceinline__ void add2(float (&a)[2], const float (&b)[2]) {
    asm("{\n\t.reg .b64 x, y, r;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tadd.rn.f32x2 r, x, y;\n\tmov.b64 {%0, %1}, r;\n\t}"
        : "+f"(a[0]), "+f"(a[1]) : "f"(b[0]), "f"(b[1]));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Four floats (G = 2) or two.
template <int G>
__device__ __forceinline__ void lds_factors(uint32_t a, float (&f)[2 * G]) {
    if constexpr (G == 2) asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f[0]), "=f"(f[1]), "=f"(f[2 * G - 2]), "=f"(f[2 * G - 1]) : "r"(a));
    else asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(f[0]), "=f"(f[1]) : "r"(a));
}
template <int G>
__device__ __forceinline__ void sts_factors(uint32_t a, const float (&f)[2 * G]) {
    if constexpr (G == 2) asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(a), "f"(f[0]), "f"(f[1]), "f"(f[2 * G - 2]), "f"(f[2 * G - 1]) : "memory");
    else asm volatile("st.shared.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(f[0]), "f"(f[1]) : "memory");
}
// The pairs of a key.
template <int G>
__device__ __forceinline__ void ldg_pairs(const __half2* p, uint32_t (&u)[G]) {
    if constexpr (G == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        u[0] = x.x;
        u[G - 1] = x.y;
    } else {
        u[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
// Four 8 x 8 tiles of 16-bit values, whose rows the lanes' addresses name (8 lanes a tile); TRANS: by columns.
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&r)[4]) {
    if constexpr (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}

// D = A B + C, m16n8k16, fp16 operands, fp32 accumulation.
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same with C the same in both halves of the rows: c0 in the first column of a thread, c1 in the second.
__device__ __forceinline__ void mma_from(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
// An 8 x 8 tile of 16-bit values, rows to columns, across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t hadd2(uint32_t x, float y) {
    const __half2 z = __hadd2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(y));
    return *reinterpret_cast<const uint32_t*>(&z);
}

// Nibble N (0..3) of both halves of a word as code + BIAS in fp16.  A nibble in bits 0-3 of the mantissa of 1024.0 is
// 1024 + code, one in bits 4-7 of that of 64.0 is 64 + code: a logic instruction each, the word shifted once for
// nibbles 2 and 3, and an exact addition where the bias wanted is another.  (Shifting every nibble to the same place costs
// three shifts a word on the integer pipe, which runs at half the rate and was the kernel's limit.)
template <int N, int BIAS>
__device__ __forceinline__ uint32_t code16(uint32_t x) {
    constexpr bool odd = N & 1;
    const uint32_t y = N < 2 ? x : x >> 8;
    // (y & mask) | one as one instruction, which takes one of the two constants from a register
    uint32_t c;
    if constexpr (odd) asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(c) : "r"(y), "n"(0x00F000F0), "r"(0x54005400));
    else asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(c) : "r"(y), "n"(0x000F000F), "r"(0x64006400));
    return (odd ? 64 : 1024) == BIAS ? c : hadd2(c, (float)(BIAS - (odd ? 64 : 1024)));
}

// The 16-byte piece of row r in which piece c of the row lies: the exchange of TMA's 64-byte (d_head 128) and 32-byte swizzle,
// under which the eight rows of a tile of ldmatrix touch every bank once.
template <int D>
__device__ __forceinline__ int piece(int r, int c) { return D == 128 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1); }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Four floats to where CTA `rank` of the cluster has this CTA's shared address `p`.
__device__ __forceinline__ void st_cluster4(const float* p, int rank, const float4& x) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(x.x), "f"(x.y), "f"(x.z), "f"(x.w) : "memory");
}

// Weight of a record (its max in powers of two, its sum) in a merge with maximum `mx`: none if it is empty; a NaN sum without a
// max is kept.
__device__ __forceinline__ float record_weight(float m, float l, float mx) { return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : ex2(m - mx); }

__device__ __forceinline__ void add_record(float4& f, float& sum, float m, float l, float mx, const float* o) {
    const float w = record_weight(m, l, mx);
    const float4 z = *reinterpret_cast<const float4*>(o);
    sum = fmaf(w, l, sum);
    f.x = fmaf(w, z.x, f.x); f.y = fmaf(w, z.y, f.y); f.z = fmaf(w, z.z, f.z); f.w = fmaf(w, z.w, f.w);
}

// Four elements of an output row from its sums, and the row's LSE with the first of them.
template <int D, bool BF16>
__device__ __forceinline__ void store_quad(const U4Args& a, long long row, int d, const float4& f, float m, float l) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    *reinterpret_cast<uint2*>(a.o + row * D + d) = make_uint2(pack16<BF16>(f.x * inv, f.y * inv), pack16<BF16>(f.z * inv, f.w * inv));
    if (d == 0 && a.lse != nullptr) a.lse[row] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
}

struct Item {
    int b, h, rb, len, tiles;      // sequence, KV head, row block, its keys, tiles of them (at least one)
};
template <int KEYS>
__device__ __forceinline__ int tiles_of(int len) { return max(1, (len + KEYS - 1) / KEYS); }

template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(kWarps * 32, 1) u4_kernel(const __grid_constant__ U4Args a) {
    using S = Shape<D, NT>;
    constexpr int G = S::G;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);      // the swizzle goes by the address
    constexpr int kRecords = 2 * kWarps;                       // of a CTA, in the order of the line: head and tail of warp 0, of warp 1, ...
    __shared__ __align__(8) uint64_t s_full[kWarps][S::Stages];
    __shared__ int s_abort, s_never;
    __shared__ int s_prefix[kWarps * 32], s_warp[kWarps];      // tiles (of one head and row block) before a thread's sequences
    __shared__ int s_len[kWarps * 32];                         // keys of the last of them
    __shared__ int s_item[kRecords], s_before[kWarps], s_after[kWarps];
    __shared__ float s_m[kRecords][S::Rows], s_l[kRecords][S::Rows];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    if (tid == 0) {
        prefetch_tensormap(&a.tk);
        prefetch_tensormap(&a.tv);
        s_abort = s_never = 0;
        for (int i = 0; i < kWarps * S::Stages; i++) mbar_init(smem_u32(&s_full[0][0] + i), 1);
        fence_mbar_init();
    }
    const WaitCtl ctl{&s_abort, a.status};
    if (a.cluster > 1) cluster_arrive();                       // waited for before the first access to another CTA
    grid_dependency_wait();
    grid_launch_dependents();

    // ---- this warp's part of the line, and the item that it begins in
    const int per_b = a.hkv * a.row_blocks;                    // items of a sequence
    Item it{0, 0, 0, 0, 0};
    int item_start = 0, chunk = 0, rank = 0;
    int c_begin, c_end, w_begin, w_end;
    if (a.cluster > 0) {                                       // an item of its own: the line is that item
        const int item = a.by_cluster.quot(blockIdx.x), bh = a.by_row_blocks.quot(item);
        rank = blockIdx.x - item * a.cluster;
        it.rb = item - bh * a.row_blocks;
        it.b = a.by_hkv.quot(bh);
        it.h = bh - it.b * a.hkv;
        it.len = sequence_length(a.seq_lens, it.b, a.kv_len);
        it.tiles = tiles_of<S::Keys>(it.len);
        c_begin = a.by_cluster.quot(it.tiles * rank);
        c_end = a.by_cluster.quot(it.tiles * (rank + 1));
        __syncthreads();                                       // the barriers are ready
    } else {
        const int per_thread = (a.batch + kWarps * 32 - 1) / (kWarps * 32);   // sequences of a thread
        int total = a.batch * tiles_of<S::Keys>(a.kv_len);
        if (a.seq_lens != nullptr) {
            int sum = 0, len = 0;
            for (int i = 0; i < per_thread; i++) {
                const int b = tid * per_thread + i;
                if (b >= a.batch) break;
                len = sequence_length(a.seq_lens, b, a.kv_len);
                sum += tiles_of<S::Keys>(len);
            }
            s_len[tid] = len;
            int inc = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            if (lane == 31) s_warp[warp] = inc;
            __syncthreads();
            int base = 0;
            total = 0;
#pragma unroll
            for (int w = 0; w < kWarps; w++) {
                if (w < warp) base += s_warp[w];
                total += s_warp[w];
            }
            s_prefix[tid] = base + inc - sum;
        }
        __syncthreads();
        total *= per_b;
        // equal parts of at least one tile a warp: CTAs without tiles come last, so those of an item follow one another
        chunk = max((total + (int)gridDim.x - 1) / (int)gridDim.x, kWarps);
        c_begin = (int)min((long long)total, (long long)chunk * blockIdx.x);
        c_end = min(total - c_begin, chunk) + c_begin;
    }
    {
        const int n = c_end - c_begin, q = n / kWarps, rest = n % kWarps;
        w_begin = c_begin + warp * q + min(warp, rest);
        w_end = w_begin + q + (warp < rest ? 1 : 0);
    }
    if (a.cluster == 0 && w_begin < w_end) {
        int b_start;                                           // first tile of sequence it.b
        if (a.seq_lens == nullptr) {
            it.tiles = tiles_of<S::Keys>(a.kv_len);
            it.len = a.kv_len;
            it.b = w_begin / (it.tiles * per_b);
            b_start = it.b * it.tiles * per_b;
        } else {
            const int per_thread = (a.batch + kWarps * 32 - 1) / (kWarps * 32);
            int lo = -1;                                       // last thread whose sequences begin at or before w_begin
#pragma unroll
            for (int i = 0; i < kWarps; i++) {
                const int y = i * 32 + lane;
                lo += __popc(__ballot_sync(0xffffffffu, s_prefix[y] * per_b <= w_begin && y * per_thread < a.batch));
            }
            it.b = lo * per_thread;
            b_start = s_prefix[lo] * per_b;
            for (;;) {
                it.len = per_thread == 1 ? s_len[lo] : sequence_length(a.seq_lens, it.b, a.kv_len);
                it.tiles = tiles_of<S::Keys>(it.len);
                const int end = b_start + it.tiles * per_b;
                if (w_begin < end || it.b + 1 >= a.batch) break;
                b_start = end;
                it.b++;
            }
        }
        const int i = (w_begin - b_start) / it.tiles;          // item of the sequence
        it.h = a.by_row_blocks.quot(i);
        it.rb = i - it.h * a.row_blocks;
        item_start = b_start + i * it.tiles;
    }

    const uint32_t ring = smem_u32(smem) + warp * S::WarpBytes;
    float* tail_record = reinterpret_cast<float*>(smem + warp * S::WarpBytes);
    float* head_record = a.scratch + (size_t)(blockIdx.x * kWarps + warp) * S::Record;
    int head_item = -1, tail_item = -1, before = 0, after = 0;

    // ---- the warp's ring: a barrier a stage, which TMA's copies of the codes complete.  The scales and offsets of a key, 4 or 8 bytes
    // of any row stride, come by ordinary loads a tile ahead, a lane a key; it unpacks them once for the four that need them.
    constexpr int P = D / 32;                                  // pieces of a row as the products see them: 32 elements, 16 bytes
    const uint32_t full0 = smem_u32(&s_full[warp][0]);
    const int box_shift = a.box_shift, boxes = S::Keys >> box_shift;        // rows of a TMA box; boxes of a tile
    const uint32_t factors = ring + S::Stages * S::StageBytes;
    const int in_page = a.map.page_shift < 0 ? 0x7FFFFFFF : (1 << a.map.page_shift) - 1;
    int stage = 0, load_stage = 0, in_flight = 0;
    uint32_t phase = 0;
    bool alive = true;
    // row and first piece of the lane's address for ldmatrix: keys 0-7, 8-15 of piece c, then of piece c + 1
    const int m_row = lane & 15;
    uint32_t m_at[P / 2];
#pragma unroll
    for (int c = 0; c < P / 2; c++) m_at[c] = ring + m_row * S::RowBytes + piece<D>(m_row, 2 * c + (lane >> 4)) * 16;

    // ---- loads: of the item `ld`, which the warp works on or is about to begin
    Item ld = it;
    auto page_of = [&](int key) -> int {                       // -1: names none, or past the end
        if (key >= ld.len) return -1;
        if (a.map.page_shift < 0) return ld.b;
        const int p = a.map.block_table[(long long)ld.b * a.map.table_stride + (key >> a.map.page_shift)];
        return (unsigned)p < (unsigned)a.map.n_pages ? p : -1;
    };
    // pages of a tile's boxes, one a lane
    auto pages_of = [&](int tile) { return lane < boxes ? page_of(tile * S::Keys + (lane << box_shift)) : -1; };
    auto load_codes = [&](int tile, int pages) {
        const int k0 = tile * S::Keys;
        const uint32_t dst = ring + load_stage * S::StageBytes, bar = full0 + load_stage * 8;
        load_stage = load_stage + 1 == S::Stages ? 0 : load_stage + 1;
        in_flight++;
        if (boxes == 1) {
            const int p = __shfl_sync(0xffffffffu, pages, 0);
            if (elect_one()) {
                // rows past the block and pages that name none read as zero; rows past the sequence's end hold any codes, and are masked
                mbar_arrive_expect_tx(bar, 2 * S::CodeBytes);
                tma_load_4d(dst, &a.tk, bar, 0, k0 & in_page, ld.h, p);
                tma_load_4d(dst + S::CodeBytes, &a.tv, bar, 0, k0 & in_page, ld.h, p);
            }
        } else {
            if (elect_one()) mbar_arrive_expect_tx(bar, 2 * S::CodeBytes);
            __syncwarp();
            if (lane < boxes) {
                const uint32_t at = dst + (lane << box_shift) * S::RowBytes;
                const int row = (k0 + (lane << box_shift)) & in_page;
                tma_load_4d(at, &a.tk, bar, 0, row, ld.h, pages);
                tma_load_4d(at + S::CodeBytes, &a.tv, bar, 0, row, ld.h, pages);
            }
            __syncwarp();
        }
    };
    constexpr int KPL = S::Keys / 32;                          // keys of a lane
    uint32_t kraw[KPL][G], vraw[KPL][G];
    auto load_pairs = [&](int tile, int pages) {
#pragma unroll
        for (int i = 0; i < KPL; i++) {
            const int key = tile * S::Keys + i * 32 + lane, p = __shfl_sync(0xffffffffu, pages, (i * 32 + lane) >> box_shift);
#pragma unroll
            for (int gi = 0; gi < G; gi++) kraw[i][gi] = vraw[i][gi] = 0;
            if (key < ld.len && p >= 0) {
                const long long off = p * a.p_block_stride + (long long)ld.h * a.p_head_stride + (long long)(key & in_page) * a.p_row_stride;
                ldg_pairs<G>(a.kp + off, kraw[i]);
                ldg_pairs<G>(a.vp + off, vraw[i]);
            }
        }
    };
    int ahead = -1, next_pages = -1;                           // pages of the tile whose pairs are loaded next, and of the one whose codes are
    static_assert(S::Stages == 3, "two tiles of codes are under way, and one of pairs");
    auto start = [&](int tile0, int tile1) {                   // the look-ups first, so that they wait together
        const int pages = pages_of(tile0);
        ahead = tile0 + 1 < tile1 ? pages_of(tile0 + 1) : -1;
        next_pages = tile0 + 2 < tile1 ? pages_of(tile0 + 2) : -1;
        load_pairs(tile0, pages);
        load_codes(tile0, pages);
        if (tile0 + 1 < tile1) load_codes(tile0 + 1, ahead);
    };
    if (w_begin < w_end) start(w_begin - item_start, min(it.tiles, w_end - item_start));

    // ---- item by item
    for (int x = w_begin; x < w_end && alive;) {
        const int tile0 = x - item_start, tile1 = min(it.tiles, tile0 + w_end - x);
        const int row0 = it.rb * S::Rows;

        // q as operand B: column g of the n-th 8 rows; 8 elements of a 16-byte piece of codes are two steps of k, in pairs
        // (i, i + 4) as the codes lie in a word.  bf16 rows are brought to fp16 by a power of two that puts their
        // largest element at 2^14: exact for elements down to 2^-28 of that one, and the rest is below its 32-bit rounding.
        uint32_t qf[NT][P][4];
        float q_init[NT][G][2];                                // -72 sum of q over the group
        float sc[NT][2];                                       // softmax scale (log2) of the columns that this thread has in S^T
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int r = row0 + n * 8 + g;
            const uint16_t* qp = a.q + out_row(a, it.b, it.h, r) * D;
            uint4 u[P];
#pragma unroll
            for (int c = 0; c < P; c++) u[c] = r < a.rows ? *reinterpret_cast<const uint4*>(qp + c * 32 + t * 8) : make_uint4(0, 0, 0, 0);
            if constexpr (BF16) {
                uint32_t top = 0;
#pragma unroll
                for (int c = 0; c < P; c++) {
                    const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const uint32_t e = max(top >> 7, 15u);         // exponent field of the largest element
                const float up = __uint_as_float((268u - e) << 23), down = __uint_as_float((e - 14u) << 23);
#pragma unroll
                for (int c = 0; c < P; c++) {
                    uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float2 f = unpack16<true>(w[i]);
                        w[i] = pack16<false>(f.x * up, f.y * up);
                    }
                    u[c] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                sc[n][0] = row_scale(a.scale_log2, __shfl_sync(0xffffffffu, down, 8 * t));
                sc[n][1] = row_scale(a.scale_log2, __shfl_sync(0xffffffffu, down, 8 * t + 4));
            } else {
                sc[n][0] = sc[n][1] = a.scale_log2;
            }
#pragma unroll
            for (int gi = 0; gi < G; gi++) {
                float sum = 0.0f;
#pragma unroll
                for (int c = 2 * gi; c < 2 * gi + 2; c++) {
                    const float2 f0 = unpack16<false>(u[c].x), f1 = unpack16<false>(u[c].y), f2 = unpack16<false>(u[c].z), f3 = unpack16<false>(u[c].w);
                    sum += ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
                    qf[n][c][0] = __byte_perm(u[c].x, u[c].z, 0x5410);
                    qf[n][c][1] = __byte_perm(u[c].x, u[c].z, 0x7632);
                    qf[n][c][2] = __byte_perm(u[c].y, u[c].w, 0x5410);
                    qf[n][c][3] = __byte_perm(u[c].y, u[c].w, 0x7632);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                q_init[n][gi][0] = -72.0f * __shfl_sync(0xffffffffu, sum, 8 * t);
                q_init[n][gi][1] = -72.0f * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            }
        }

        float o[NT][P][2][4], l[NT][2], m[NT][2], mc[NT][2], zs[NT][G][2];
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int c = 0; c < P; c++)
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][c][i][e] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; c++) {
                l[n][c] = mc[n][c] = 0.0f;                     // mc: the max as it is taken off, scaled; 0 as long as there is none
                m[n][c] = -INFINITY;
#pragma unroll
                for (int gi = 0; gi < G; gi++) zs[n][gi][c] = 0.0f;
            }
        }
        float s_limit = 0.0f, s_low = 0.0f, s_down = 0.0f;     // V's scales: the largest and least that E is kept for, 2^-E

        const int first_hidden = it.len - a.n_tok + a.by_group.quot(row0) + 1;       // first key that the block's first token does not see
        for (int tile = tile0; tile < tile1 && alive; tile++) {
            // this tile's factors: K's scale and offset of code 8 over -72, as it meets q_init; V's offset of code 8, and its scale
            // over 2^E, E such that the largest becomes 16 .. 32 when it is set: with P up to 2^8 and scales up to 2^7 times
            // 2^E a bracket stays below 2^15.  Below 2^-14 brackets lose digits, so E comes down again for a tile whose
            // scales are all far below what it allows (kScaleRange): a row of huge V^ costs its own tile alone.  (The second
            // vote: B=32 Hkv=8 Skv=16384 126.1 -> 127.1 us with 4 heads a KV head, 125.3 -> 126.9 in bf16, 196.7 -> 198.3 with 16 rows.)
            float s_max = 0.0f;
#pragma unroll
            for (int i = 0; i < KPL; i++)
#pragma unroll
                for (int gi = 0; gi < G; gi++) s_max = fmaxf(s_max, fabsf(unpack16<false>(vraw[i][gi]).x));
            if (__any_sync(0xffffffffu, s_max > s_limit) || (__all_sync(0xffffffffu, s_max < s_low) && __any_sync(0xffffffffu, s_max > 0.0f))) {
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) s_max = fmaxf(s_max, __shfl_xor_sync(0xffffffffu, s_max, off));
                s_max = fminf(s_max, kU4Max);                  // an infinite scale is lost by itself, not by what it does to E
                const float down = __uint_as_float(((254u + 4u) << 23) - (__float_as_uint(s_max) & 0x7F800000u));
                const float ratio = s_down == 0.0f ? 1.0f : down / s_down;
                s_down = down;
                s_limit = 128.0f / down;
                s_low = s_limit * kScaleRange;
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int i = 0; i < 2 * P; i++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[n][i / 2][i % 2][e] *= ratio;
            }
            // (the last tile's factors have been read: its products are issued, and below it the warp met)
#pragma unroll
            for (int i = 0; i < KPL; i++) {
                float fk[2 * G], fv[2 * G];
#pragma unroll
                for (int gi = 0; gi < G; gi++) {
                    const float2 k = unpack16<false>(kraw[i][gi]), v = unpack16<false>(vraw[i][gi]);
                    fk[gi] = k.x;
                    fk[G + gi] = fmaf(8.0f, k.x, k.y) * (-1.0f / 72.0f);
                    fv[gi] = v.x * s_down;
                    fv[G + gi] = fmaf(8.0f, v.x, v.y);
                }
                sts_factors<G>(factors + (i * 32 + lane) * 8 * G, fk);
                sts_factors<G>(factors + S::Keys * 8 * G + (i * 32 + lane) * 8 * G, fv);
            }
            alive = mbar_wait(full0 + stage * 8, phase, ctl, 1);       // the warp votes
            if (!alive) break;
            in_flight--;
            __syncwarp();                                      // the factors are written, and nobody reads the oldest stage any more
            if (tile + 2 < tile1) load_codes(tile + 2, next_pages);
            if (tile + 1 < tile1) {
                load_pairs(tile + 1, ahead);
                ahead = next_pages;
                next_pages = tile + 3 < tile1 ? pages_of(tile + 3) : -1;
            }
            const uint32_t at = stage * S::StageBytes;
            if (++stage == S::Stages) { stage = 0; phase ^= 1; }

            // S^T: keys j * 16 + g and + 8, columns 2t and 2t + 1 of each 8 rows
            float s[S::J][NT][4];
#pragma unroll
            for (int j = 0; j < S::J; j++) {
                float acc[G][NT][4];
#pragma unroll
                for (int gi = 0; gi < G; gi++) {
                    uint32_t w[4];                             // keys g, g + 8 of piece 2 gi, then of piece 2 gi + 1
                    ldmatrix4<false>(m_at[gi] + at + j * 16 * S::RowBytes, w);
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const uint32_t w0 = w[2 * c], w1 = w[2 * c + 1];
                        const uint32_t a0[4] = {code16<0, 64>(w0), code16<0, 64>(w1), code16<1, 64>(w0), code16<1, 64>(w1)};
                        const uint32_t a1[4] = {code16<2, 64>(w0), code16<2, 64>(w1), code16<3, 64>(w0), code16<3, 64>(w1)};
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            if (c == 0) mma_from(acc[gi][n], a0, qf[n][2 * gi][0], qf[n][2 * gi][1], q_init[n][gi][0], q_init[n][gi][1]);
                            else mma(acc[gi][n], a0, qf[n][2 * gi + c][0], qf[n][2 * gi + c][1]);
                            mma(acc[gi][n], a1, qf[n][2 * gi + c][2], qf[n][2 * gi + c][3]);
                        }
                    }
                }
#pragma unroll
                for (int e2 = 0; e2 < 2; e2++) {
                    float fk[2 * G];
                    lds_factors<G>(factors + (j * 16 + e2 * 8 + g) * 8 * G, fk);
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            float v = fk[G] * q_init[n][0][c];
                            if constexpr (G == 2) v = fmaf(fk[2 * G - 1], q_init[n][G - 1][c], v);
                            v = fmaf(fk[0], acc[0][n][e2 * 2 + c], v);
                            if constexpr (G == 2) v = fmaf(fk[G - 1], acc[G - 1][n][e2 * 2 + c], v);
                            s[j][n][e2 * 2 + c] = v;
                        }
                }
            }
            // masked keys: past what the row's token sees (only the last tiles have any)
            if ((tile + 1) * S::Keys > first_hidden) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int limit = it.len - a.n_tok + a.by_group.quot(row0 + n * 8 + 2 * t + c) + 1 - tile * S::Keys;
#pragma unroll
                        for (int j = 0; j < S::J; j++)
#pragma unroll
                            for (int e2 = 0; e2 < 2; e2++)
                                if (j * 16 + e2 * 8 + g >= limit || tile * S::Keys + j * 16 + e2 * 8 + g >= it.len) s[j][n][e2 * 2 + c] = -INFINITY;
                    }
            }
            // the running max may be exceeded by 2^8 before the sums are brought to a new one
            float t_max[NT][2];
            bool raise = false;
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    t_max[n][c] = fmaxf(s[0][n][c], s[0][n][2 + c]);
#pragma unroll
                    for (int j = 1; j < S::J; j++) t_max[n][c] = fmaxf(t_max[n][c], fmaxf(s[j][n][c], s[j][n][2 + c]));
                    raise |= (t_max[n][c] - m[n][c]) * sc[n][c] > kGrow;       // no max yet: inf, unless every key is masked
                }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float mx = t_max[n][c];
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
                        mx = fmaxf(mx, m[n][c]);
                        const float alpha = m[n][c] == -INFINITY ? 1.0f : ex2((m[n][c] - mx) * sc[n][c]);   // nothing summed so far: leave it
                        m[n][c] = mx;
                        mc[n][c] = mx == -INFINITY ? 0.0f : mx * sc[n][c];
                        l[n][c] *= alpha;
#pragma unroll
                        for (int gi = 0; gi < G; gi++) zs[n][gi][c] *= alpha;
#pragma unroll
                        for (int i = 0; i < 2 * P; i++) { o[n][i / 2][i % 2][c] *= alpha; o[n][i / 2][i % 2][2 + c] *= alpha; }
                    }
            }
            // P, its sums, and the brackets as operand B: columns to rows across the warp
            uint32_t pf[S::J][NT][G][2];
#pragma unroll
            for (int j = 0; j < S::J; j++)
#pragma unroll
                for (int e2 = 0; e2 < 2; e2++) {
                    float fv[2 * G];
                    lds_factors<G>(factors + S::Keys * 8 * G + (j * 16 + e2 * 8 + g) * 8 * G, fv);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        float x[2], p[2];
                        fma2(x, s[j][n] + e2 * 2, sc[n], mc[n]);
                        p[0] = ex2(x[0]);
                        p[1] = ex2(x[1]);
                        add2(l[n], p);
#pragma unroll
                        for (int gi = 0; gi < G; gi++) {
                            zs[n][gi][0] = fmaf(p[0], fv[G + gi], zs[n][gi][0]);
                            zs[n][gi][1] = fmaf(p[1], fv[G + gi], zs[n][gi][1]);
                            pf[j][n][gi][e2] = transpose8x8(pack16<false>(p[0] * fv[gi], p[1] * fv[gi]));
                        }
                    }
                }
            // O^T: elements 4g .. 4g + 3 of each piece, two of them per product of 16 rows
#pragma unroll
            for (int j = 0; j < S::J; j++)
#pragma unroll
                for (int gi = 0; gi < G; gi++) {
                    uint32_t y[4];                             // keys 2t, 2t + 1 and 2t + 8, 2t + 9 of piece 2 gi, then of piece 2 gi + 1
                    ldmatrix4<true>(m_at[gi] + at + S::CodeBytes + j * 16 * S::RowBytes, y);
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const uint32_t y0 = y[2 * c], y1 = y[2 * c + 1];
                        const uint32_t a0[4] = {code16<0, -8>(y0), code16<1, -8>(y0), code16<0, -8>(y1), code16<1, -8>(y1)};
                        const uint32_t a1[4] = {code16<2, -8>(y0), code16<3, -8>(y0), code16<2, -8>(y1), code16<3, -8>(y1)};
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            mma(o[n][2 * gi + c][0], a0, pf[j][n][gi][0], pf[j][n][gi][1]);
                            mma(o[n][2 * gi + c][1], a1, pf[j][n][gi][0], pf[j][n][gi][1]);
                        }
                    }
                }
        }
        if (!alive) {
            // a copy did not arrive: the status word says so.  Give those under way as long again, so that none lands in the
            // shared memory of another CTA, and leave the results as they are.
            const WaitCtl last{&s_never, a.status};
            for (; in_flight > 0; in_flight--) {
                mbar_wait(full0 + stage * 8, phase, last, 2);
                if (++stage == S::Stages) { stage = 0; phase ^= 1; }
            }
        }
        __syncwarp();

        // ---- the next item's first loads, before this one's sums are written
        const int x_next = x + tile1 - tile0, start_next = item_start + it.tiles;
        const bool last = x_next >= w_end;
        if (!last && alive) {
            if (++ld.rb == a.row_blocks) {
                ld.rb = 0;
                if (++ld.h == a.hkv) {
                    ld.h = 0;
                    ld.b++;
                    ld.len = sequence_length(a.seq_lens, ld.b, a.kv_len);
                    ld.tiles = tiles_of<S::Keys>(ld.len);
                }
            }
            start(0, min(ld.tiles, w_end - x_next));
        }

        // ---- the item's sums, or this warp's part of them
        const float up = s_down == 0.0f ? 0.0f : 1.0f / s_down;
        const bool whole = tile0 == 0 && tile1 == it.tiles && a.cluster <= 1;     // a cluster's result is its last step's
        const int item = (it.b * a.hkv + it.h) * a.row_blocks + it.rb;
        float* record = last ? tail_record : head_record;
        if (!whole) {
            if (last) tail_item = item;
            else head_item = item;
            if (item_start < c_begin) before = 1;              // only the CTA's first item can begin before it, only its last end after it
            if (item_start + it.tiles > c_end) after = item_start + it.tiles;
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], off);
#pragma unroll
                    for (int gi = 0; gi < G; gi++) zs[n][gi][c] += __shfl_xor_sync(0xffffffffu, zs[n][gi][c], off);
                }
                const int r = n * 8 + 2 * t + c;
                const float inv = l[n][c] == 0.0f ? 0.0f : 1.0f / l[n][c];
                const long long row = out_row(a, it.b, it.h, row0 + r);
#pragma unroll
                for (int i = 0; i < P; i++) {
                    const float z = zs[n][i / 2][c];
                    const float4 f = make_float4(fmaf(o[n][i][0][c], up, z), fmaf(o[n][i][0][2 + c], up, z), fmaf(o[n][i][1][c], up, z), fmaf(o[n][i][1][2 + c], up, z));
                    if (!whole) {
                        *reinterpret_cast<float4*>(record + r * D + i * 32 + g * 4) = f;
                    } else if (row0 + r < a.rows) {
                        *reinterpret_cast<uint2*>(a.o + row * D + i * 32 + g * 4) = make_uint2(pack16<BF16>(f.x * inv, f.y * inv), pack16<BF16>(f.z * inv, f.w * inv));
                    }
                }
                if (whole && row0 + r < a.rows && g == 0 && a.lse != nullptr)
                    a.lse[row] = l[n][c] == 0.0f ? -INFINITY : kLn2 * (mc[n][c] + log2f(l[n][c]));
                if (!whole && g == 0) {
                    s_m[2 * warp + last][r] = m[n][c] == -INFINITY ? -INFINITY : mc[n][c];
                    s_l[2 * warp + last][r] = l[n][c];
                }
            }
        x = x_next;
        item_start = start_next;
        it = ld;
    }

    // ---- the CTA's records
    if (lane == 0) {
        s_item[2 * warp] = head_item;
        s_item[2 * warp + 1] = tail_item;
        s_before[warp] = before;
        s_after[warp] = after;
    }
    __threadfence_block();
    __syncthreads();
    constexpr int kQuads = S::Rows * (D / 4);                  // four elements of a row
    if (a.cluster > 0) {
        // all of one item, a warp's (it has none if it had no tile, or wrote the whole item)
        const int cl = a.cluster, per_rank = a.by_cluster.quot(S::Rows + cl - 1);       // rows of a CTA
        if (cl > 1) cluster_wait();                            // the others run: their shared memory may be written
        for (int i = tid; i < kQuads; i += kWarps * 32) {
            const int r = i / (D / 4), d = (i % (D / 4)) * 4;
            float mx = -INFINITY, sum = 0.0f;
            bool any = false;
#pragma unroll
            for (int w = 0; w < kWarps; w++)
                if (s_item[2 * w + 1] >= 0) { mx = fmaxf(mx, s_m[2 * w + 1][r]); any = true; }
            float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; w++)
                if (s_item[2 * w + 1] >= 0)
                    add_record(f, sum, s_m[2 * w + 1][r], s_l[2 * w + 1][r], mx, reinterpret_cast<const float*>(smem + w * S::WarpBytes) + r * D + d);
            if (cl > 1) {
                // row r is CTA (r % cl)'s: into its shared memory, where it waits for those of the others
                const int owner = r - a.by_cluster.quot(r) * cl;
                const float* to = reinterpret_cast<const float*>(smem + kWarps * S::WarpBytes) + (rank * per_rank + a.by_cluster.quot(r)) * (D + 4);
                st_cluster4(to + d, owner, f);
                if (d == 0) st_cluster4(to + D, owner, make_float4(mx, sum, 0.0f, 0.0f));
            } else if (any && it.rb * S::Rows + r < a.rows) {
                store_quad<D, BF16>(a, out_row(a, it.b, it.h, it.rb * S::Rows + r), d, f, mx, sum);
            }
        }
        if (cl > 1) {
            __syncwarp();
            cluster_arrive();
            cluster_wait();
            const float* from = reinterpret_cast<const float*>(smem + kWarps * S::WarpBytes);
            for (int i = tid; i < kQuads; i += kWarps * 32) {
                const int y = i / (D / 4), d = (i % (D / 4)) * 4, r = y * cl + rank;
                if (r >= S::Rows || it.rb * S::Rows + r >= a.rows) break;
                float mx = -INFINITY, sum = 0.0f;
                float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int c = 0; c < cl; c++) mx = fmaxf(mx, from[(c * per_rank + y) * (D + 4) + D]);
                for (int c = 0; c < cl; c++) {
                    const float* rec = from + (c * per_rank + y) * (D + 4);
                    add_record(f, sum, rec[D], rec[D + 1], mx, rec + d);
                }
                store_quad<D, BF16>(a, out_row(a, it.b, it.h, it.rb * S::Rows + r), d, f, mx, sum);
            }
        }
        return;
    }
    // items of the line: the records of each are members of a mask, and their loads wait together
    const int my_item = lane < kRecords ? s_item[lane] : -1;
    int2 carried = make_int2(-1, 0);
    for (unsigned left = __ballot_sync(0xffffffffu, my_item >= 0); left != 0;) {
        const int k = __ffs(left) - 1, item = __shfl_sync(0xffffffffu, my_item, k);
        const unsigned members = __ballot_sync(0xffffffffu, my_item == item);
        left &= ~members;
        // it begins before this CTA's part if its first warp says so and this is that warp's first record, and ends after it likewise
        const int w0 = k >> 1, w1 = (31 - __clz(members)) >> 1;
        const bool starts_before = s_before[w0] != 0 && item == (s_item[2 * w0] >= 0 ? s_item[2 * w0] : s_item[2 * w0 + 1]);
        const bool ends_after = s_after[w1] != 0 && item == (s_item[2 * w1 + 1] >= 0 ? s_item[2 * w1 + 1] : s_item[2 * w1]);
        float* slot = a.scratch + ((size_t)gridDim.x * kWarps + 2 * blockIdx.x + (starts_before ? 0 : 1)) * S::Record;
        const int bh = a.by_row_blocks.quot(item), rb = item - bh * a.row_blocks, b = a.by_hkv.quot(bh), h = bh - b * a.hkv;
        if (ends_after && !starts_before) carried = make_int2(item, (s_after[w1] - 1) / chunk + 1);
        for (int i = tid; i < kQuads; i += kWarps * 32) {
            const int r = i / (D / 4), d = (i % (D / 4)) * 4;
            float mx = -INFINITY, sum = 0.0f;
            float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int y = 0; y < kRecords; y++)
                if (members >> y & 1) mx = fmaxf(mx, s_m[y][r]);
#pragma unroll
            for (int y = 1; y < kRecords; y += 2)              // a warp's last item: in its ring
                if (members >> y & 1) add_record(f, sum, s_m[y][r], s_l[y][r], mx, reinterpret_cast<const float*>(smem + (y >> 1) * S::WarpBytes) + r * D + d);
            if (members & 0x55555555u)
#pragma unroll
                for (int y = 0; y < kRecords; y += 2)          // its first: in the workspace
                    if (members >> y & 1) add_record(f, sum, s_m[y][r], s_l[y][r], mx, a.scratch + (size_t)(blockIdx.x * kWarps + (y >> 1)) * S::Record + r * D + d);
            if (starts_before || ends_after) {
                *reinterpret_cast<float4*>(slot + r * D + d) = f;
                if (d == 0) { slot[S::Rows * D + r] = mx; slot[S::Rows * (D + 1) + r] = sum; }
            } else if (rb * S::Rows + r < a.rows) {
                store_quad<D, BF16>(a, out_row(a, b, h, rb * S::Rows + r), d, f, mx, sum);
            }
        }
    }
    if (tid == 0) a.meta[blockIdx.x] = carried;
}

// Items that lie in several CTAs: a block takes 8 rows of the item that begins in CTA c and goes on, four warps a row, and
// merges c's second record and the first records of the CTAs up to the item's last.
template <int D, bool BF16, int NT>
__global__ void __launch_bounds__(1024) u4_merge_kernel(const __grid_constant__ U4Args a, int n_ctas) {
    using S = Shape<D, NT>;
    constexpr int kSubs = 4;                                   // warps of a row
    __shared__ float4 part[kSubs][8][32];
    __shared__ float part_l[kSubs][8];
    grid_dependency_wait();
    grid_launch_dependents();
    const int c = blockIdx.x / NT, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp >> 3, r = blockIdx.x % NT * 8 + (warp & 7);
    const int2 carried = a.meta[c];
    if (carried.x < 0) return;
    const int item = carried.x, last = carried.y;
    const int bh = a.by_row_blocks.quot(item), rb = item - bh * a.row_blocks, b = a.by_hkv.quot(bh), h = bh - b * a.hkv;
    const bool live = rb * S::Rows + r < a.rows;
    const float* base = a.scratch + (size_t)n_ctas * kWarps * S::Record;
    auto record = [&](int i) { return base + (size_t)(2 * i + (i == c ? 1 : 0)) * S::Record; };
    float mx = -INFINITY, sum = 0.0f;
    float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (live) {
        for (int i = c + lane; i < last; i += 32) mx = fmaxf(mx, record(i)[S::Rows * D + r]);
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
#pragma unroll 4
        for (int i = c + sub; i < last; i += kSubs) {
            const float* rec = record(i);
            const float yl = rec[S::Rows * (D + 1) + r], w = record_weight(rec[S::Rows * D + r], yl, mx);
            const float4 z = lane < D / 4 ? *reinterpret_cast<const float4*>(rec + r * D + lane * 4) : f;
            sum = fmaf(w, yl, sum);
            f.x = fmaf(w, z.x, f.x); f.y = fmaf(w, z.y, f.y); f.z = fmaf(w, z.z, f.z); f.w = fmaf(w, z.w, f.w);
        }
        part[sub][warp & 7][lane] = f;
        if (lane == 0) part_l[sub][warp & 7] = sum;
    }
    __syncthreads();
    if (sub == 0 && live && lane < D / 4) {
#pragma unroll
        for (int y = 1; y < kSubs; y++) {
            const float4 z = part[y][warp][lane];
            f.x += z.x; f.y += z.y; f.z += z.z; f.w += z.w;
            sum += part_l[y][warp];
        }
        store_quad<D, BF16>(a, out_row(a, b, h, rb * S::Rows + r), lane * 4, f, mx, sum);
    }
}

// ------------------------------------------------------------------------------------------ many tokens
// bf16 q as fp16 for the 16-bit kernel: a power of two for each row puts its largest element at 2^14 .. 2^15 and goes back
// into the row's softmax scale, as in u4_kernel.  Of each row: what one row holds (a padded token's garbage, an infinity)
// must not decide what is left of another.  A row is D / 8 lanes.
template <int D>
__global__ void __launch_bounds__(256) q_f16_kernel(const uint4* q, uint4* out, float* factor, long long pieces) {
    constexpr int LPR = D / 8;
    grid_dependency_wait();
    grid_launch_dependents();
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const bool live = i < pieces;                              // of whole rows: the lanes of a row agree
    const uint4 u = live ? q[i] : make_uint4(0, 0, 0, 0);
    uint32_t w[4] = {u.x, u.y, u.z, u.w}, top = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) top = max(top, max(w[j] & 0x7FFFu, (w[j] >> 16) & 0x7FFFu));
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) return;
    const uint32_t e = max(top >> 7, 15u);                     // exponent field of the largest element
    const float up = __uint_as_float((268u - e) << 23);
    if (i % LPR == 0) factor[i / LPR] = __uint_as_float((e - 14u) << 23);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float2 f = unpack16<true>(w[j]);
        w[j] = pack16<false>(f.x * up, f.y * up);
    }
    out[i] = make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------------------------------ host
struct Plan {
    int nt;                 // 8-row columns of a block
    int row_blocks;
    int cluster;            // CTAs of an item; 0: equal parts of the line of all tiles
    int ctas;
    long long tiles;        // at most, of all items
    size_t record;          // bytes
    size_t bytes;           // of the workspace
};
size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// Clusters of `size` CTAs that the current device holds at once (every instance has one CTA an SM); the GPCs have unequal
// numbers of SMs, so that these are fewer than sm_count / size.
int clusters_at_once(DeviceState* st, int size) {
    if (size == 1) return st ? st->sm_count : 148;
    if (!st) return 100 / size;
    static std::atomic<int> known[64][kMaxCluster + 1];
    std::atomic<int>& k = known[st->device][size];
    int n = k.load(std::memory_order_relaxed);
    if (n > 0) return n;
    constexpr int smem = Shape<128, 1>::SmemBytes;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = size;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(u4_kernel<128, false, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&n, u4_kernel<128, false, 1>, &cfg) != cudaSuccess || n <= 0) {
        cudaGetLastError();
        n = 1;
    }
    k.store(n, std::memory_order_relaxed);
    return n;
}

Plan make_plan(int batch, int hq, int hkv, int n_tok, int kv_len, bool own_lengths, int d_head, DeviceState* st) {
    Plan p;
    const long long rows = (long long)n_tok * (hq / hkv);
    p.nt = rows <= 8 ? 1 : 2;
    p.row_blocks = (int)((rows + 8 * p.nt - 1) / (8 * p.nt));
    const long long items = (long long)batch * hkv * p.row_blocks, item_tiles = (kv_len + tile_keys(p.nt) - 1) / tile_keys(p.nt);
    p.tiles = items * item_tiles;
    const long long slots = st ? st->sm_count : 148;
    // A cluster an item, the largest of which all are on the GPU at once, if its warps get at most one tile beyond an equal share
    // (us in a graph, line / clusters, D = 128, Hkv = 8: B=16 Skv=1024 13.7 / 10.8, B=16 Skv=4096, a tile more, 26.1 / 22.7; B=1
    // Skv=8192, a tile more, 12.1 / 12.1; B=1 Skv=16384, two more, 14.5 / 15.9; B=16 Skv=16384, four more, 69 / 72).  Sequences of
    // their own lengths are taken to be half as long as they may be on average, which the line deals evenly.
    p.cluster = 0;
    if (items <= slots) {
        const long long want = (item_tiles + kWarps - 1) / kWarps;
        int cl = (int)(want < kMaxCluster ? want : kMaxCluster);
        while (cl > 1 && clusters_at_once(st, cl) < items) cl--;
        const long long each = (item_tiles + cl * kWarps - 1) / (cl * kWarps), share = (p.tiles / (own_lengths ? 2 : 1) + slots * kWarps - 1) / (slots * kWarps);
        if (each <= share + kClusterTiles) p.cluster = cl;
    }
    const long long want = (p.tiles + kWarps - 1) / kWarps;
    p.ctas = (int)(want < slots ? want : slots);
    p.record = (size_t)8 * p.nt * (d_head + 2) * sizeof(float);
    p.bytes = align256(p.record * p.ctas * (kWarps + 2)) + align256((size_t)p.ctas * sizeof(int2));      // clusters need none
    if (p.cluster) p.ctas = (int)(items * p.cluster);
    return p;
}

template <int D, bool BF16, int NT>
int run_u4(const U4Args& a, int ctas, DeviceState* st, cudaStream_t stream) {
    using S = Shape<D, NT>;
    static bool configured[64] = {};
    const int smem = S::SmemBytes;
    if (!configured[st->device]) {
        FA_CUDA_TRY(cudaFuncSetAttribute(u4_kernel<D, BF16, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        configured[st->device] = true;
    }
    const int rc = launch_dependent(u4_kernel<D, BF16, NT>, ctas, kWarps * 32, smem, stream, a.cluster > 1 ? a.cluster : 1, a);
    if (rc != FA_OK || a.cluster > 0 || ctas == 1) return rc;
    return launch_dependent(u4_merge_kernel<D, BF16, NT>, ctas * NT, 1024, 0, stream, 1, a, ctas);
}
template <int D, bool BF16>
int run_u4_rows(const U4Args& a, const Plan& p, DeviceState* st, cudaStream_t stream) {
    if (p.nt == 1) return run_u4<D, BF16, 1>(a, p.ctas, st, stream);
    return run_u4<D, BF16, 2>(a, p.ctas, st, stream);
}

// Many query rows: the 16-bit kernel (tcgen05) over a copy of the cache in fp16.  mma.sync runs at a quarter of tcgen05's rate,
// and a block of 16 rows reads and unpacks the whole cache again; the copy is written once.  For f16 the copy holds K^ and V^ as fp16
// values and fp16 remainders, and both go through the products (22 bits of them count): rounded to fp16 alone they cost half of
// the digits that an fp16 O can show (4.1e-4 of its norm off instead of 2.9e-4, of which P and O's own rounding are all), at
// 290 instead of 459 us for 8 x 512 tokens on 3584 keys, Hq=32 Hkv=8 D=128.  A bf16 O has no such digits (1.7e-3 either way, its LSE off by up to
// 1e-4 where a row sees few keys): there the values alone go in.
// From which number of rows, us in a graph, row blocks / copy, Hkv=8: bf16 D=128 B=8 Skv=4096 80 rows 76 / 65, 96 88 / 66, B=1 Skv=4096
// 80 17.5 / 18.9, 96 26 / 19.5; D=64 B=8 Skv=4096 80 53 / 41, B=1 Skv=4096 80 12.7 / 15.1, 96 19 / 15; f16 D=128 B=8 Skv=4096 96 85 / 106, 128
// 110 / 108, B=1 Skv=16384 96 49 / 55, 128 60 / 57; D=64 B=8 Skv=4096 80 53 / 55, 96 61 / 55.  (Blocks of 32 rows need more registers than there
// are: 97 and 163 us where those of 16 take 61 and 109.)  In caches of fewer than 512 rows the copy is
// faster with a batch too (511 rows, a copy of the values alone: B=1 256 query rows 10.5 / 11.8, 2000 54.9 / 15.6; B=8 96 27.8 / 17.0, 2000
// 239 / 45), but what the exact codes in one launch cost is bounded there, so they stay.  The rule asks for the cache's capacity,
// which the host knows; the lengths are on the device.
struct ManyPlan {
    int batch;                                // sequences of a copy
    int splits;                               // KV splits of the 16-bit kernel
    size_t cache, partial, q, factor;         // bytes: K's copy (V's as much), partial results, q in fp16, its rows' factors
    size_t bytes() const { return 2 * cache + partial + q + factor; }
};
bool many_rows(int hq, int hkv, int n_tok, int kv_len, int d_head, bool bf) {
    const long long rows = (long long)n_tok * (hq / hkv);
    return rows >= (d_head == 128 && !bf ? kManyRowsF16 : kManyRows) && kv_len >= kManyKeys && hq / hkv <= 128;
}
ManyPlan make_many_plan(int batch, int hq, int hkv, int n_tok, int kv_len, int d_head, bool bf) {
    ManyPlan p;
    const size_t one = (size_t)hkv * kv_len * d_head * 2 * (bf ? 1 : 2);         // f16: values and remainders
    const size_t fit = kCopyBytes / (2 * one);
    p.batch = fit < 1 ? 1 : fit < (size_t)batch ? (int)fit : batch;
    p.cache = align256(one * p.batch);
    const int group = hq / hkv, per_tile = 128 / group < n_tok ? 128 / group : n_tok, n_qt = (n_tok + per_tile - 1) / per_tile;
    p.splits = fa_decode_gqa_default_splits(p.batch * n_qt, hkv, kv_len);
    p.partial = align256(fa_decode_workspace_bytes(p.batch, n_tok * hq, d_head, p.splits));
    p.q = bf ? align256((size_t)batch * n_tok * hq * d_head * 2) : 0;
    p.factor = bf ? align256((size_t)batch * n_tok * hq * sizeof(float)) : 0;
    return p;
}

// Workspace of a call of either type: the caller is not asked for it.
size_t workspace_bytes(int batch, int hq, int hkv, int n_tok, int kv_len, int d_head, DeviceState* st) {
    size_t most = 0;
    for (const bool bf : {false, true}) {
        const size_t n = many_rows(hq, hkv, n_tok, kv_len, d_head, bf) ? make_many_plan(batch, hq, hkv, n_tok, kv_len, d_head, bf).bytes()
                                                                       : make_plan(batch, hq, hkv, n_tok, kv_len, false, d_head, st).bytes;
        most = n > most ? n : most;
    }
    return most;
}

// f16: values and remainders of K^ and V^.  bf16: q goes in as fp16 with a factor a row, O comes out as bf16 from the kernel and its
// merge, rounded once.
int run_many(const fa_decode_gqa_u4_args* p, int n_tok, DeviceState* st) {
    const ManyPlan m = make_many_plan(p->batch_size, p->num_q_heads, p->num_kv_heads, n_tok, p->seq_len_kv, p->d_head, p->dtype == FA_DTYPE_BF16);
    cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
    uint8_t* at = static_cast<uint8_t*>(p->workspace);
    uint8_t *k16 = at, *v16 = k16 + m.cache, *partial = v16 + m.cache, *q16 = partial + m.partial;
    float* factor = reinterpret_cast<float*>(q16 + m.q);
    const bool bf = p->dtype == FA_DTYPE_BF16;
    const size_t row = (size_t)p->num_q_heads * p->d_head;                       // elements of a token
    const long long pieces = (long long)p->batch_size * n_tok * row / 8;         // of 16 bytes: below 2^35, 2^27 blocks of them
    const int hkv = p->num_kv_heads;
    int rc;
    if (bf) {
        auto kernel = p->d_head == 64 ? q_f16_kernel<64> : q_f16_kernel<128>;
        rc = launch_dependent(kernel, (unsigned)((pieces + 255) / 256), 256, 0, stream, 1, static_cast<const uint4*>(p->q), reinterpret_cast<uint4*>(q16), factor, pieces);
        if (rc != FA_OK) return rc;
    }
    for (int b0 = 0; b0 < p->batch_size; b0 += m.batch) {
        const int nb = p->batch_size - b0 < m.batch ? p->batch_size - b0 : m.batch;
        fa_cache_read_args r = {};
        r.layout = p->layout;
        if (r.layout.seq_lens) r.layout.seq_lens += b0;
        const bool paged = r.layout.block_table != nullptr;
        if (paged) r.layout.block_table += (size_t)b0 * r.layout.block_table_stride;
        const size_t skip = paged ? 0 : (size_t)b0 * r.layout.block_stride, pskip = paged ? 0 : (size_t)b0 * r.layout.param_block_stride * 4;
        r.k_cache = static_cast<const uint8_t*>(p->k_cache) + skip;
        r.v_cache = static_cast<const uint8_t*>(p->v_cache) + skip;
        r.k_params = static_cast<const uint8_t*>(p->k_params) + pskip;
        r.v_params = static_cast<const uint8_t*>(p->v_params) + pskip;
        r.k_out = k16;
        r.v_out = v16;
        r.batch_size = nb;
        r.num_kv_heads = hkv;
        r.seq_len_kv = r.num_rows = p->seq_len_kv;
        r.d_head = p->d_head;
        r.dtype = FA_DTYPE_F16;
        r.stream = p->stream;
        const long long head = (long long)p->seq_len_kv * p->d_head;
        if ((rc = launch_copy_u4(r, head * hkv, p->d_head, head, bf ? 0 : nb * hkv * head)) != FA_OK) return rc;
        fa_decode_gqa_args g = {};
        const size_t q0 = (size_t)b0 * n_tok * row;
        g.q = bf ? static_cast<const void*>(q16 + 2 * q0) : static_cast<const uint16_t*>(p->q) + q0;
        g.k = k16;
        g.v = v16;
        g.o = static_cast<uint16_t*>(p->o) + q0;
        g.lse = p->lse ? p->lse + (size_t)b0 * n_tok * p->num_q_heads : nullptr;
        g.batch_size = nb;
        g.num_q_heads = p->num_q_heads;
        g.num_kv_heads = hkv;
        g.seq_len_kv = p->seq_len_kv;
        g.d_head = p->d_head;
        g.scale = p->scale;
        g.dtype = FA_DTYPE_F16;
        g.num_splits = m.splits;
        g.kv_batch_stride = head * hkv;
        g.kv_head_stride = head;
        g.kv_row_stride = p->d_head;
        g.seq_lens = r.layout.seq_lens;
        g.num_q_tokens = n_tok;
        g.workspace = partial;
        g.workspace_bytes = m.partial;
        g.stream = p->stream;
        if ((rc = decode_gqa(&g, bf ? factor + (size_t)b0 * n_tok * p->num_q_heads : nullptr, !bf)) != FA_OK) return rc;
    }
    return FA_OK;
}

}  // namespace
}  // namespace fa

using namespace fa;

FA_EXPORT size_t fa_decode_gqa_u4_workspace_bytes(int batch_size, int num_q_heads, int num_kv_heads, int num_q_tokens,
                                                  int seq_len_kv, int d_head) {
    if (batch_size <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0 || num_q_tokens < 0 || seq_len_kv <= 0)
        return 0;
    if (d_head != 64 && d_head != 128) return 0;
    DeviceState* st = device_state();
    const int n_tok = num_q_tokens > 0 ? num_q_tokens : 1;
    return workspace_bytes(batch_size, num_q_heads, num_kv_heads, n_tok, seq_len_kv, d_head, st);
}

FA_EXPORT int fa_decode_gqa_u4(const fa_decode_gqa_u4_args* p) {
    if (!p || !p->q || !p->k_cache || !p->k_params || !p->v_cache || !p->v_params || !p->o) return FA_ERR_INVALID_ARGUMENT;
    if (p->batch_size <= 0 || p->num_q_heads <= 0 || p->num_kv_heads <= 0 || p->seq_len_kv <= 0) return FA_ERR_INVALID_ARGUMENT;
    if (p->num_q_heads % p->num_kv_heads != 0) return FA_ERR_INVALID_ARGUMENT;
    if (!(p->scale > 0.0f) || !std::isfinite(p->scale)) return FA_ERR_INVALID_ARGUMENT;
    const int n_tok = p->num_q_tokens > 0 ? p->num_q_tokens : 1;
    if (p->num_q_tokens < 0 || n_tok > p->seq_len_kv) return FA_ERR_INVALID_ARGUMENT;
    if (p->d_head != 64 && p->d_head != 128) return FA_ERR_UNSUPPORTED;
    if (p->dtype != FA_DTYPE_F16 && p->dtype != FA_DTYPE_BF16) return FA_ERR_UNSUPPORTED;
    if ((long long)p->batch_size * n_tok * p->num_q_heads > 0x7FFFFFFFll || p->seq_len_kv > 0x7FFFFFFF - 64) return FA_ERR_INVALID_ARGUMENT;
    U4Args a;
    int rc = check_layout(p->layout, FA_CACHE_U4, p->d_head, p->seq_len_kv, 0, &a.map);
    if (rc != FA_OK) return rc;
    if (!aligned16(p->q) || !aligned16(p->k_cache) || !aligned16(p->v_cache) || !aligned16(p->k_params) || !aligned16(p->v_params) || !aligned16(p->o))
        return FA_ERR_MISALIGNED;
    if (reinterpret_cast<uintptr_t>(p->lse) & 3u) return FA_ERR_MISALIGNED;
    DeviceState* st = device_state();
    if (!st) return FA_ERR_CUDA;
    if (st->cc_major != 10) return FA_ERR_NOT_SM100;
    const bool many = many_rows(p->num_q_heads, p->num_kv_heads, n_tok, p->seq_len_kv, p->d_head, p->dtype == FA_DTYPE_BF16);
    const size_t need = workspace_bytes(p->batch_size, p->num_q_heads, p->num_kv_heads, n_tok, p->seq_len_kv, p->d_head, st);
    const bool room = p->workspace && p->workspace_bytes >= need && aligned16(p->workspace);
    if (many) return room ? run_many(p, n_tok, st) : FA_ERR_WORKSPACE;
    const Plan plan = make_plan(p->batch_size, p->num_q_heads, p->num_kv_heads, n_tok, p->seq_len_kv, p->layout.seq_lens != nullptr, p->d_head, st);
    if (plan.tiles > 0x7FFF0000ll) return FA_ERR_INVALID_ARGUMENT;
    if (!room) return FA_ERR_WORKSPACE;
    const bool paged = p->layout.block_table != nullptr;
    const int keys = tile_keys(plan.nt), box_rows = paged && p->layout.page_size < keys ? p->layout.page_size : keys;
    for (a.box_shift = 0; (1 << a.box_shift) < box_rows;) a.box_shift++;
    const int block_rows = paged ? p->layout.page_size : p->seq_len_kv, blocks = paged ? p->layout.num_pages : p->batch_size;
    for (int i = 0; i < 2; i++) {
        rc = make_tensor_map_u4(i ? &a.tv : &a.tk, i ? p->v_cache : p->k_cache, p->d_head / 2, block_rows, p->num_kv_heads, blocks,
                                p->layout.row_stride, p->layout.head_stride, p->layout.block_stride, box_rows);
        if (rc != FA_OK) return rc;
    }
    a.status = st->status;
    a.q = static_cast<const uint16_t*>(p->q);
    a.kp = static_cast<const __half2*>(p->k_params);
    a.vp = static_cast<const __half2*>(p->v_params);
    a.o = static_cast<uint16_t*>(p->o);
    a.lse = p->lse;
    a.scratch = static_cast<float*>(p->workspace);
    a.meta = reinterpret_cast<int2*>(static_cast<uint8_t*>(p->workspace) + align256(plan.record * plan.ctas * (kWarps + 2)));     // the line's
    a.p_block_stride = p->layout.param_block_stride;
    a.p_head_stride = p->layout.param_head_stride;
    a.p_row_stride = p->layout.param_row_stride;
    a.seq_lens = p->layout.seq_lens;
    a.batch = p->batch_size;
    a.hq = p->num_q_heads;
    a.hkv = p->num_kv_heads;
    a.n_tok = n_tok;
    a.group = p->num_q_heads / p->num_kv_heads;
    a.rows = n_tok * a.group;
    a.row_blocks = plan.row_blocks;
    a.cluster = plan.cluster;
    a.by_group = FastDiv(a.group);
    a.by_row_blocks = FastDiv(plan.row_blocks);
    a.by_hkv = FastDiv(p->num_kv_heads);
    a.by_cluster = FastDiv(plan.cluster > 0 ? plan.cluster : 1);
    a.kv_len = p->seq_len_kv;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    cudaStream_t stream = static_cast<cudaStream_t>(p->stream);
    const bool bf = p->dtype == FA_DTYPE_BF16;
    if (p->d_head == 64) return bf ? run_u4_rows<64, true>(a, plan, st, stream) : run_u4_rows<64, false>(a, plan, st, stream);
    return bf ? run_u4_rows<128, true>(a, plan, st, stream) : run_u4_rows<128, false>(a, plan, st, stream);
}
