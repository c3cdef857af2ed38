// Tile helpers of the attention kernels (attention.hip, diff_attention.hip): LDS image of a [32 rows][64 columns] bf16 tile, its MFMA
// operand fragments in both directions, LDS-DMA pieces, XCD-aware block decode.  Included inside each file's anonymous namespace.

// raised priority while a wave issues its MFMA groups: the matrix pipe is fed first, other waves' VALU fills the issue gaps
#define ATTN_PRIO(x) __builtin_amdgcn_s_setprio(x)

constexpr int HD = 64;
constexpr int RS = 128;              // LDS row stride in bytes (no padding)
constexpr int TILE = 32 * RS;        // one 32-row tile
// One LDS image serves BOTH the row reads (ds_read_b128, MFMA operand = rows of the tile) and the transposed reads
// (ds_read_b64_tr_b16, MFMA operand = columns): 16-B chunk c of row r is stored at chunk c ^ swz(r),
// swz(r) = ((r>>1)&1)<<2 | (r>>2)&3.  Brute-force checked conflict-free for every fragment of both kinds (the padded
// 144-B rows were 2-way conflicted on the transposed reads: 23-26 % of the LDS cycles, and these kernels are LDS-bound).
__device__ __forceinline__ int swz(int r) { return (((r >> 1) & 1) << 2) | ((r >> 2) & 3); }
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float fast_log2(float x) { return __builtin_amdgcn_logf(x); }
__device__ __forceinline__ int acc_row(int r, int hh) { return (r & 3) + 8 * (r >> 2) + 4 * hh; }

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// A operand = rows of a [32][64] LDS tile: A[row = lane&31][k = 16 ks + 8 hh + j]
__device__ __forceinline__ bf16x8 row_frag(const unsigned char* tile, int ks, int lane) {
    const int r = lane & 31;
    return *(const bf16x8*)(tile + r * RS + (((2 * ks + (lane >> 5)) ^ swz(r)) << 4));
}

// A operand = TRANSPOSE of a [32 seq][64 d] LDS tile for k-step s2 (16 seq rows) and d-tile dt (32 d):
// A[row = d = 32 dt + (lane&31)][slot (hh, j)] = tile[seq = 16 s2 + 8 (j>>2) + 4 hh + (j&3)][d]
__device__ __forceinline__ bf16x8 tr_frag(const unsigned char* tile, int s2, int dt, int lane) {
    const int g = lane >> 4, i = lane & 15, q = i >> 2, pp = i & 3, hh = lane >> 5;
    const int r0 = 16 * s2 + 4 * hh + q, r1 = r0 + 8;
    const int chunk = 4 * dt + 2 * (g & 1) + (pp >> 1), sub = (pp & 1) * 8;
    const unsigned char* a0 = tile + r0 * RS + ((chunk ^ swz(r0)) << 4) + sub;
    const unsigned char* a1 = tile + r1 * RS + ((chunk ^ swz(r1)) << 4) + sub;
    s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)LDS_PTR(a0));
    s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)LDS_PTR(a1));
    // compose as 32-bit words (element-wise 16-bit assembly made hipcc emit v_perm / v_or / v_mov chains)
    const u32x2 l2 = __builtin_bit_cast(u32x2, lo), h2 = __builtin_bit_cast(u32x2, hi);
    const u32x4 r = {l2[0], l2[1], h2[0], h2[1]};
    return __builtin_bit_cast(bf16x8, r);
}

// pack accumulator registers 8 s .. 8 s + 7 into the B fragment of k-step s
__device__ __forceinline__ bf16x8 pack_frag(const float* p, int s) {
    bf16x8 f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (__bf16)p[8 * s + j];
    return f;
}

// store an accumulator tile pair D[d][seq] (seq on the lane) as bf16 rows dst[seq][d], scaled
__device__ __forceinline__ void store_T(bf16_t* dst_row, const f32x16& a0, const f32x16& a1, float mul, int hh) {
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) {
        const f32x16& a = dt ? a1 : a0;
#pragma unroll
        for (int rg = 0; rg < 4; ++rg) {
            u32x2 o = {pack_bf16x2(a[4 * rg] * mul, a[4 * rg + 1] * mul), pack_bf16x2(a[4 * rg + 2] * mul, a[4 * rg + 3] * mul)};
            *(u32x2*)(dst_row + 32 * dt + 8 * rg + 4 * hh) = o;
        }
    }
}

// XCD-aware block decode.  Blocks are dealt round-robin over the 8 XCDs (private L2s), so the NX blocks that share one
// (clip, head)'s K/V (or Q/dO) must have block ids that are EQUAL mod 8, otherwise every XCD re-fetches the same K/V
// (measured: FETCH_SIZE 5x the algorithmic bytes, TA/TC 93 % busy).  1-D grid of 8 * ceil(G/8) * NX blocks:
// id -> xcd = id & 7, slot = id >> 3 -> group = (slot / NX) * 8 + xcd, x = slot % NX.  Speed only, never correctness.
__device__ __forceinline__ bool decode_block(int nx, int G, int H, int& xb, int& b, int& h) {
    const int id = blockIdx.x;
    const int xcd = id & 7, slot = id >> 3;
    const int gl = slot / nx;
    xb = slot - gl * nx;
    const int g = gl * 8 + xcd;
    if (g >= G) return false;
    b = g / H;
    h = g - b * H;
    return true;
}

// LDS-DMA (global -> LDS, no VGPR destination) as inline asm: invisible to hipcc's wait-count bookkeeping, so the loads of
// the NEXT query block can stay in flight across the barriers of a whole block (7 steps) and are drained by one explicit
// `s_waitcnt vmcnt(0)` before the block's last barrier.  Register staging (load at the top of a step, ds_write at its end)
// made every step as long as a loaded chip's global-load latency: 4 700 clk for 640 clk of MFMA.  M0 = LDS byte address of
// the wave's 1 KiB (dwordx4) / 256 B (dword) piece; lane l lands at + 16 l / + 4 l; the source address is per lane.
__device__ __forceinline__ void dma_b128(const void* gsrc, unsigned lds_dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(gsrc), "s"(lds_dst) : "memory");
}
__device__ __forceinline__ void dma_b32(const void* gsrc, unsigned lds_dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(gsrc), "s"(lds_dst) : "memory");
}
// the same with a UNIFORM base address in an SGPR pair and a 32-bit per-lane byte offset: no 64-bit vector address arithmetic per piece
__device__ __forceinline__ void dma_b128_s(const void* sbase, int voff, unsigned lds_dst) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff), "s"(sbase), "s"(lds_dst) : "memory");
}
