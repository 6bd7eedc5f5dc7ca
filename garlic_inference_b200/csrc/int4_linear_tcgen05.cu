// y = x W^T for a weight in 4 bits (layout: int4_weight.cu) and more rows of bfloat16 x than int4_linear.cu takes at once: decode batches and
// short prompts, with W read and made wide once for 32 or 64 rows.
//
// A block takes 128 outputs (with a gated unit 64 of the gate's and the 64 of the up half that meet them), a block of rows of x and, as
// one of the blocks of a cluster, a slice of K.  For each group of 128 inputs of its slice:
//   warp 8       asks for codes and steps, two groups of a row of tiles a copy, into a ring of shared memory (a copy costs 90 cycles: in pieces
//                of 512 bytes W came at 1.1 us a group).  W is nobody's output: in a recorded step the ring fills before the kernel
//                waits for the one that makes x.
//   warps 0-7    make it wide, two groups of four warps in turn: step * q + low in bfloat16 (one rounding, by fma), a thread an output, into
//                tensor memory: the 128-row operand never passes through shared memory again, 32 KB a group.  bfloat16, since both operands
//                are of one type and x is that: an f16 would round less, but have no room for what x and a step may be without a scale for
//                every row of x and every output, which would have to be known before the first group.
//   warp 9       brings the rows of x.
//   warp 10      products, 128 x BN x 16, accumulated in float32 in tensor memory over the whole slice.
// Then the sums go to shared memory, the blocks of the cluster add up a share of the rows each, in the order of the ranks (the same bits from
// run to run), and write.
//
// Reading W is 8,704 bytes a group, 0.2 us of an SM's share of the memory rate.  Measured 0.5 us a group and SM, with one block or two: without the
// arithmetic of unpacking (17 instructions for 8 numbers, 1,150 of a warp a group) 0.3, without the products 0.48; more warps that unpack,
// deeper rings and waits that sleep change nothing.  (Two of the 17 keep the numbers in their order, so that x can come by tensor copies: four
// warps that reordered x instead took 880 instructions a group.)  32 rows, us: 4,096 x 4,096 10.8, 5,120 x 17,408 28.4, 24,576 x 4,096 31.6;
// 64 rows 12.9, -, 34.8; 128 rows 24,576 x 4,096 53.
#include "int4.cuh"
#include "glu.cuh"
#include "tcgen05.cuh"

#define I4W_THREADS 352
#define I4W_SG 2                   // groups of one copy of a row of tiles
#define I4W_RING 3                 // copies of the eight rows on their way or in use
#define I4W_A 3                    // groups made wide (64 columns of tensor memory each) with their x
#define I4W_ROW (I4W_SG * I4_TILE + 16)      // a row of tiles in shared memory; rows lie one more bank group apart, and lanes read eight rows at once
#define I4W_STAGE (8 * I4W_ROW)
#define I4W_LD 144                 // a row of the block's sums: 16 pieces, 9 floats apart
#define I4W_POLLS (1 << 22)        // then a wait gives up
#define I4W_ERR_COPY 98            // a copy of W did not land, or its place was not given back
#define I4W_ERR_PRODUCT 99         // an operand or the sums did not come

struct Int4WideControl {
    unsigned long long w_full[I4W_RING], w_empty[I4W_RING], ready[I4W_A], done[I4W_A], x_full[I4W_A], sums;
    unsigned int tmem;
    int abort;
};

__device__ __forceinline__ void i4w_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// Two numbers: `t` holds 128 + q each, which bfloat16 can; the subtraction is exact
__device__ __forceinline__ uint32_t i4w_wide(uint32_t t, __nv_bfloat162 step, __nv_bfloat162 low) {
    const __nv_bfloat162 q = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&t), __floats2bfloat162_rn(128.f, 128.f));
    const __nv_bfloat162 r = __hfma2(q, step, low);
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float i4w_remote(uint32_t address, int rank) {
    uint32_t there;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}
__device__ __forceinline__ void i4w_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A warp's wait for a barrier's phase, asked for by one lane; bounded
__device__ __forceinline__ bool i4w_wait(void* bar, uint32_t parity, volatile int* abort, int* error_flag, int code) {
    bool there = true;
    if ((threadIdx.x & 31) == 0) {
        there = t5_bar_test(bar, parity);
        for (int i = 0; !there && i < I4W_POLLS && !*abort; ++i) there = t5_bar_test(bar, parity);
    }
    if (__all_sync(0xffffffffu, there)) return true;
    if ((threadIdx.x & 31) == 0 && !*abort) { *abort = 1; atomicExch(error_flag, code); }
    return false;
}

template <int BN, bool GLU>
__global__ void __launch_bounds__(I4W_THREADS, BN <= 64 ? 2 : 1)
int4_linear_tcgen05_kernel(const __grid_constant__ CUtensorMap map_x, const unsigned char* __restrict__ tiles, void* __restrict__ out, int f32, long long ld_out,
                           int M, int N, int K, GluShape unit, int ranks, int* __restrict__ error_flag) {
    constexpr int X_BYTES = BN * 256, TMEM = BN <= 64 ? 256 : 512, ACC = I4W_A * 64;      // up to 64 rows two blocks share an SM
    static_assert(ACC + BN <= TMEM, "tensor memory");
    extern __shared__ unsigned char i4w_raw[];
    unsigned char* const smem = (unsigned char*)(((uintptr_t)i4w_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* const ring = smem + I4W_A * X_BYTES;
    Int4WideControl* const ctl = reinterpret_cast<Int4WideControl*>(ring + I4W_RING * I4W_STAGE);
    volatile int* const abort = &ctl->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x, block = blockIdx.y, m0 = blockIdx.z * BN;
    const int groups = (K + I4_GROUP_W - 1) / I4_GROUP_W, ga = (int)((long long)groups * rank / ranks), n = (int)((long long)groups * (rank + 1) / ranks) - ga;
    gi_pdl_launch_dependents();
    if (threadIdx.x == 8 * 32) {
        for (int i = 0; i < I4W_RING; ++i) t5_bar_init(&ctl->w_full[i], 1), t5_bar_init(&ctl->w_empty[i], 8);
        for (int i = 0; i < I4W_A; ++i) t5_bar_init(&ctl->ready[i], 4), t5_bar_init(&ctl->done[i], 1), t5_bar_init(&ctl->x_full[i], 1);
        t5_bar_init(&ctl->sums, 1);
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 10) t5_alloc(&ctl->tmem, TMEM);
    t5_fence_before();
    __syncthreads();
    t5_fence_after();
    const uint32_t tmem = ctl->tmem;
    int sent = 0;                                                              // copies, or groups multiplied, of this warp's role

    if (warp == 8) {
        // lane l asks for row l of the block's eight rows of tiles
        const int half = N / 32;                                               // rows of tiles of the gate
        const int first = GLU ? block * 4 : block * 8, have = GLU ? half : (N + 15) / 16;
        const int row = GLU ? first + (lane & 3) : first + lane;
        const bool mine = lane < 8 && row < have;
        const int total = GLU ? 2 * min(4, have - first) : min(8, have - first);
        const unsigned char* src = tiles + ((size_t)(row + (GLU && lane >= 4 ? half : 0)) * groups + ga) * I4_TILE;
        const int copies = (n + I4W_SG - 1) / I4W_SG;
        for (int i = 0; i < copies; ++i, src += I4W_SG * I4_TILE, sent = i) {
            const int s = i % I4W_RING;
            const uint32_t bytes = min(I4W_SG, n - i * I4W_SG) * I4_TILE;
            if (i >= I4W_RING && !i4w_wait(&ctl->w_empty[s], (i / I4W_RING - 1) & 1, abort, error_flag, I4W_ERR_COPY)) break;
            if (lane == 0) t5_bar_expect(&ctl->w_full[s], total * bytes);
            __syncwarp();
            if (mine) i4w_copy(t5_smem(ring + s * I4W_STAGE + lane * I4W_ROW), src, bytes, t5_smem(&ctl->w_full[s]));
        }
    } else if (warp == 9) {
        gi_pdl_wait();
        for (int i = 0; i < n; sent = ++i) {
            const int s = i % I4W_A;
            if (i >= I4W_A && !i4w_wait(&ctl->done[s], (i / I4W_A - 1) & 1, abort, error_flag, I4W_ERR_PRODUCT)) break;
            if (lane == 0) {
                t5_bar_expect(&ctl->x_full[s], X_BYTES);
                t5_load_2d(smem + s * X_BYTES, &map_x, (ga + i) * I4_GROUP_W, m0, &ctl->x_full[s]);
                t5_load_2d(smem + s * X_BYTES + X_BYTES / 2, &map_x, (ga + i) * I4_GROUP_W + 64, m0, &ctl->x_full[s]);
            }
        }
    } else if (warp == 10) {
        // whole, so that the operands' addresses are known to be alike: issued by one lane of a divided warp, eight products took 650 cycles
        constexpr uint32_t idesc = t5_idesc(128, BN);
        const uint64_t xd = t5_desc<128>(t5_smem(smem));
        for (int i = 0; i < n; sent = ++i) {
            const int s = i % I4W_A;
            if (!i4w_wait(&ctl->x_full[s], (i / I4W_A) & 1, abort, error_flag, I4W_ERR_PRODUCT)) break;
            if (!i4w_wait(&ctl->ready[s], (i / I4W_A) & 1, abort, error_flag, I4W_ERR_PRODUCT)) break;
            t5_fence_after();
            if (t5_elect()) {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    t5_mma_ts(tmem + ACC, tmem + s * 64 + k * 8, xd + ((s * X_BYTES + (k >> 2) * BN * 128 + (k & 3) * 32) >> 4), idesc, (i | k) != 0);
                t5_commit(&ctl->done[s]);
                if (i == n - 1) t5_commit(&ctl->sums);
            }
            __syncwarp();
        }
    } else {
        // lane's output: its row of tiles, so that the eight lanes of a shared-memory phase read eight rows, and its place in it
        const int row = lane & 7, place = ((lane >> 3) & 1) * 8 + 2 * (warp & 3) + (lane >> 4);
        const int codes = row * I4W_ROW + place * 64, meta = row * I4W_ROW + I4_TILE_CODES + place * 4;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        for (int i = warp >> 2, seen = -1; i < n; i += 2) {
            const int copy = i / I4W_SG, s = copy % I4W_RING, a = i % I4W_A;
            if (copy != seen && !i4w_wait(&ctl->w_full[s], (copy / I4W_RING) & 1, abort, error_flag, I4W_ERR_COPY)) break;
            if (i >= I4W_A && !i4w_wait(&ctl->done[a], (i / I4W_A - 1) & 1, abort, error_flag, I4W_ERR_PRODUCT)) break;
            seen = copy;
            t5_fence_after();
            const unsigned char* w = ring + s * I4W_STAGE + i % I4W_SG * I4_TILE;
            const uint32_t pair = *reinterpret_cast<const uint32_t*>(w + meta), ss = __byte_perm(pair, 0, 0x1010), ll = __byte_perm(pair, 0, 0x3232);
            const __nv_bfloat162 step = *reinterpret_cast<const __nv_bfloat162*>(&ss), low = *reinterpret_cast<const __nv_bfloat162*>(&ll);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint4 c = *reinterpret_cast<const uint4*>(w + codes + q * 16);
                const uint32_t word[4] = {c.x, c.y, c.z, c.w};
                uint32_t r[16];
#pragma unroll
                for (int j = 0; j < 4; ++j) {                                  // numbers 0-3 below 1-4, 4-7 below 5-8: the pairs lie 16 bits apart
                    const uint32_t up = word[j] >> 4, lo = __byte_perm(word[j], up, 0x5410), hi = __byte_perm(word[j], up, 0x7632);
                    r[4 * j] = i4w_wide((lo & I4_NEAR) | 0x43004300u, step, low);
                    r[4 * j + 1] = i4w_wide((lo >> 8 & I4_NEAR) | 0x43004300u, step, low);
                    r[4 * j + 2] = i4w_wide((hi & I4_NEAR) | 0x43004300u, step, low);
                    r[4 * j + 3] = i4w_wide((hi >> 8 & I4_NEAR) | 0x43004300u, step, low);
                }
                t5_st16(lanes + a * 64 + q * 16, r);
            }
            t5_wait_st();
            t5_fence_before();
            __syncwarp();
            if (lane == 0) {
                if ((i + 2) / I4W_SG != copy) t5_bar_arrive(&ctl->w_empty[s]);
                t5_bar_arrive(&ctl->ready[a]);
            }
        }
        if (warp < 4 && i4w_wait(&ctl->sums, 0, abort, error_flag, I4W_ERR_PRODUCT)) {
            t5_fence_after();
            float* const sums = reinterpret_cast<float*>(smem) + row * 18 + (place >> 3) * 9 + (place & 7);
#pragma unroll 1
            for (int part = 0; part < BN; part += 16) {
                float v[16];
                t5_ld<16>(lanes + ACC + part, v);
                t5_wait_ld();
#pragma unroll
                for (int m = 0; m < 16; ++m) sums[(part + m) * I4W_LD] = v[m];
            }
            t5_fence_before();
        }
    }
    __syncwarp();
    gi_pdl_wait();                                                             // what follows writes
    if (ranks > 1) i4w_cluster_sync();
    else __syncthreads();
    {
        const int outs = GLU ? N / 2 : N, per = GLU ? 64 : 128, here = min(BN, M - m0);
        const int ma = here * rank / ranks, mb = here * (rank + 1) / ranks;
        const float* const sums = reinterpret_cast<const float*>(smem);
        for (int e = threadIdx.x; e < (mb - ma) * per; e += I4W_THREADS) {
            const int m = ma + e / per, c = e % per, o = block * per + c, at = m * I4W_LD + (c >> 3) * 9 + (c & 7);
            if (o >= outs) continue;
            float v = 0.f, up = 0.f;
            if (ranks == 1) {
                v = sums[at];
                if (GLU) up = sums[at + 72];
            } else {
                const uint32_t there = t5_smem(sums + at);
#pragma unroll 1
                for (int r = 0; r < ranks; ++r) {
                    v += i4w_remote(there, r);
                    if (GLU) up += i4w_remote(there + 288, r);
                }
            }
            if (GLU) v = glu_unit(v, up, unit);
            const size_t to = (size_t)(m0 + m) * ld_out + o;
            if (f32) reinterpret_cast<float*>(out)[to] = v;
            else reinterpret_cast<bf16*>(out)[to] = __float2bfloat16_rn(v);
        }
    }
    if (ranks > 1) i4w_cluster_sync();                                         // the others have read this block's sums
    else __syncthreads();
    if (*abort && warp >= 8) {
        // some role gave up, perhaps when others had left theirs: copies in flight land, and products end, before the block leaves and its
        // tensor memory is freed.  Warp 8's copies are counted by w_full, warp 9's by x_full, warp 10's products by done
        if (lane == 0) {
            int never = 0;
            const int ring = warp == 8 ? I4W_RING : I4W_A;
            unsigned long long* const bars = warp == 8 ? ctl->w_full : warp == 9 ? ctl->x_full : ctl->done;
            for (int j = max(0, sent - ring); j < sent; ++j) t5_bar_wait(&bars[j % ring], (j / ring) & 1, &never);
        }
        __syncwarp();
    }
    if (warp == 10) {
        t5_fence_after();
        t5_free(tmem, TMEM);
    }
}

template <int BN, bool GLU>
static int launch_int4_wide(const CUtensorMap& x, const unsigned char* tiles, void* out, int f32, long long ld, int M, int N, int K, const GluShape& unit,
                            int ranks, int* error_flag, cudaStream_t stream) {
    const size_t smem = (size_t)I4W_A * BN * 256 + I4W_RING * I4W_STAGE + sizeof(Int4WideControl) + 1024;
    if (int rc = gi_reserve_smem((const void*)int4_linear_tcgen05_kernel<BN, GLU>, smem, "gi_int4_linear_tcgen05")) return rc;
    const int per = GLU ? 64 : 128, outs = GLU ? N / 2 : N;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, (outs + per - 1) / per, (M + BN - 1) / BN);
    cfg.blockDim = dim3(I4W_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = gi_pdl_enabled() ? 2 : 1;
    cudaLaunchKernelEx(&cfg, int4_linear_tcgen05_kernel<BN, GLU>, x, tiles, out, f32, ld, M, N, K, unit, ranks, error_flag);
    return gi_check_launch("gi_int4_linear_tcgen05");
}

// K: the inner size, rounded up to a multiple of 8 (x has zeros there; what the codes have counts for nothing).  `ranks`: blocks that share the
// inputs (0: chosen here).
extern "C" int gi_int4_linear_tcgen05(const void* x, const void* tiles, void* out, int out_dtype, long long ld_out, int M, int N, int K,
                                      int glu, int kind, float alpha, float gate_max, float up_limit, float up_shift, int ranks,
                                      int* error_flag, void* stream) {
    GI_REQUIRE(M >= 1 && N > 0 && K > 0 && M < (1 << 21) && N < (1 << 22) && K < (1 << 30), "gi_int4_linear_tcgen05: %d rows, a weight of %d x %d", M, N, K);
    GI_REQUIRE(K % 8 == 0 && (uintptr_t)x % 16 == 0 && (uintptr_t)tiles % 16 == 0,
               "gi_int4_linear_tcgen05: operands must start on 16 bytes, the inner size %d be a multiple of 8", K);
    GI_REQUIRE(out_dtype == GI_DTYPE_BF16 || out_dtype == GI_DTYPE_F32, "gi_int4_linear_tcgen05: output dtype %d", out_dtype);
    GI_REQUIRE(!glu || (N % 32 == 0 && kind >= 0 && kind <= 2 && up_limit >= 0.f),
               "gi_int4_linear_tcgen05: a gated unit %d of %d outputs (halves must be multiples of 16)", kind, N);
    GI_REQUIRE(ld_out >= (glu ? N / 2 : N), "gi_int4_linear_tcgen05: output rows %lld apart hold no %d columns", ld_out, glu ? N / 2 : N);
    GI_REQUIRE(error_flag != nullptr, "gi_int4_linear_tcgen05: an error flag on the device is required");
    const int groups = (K + I4_GROUP_W - 1) / I4_GROUP_W, bn = M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const long long blocks = (long long)((glu ? N / 2 + 63 : N + 127) / (glu ? 64 : 128)) * ((M + bn - 1) / bn);
    // In ns: 500 a group of 128 inputs, 450 where two blocks share an SM, 1,000 a block and 800 more for each of a cluster (128 rows: 2,000 and
    // 3,000, their sums being larger); the SMs hold 148 blocks at once, 74 clusters of 2, 33 of 4 and rarely more than 44 of 3.  us by ranks:
    //    32 rows, 40 rows of tiles x 136 groups   1: 69   2: 38   3: 29   4: 36      128 rows, 32 x 96    1: 59   2: 38   3: 30   4: 27
    //    32 rows, 48 x 32                         1: 21   2: 14   3: 16   4: 14      128 rows, 192 x 32   1: 53   2: 57   3: 79
    //    32 rows, 192 x 32                        1: 35   2: 32   3: 38   4: 40      384 rows, 32 x 96    1: 59   2: 74   4: 76
    if (ranks == 0) {
        const int held[4] = {148, 74, 44, 33};
        long long best = 0;
        for (int r = 1; r <= 4 && r <= groups; ++r) {
            const long long load = (blocks + held[r - 1] - 1) / held[r - 1], each = (groups + r - 1) / r;
            const long long ns = bn <= 64 ? load * each * (load > 1 ? 450 : 500) + (load + 1) / 2 * (1000 + 800 * r) : load * (each * 500 + 2000 + 3000 * r);
            if (ranks == 0 || ns < best) best = ns, ranks = r;
        }
    }
    GI_REQUIRE(ranks >= 1 && ranks <= 8 && ranks <= groups, "gi_int4_linear_tcgen05: a cluster of %d blocks; 1 to 8 are possible, with a group of inputs each", ranks);
    const GluShape unit = {kind, alpha, gate_max, up_limit, up_shift};
    CUtensorMap xp;
    if (int rc = t5_make_map(&xp, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, x, M, K, (long long)K * 2, bn, 64, CU_TENSOR_MAP_SWIZZLE_128B, "gi_int4_linear_tcgen05")) return rc;
    const unsigned char* tp = (const unsigned char*)tiles;
    const int f32 = out_dtype == GI_DTYPE_F32;
    cudaStream_t s = (cudaStream_t)stream;
#define GI_I4W(BN, GLU) launch_int4_wide<BN, GLU>(xp, tp, out, f32, ld_out, M, N, K, unit, ranks, error_flag, s)
    if (bn == 32) return glu ? GI_I4W(32, true) : GI_I4W(32, false);
    if (bn == 64) return glu ? GI_I4W(64, true) : GI_I4W(64, false);
    return glu ? GI_I4W(128, true) : GI_I4W(128, false);
#undef GI_I4W
}
