// y = x W^T for a weight in 4 bits (layout: int4_weight.cu) and 1 to 16 rows of bfloat16 x: decode steps.
//
//   y[m, n] = sum over groups g of 128 inputs:  step[n, g] * sum_k q[n, k] x[m, k]  +  low[n, g] * sum_k x[m, k]
//
// bound by reading W once, 0.53 bytes a number.  16 outputs are the 16 rows of mma.sync m16n8k16, rows of x its 8 columns; the
// sums over q run on the tensor cores with the codes as they are (int4.cuh), step and low join in float32 once per group.
//
//  * K is cut over the CTAs of a cluster.  A CTA turns its slice of x into operand fragments in shared memory once (scaled
//    by a power of two per row and slice) and streams its slice of rows of tiles: each of 8 warps takes a row of tiles (with a
//    gated unit: a gate's and its up's) after the other.
//  * The 1,088 bytes of a tile come with cp.async into slots that only this warp reads, a few tiles in flight, so warps never
//    wait for each other while they stream.  W is nobody's output: the first tiles are on their way before the
//    kernel waits for the one that makes x.
//  * Behind a row of tiles every block sends its sums to the block of the cluster that finishes them (16-byte stores into
//    its shared memory), which adds them in rank order (the same bits from run to run) while the next row streams: two buffers, one
//    cluster barrier per row of tiles, arrived at behind the stores and waited for behind the next row's products.
#include "int4.cuh"
#include "glu.cuh"
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

#define I4L_WARPS 8
#define I4L_THREADS (I4L_WARPS * 32)
#define I4L_ODD 0x79800000u        // bits of 2^116: sums of rows with such numbers are not scaled back in float32

__device__ __forceinline__ void i4l_cp16(void* smem, const void* gmem) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem) : "memory");
}

// Eight consecutive inputs of a row of x from k on, zeros beyond K.  vec: K is a multiple of 8 and x starts on 16 bytes.
__device__ __forceinline__ uint4 i4l_load8(const bf16* row, int k, int K, int vec) {
    if (vec) return k < K ? __ldg(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0, 0, 0, 0);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = k + 2 * i < K ? *reinterpret_cast<const uint16_t*>(row + k + 2 * i) : 0;
        const uint32_t b = k + 2 * i + 1 < K ? *reinterpret_cast<const uint16_t*>(row + k + 2 * i + 1) : 0;
        w[i] = a | (b << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// NT: blocks of 8 rows of x.  RT: rows of tiles a warp takes at once (2 with GLU: a gate's and its up's).
// SLOTS: tiles a warp has in flight or in use.
template <int NT, int RT, bool GLU, int SLOTS>
__global__ void __launch_bounds__(I4L_THREADS, 2)
int4_linear_kernel(const bf16* __restrict__ x, const unsigned char* __restrict__ tiles, void* __restrict__ out, int out_f32,
                   int M, int N, int K, int groups, int slice, int units, int vec, GluShape unit, long long ld_out) {
    static_assert(!GLU || RT == 2, "a gate and its up");
    gi_pdl_launch_dependents();
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n" ::: "memory");       // waited for before the first store into another block
    constexpr int DEPTH = SLOTS / RT;                                // steps (RT tiles of one group) in flight
    extern __shared__ __align__(16) unsigned char i4_smem[];
    unsigned char* ring = i4_smem;                                       // [8 warps][slots][1088]
    // sums that this block finishes, as the lanes of a warp hold them: [2][unit of the pass][block that sends][RT][NT][32][4]; unit of
    // warp w belongs to block w mod ranks, as its (w / ranks)-th
    float4* sums = reinterpret_cast<float4*>(ring + I4L_WARPS * SLOTS * I4_TILE);
    const int owned = (I4L_WARPS + (int)cg::this_cluster().num_blocks() - 1) / (int)cg::this_cluster().num_blocks();
    const int half = owned * (int)cg::this_cluster().num_blocks() * RT * NT * 32;        // of one buffer, in float4
    unsigned char* frag = reinterpret_cast<unsigned char*>(sums + 2 * half);             // [slice][NT][4][32][16]
    float* xsum = reinterpret_cast<float*>(frag + (size_t)slice * NT * 2048);            // [slice][8 NT]
    __shared__ uint32_t s_most[8 * NT];                                  // bits of the largest magnitude of each row of x
    __shared__ uint32_t s_odd;                                           // rows with numbers too large to scale, or not finite

    cg::cluster_group cluster = cg::this_cluster();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
    const int n_cl = gridDim.x / ranks, cl = blockIdx.x / ranks;
    const int g0 = rank * slice, G = max(0, min(slice, groups - g0));

    // unit u: the row of tiles u (GLU: rows u and units + u), taken by cluster u mod n_cl as its (u / n_cl)-th, by warp
    // (u / n_cl) mod 8
    const int passes = (units + n_cl * I4L_WARPS - 1) / (n_cl * I4L_WARPS);
    auto unit_of = [&](int p) { return (p * I4L_WARPS + warp) * n_cl + cl; };
    auto row_tile = [&](int u, int r) { return GLU ? (r == 0 ? u : units + u) : u * RT + r; };
    const int row_tiles = (N + 15) / 16;
    unsigned char* my_ring = ring + warp * SLOTS * I4_TILE;

    // ---- the queue of tiles: step i is group i mod G of the warp's unit i / G
    int ip = 0, ig = 0, islot = 0;
    auto issue = [&]() {
        const int u = unit_of(ip);
        __syncwarp();                                                    // every lane is done with the slot that is filled again
        if (ip < passes && u < units) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const int rt = min(row_tile(u, r), row_tiles - 1);
                const unsigned char* src = tiles + ((size_t)rt * groups + g0 + ig) * I4_TILE;
                unsigned char* dst = my_ring + (islot * RT + r) * I4_TILE;
                i4l_cp16(dst + lane * 16, src + lane * 16);
                i4l_cp16(dst + 512 + lane * 16, src + 512 + lane * 16);
                if (lane < 4) i4l_cp16(dst + 1024 + lane * 16, src + 1024 + lane * 16);
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");           // an empty group when nothing is left
        if (++ig >= G) ig = 0, ++ip;
        islot = islot + 1 == DEPTH ? 0 : islot + 1;
    };
    if (G > 0) {
#pragma unroll
        for (int i = 0; i < DEPTH - 1; ++i) issue();
    }
    for (int i = threadIdx.x; i < 8 * NT; i += I4L_THREADS) s_most[i] = 0;
    if (threadIdx.x == 0) s_odd = 0;
    __syncthreads();
    gi_pdl_wait();

    // ---- x: item (group, block of 8 rows) per warp, lane = (row g, quarter t of 32 inputs)
    for (int i = warp; i < G * NT; i += I4L_WARPS) {                     // the largest magnitude of every row
        const int gi = i / NT, m = (i % NT) * 8 + g, k0 = (g0 + gi) * I4_GROUP_W + t * 32;
        if (m < M) {
            uint32_t most = 0;                                           // of |x| as bits: ordered like the numbers, NaN above all
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint4 v = i4l_load8(x + (size_t)m * K, k0 + 8 * j, K, vec);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) most = max(most, max((w[e] & 0x7FFFu) << 16, w[e] & 0x7FFF0000u));
            }
            atomicMax(&s_most[m], most);
        }
    }
    __syncthreads();
    for (int i = warp; i < G * NT; i += I4L_WARPS) {
        const int gi = i / NT, nt = i % NT, m = nt * 8 + g, k0 = (g0 + gi) * I4_GROUP_W + t * 32;
        int e;
        const uint32_t most = m < M ? s_most[m] : 0;
        const bool odd = most >= I4L_ODD;                                // 2^116 and more, infinite or NaN: summed the long way
        const float f = odd ? 0.f : i4_factor(__uint_as_float(most), e);
        if (odd && t == 0) atomicOr(&s_odd, 1u << m);
        uint4* dst = reinterpret_cast<uint4*>(frag + (size_t)(gi * NT + nt) * 2048) + lane;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (m < M && !odd) v = i4l_load8(x + (size_t)m * K, k0 + 8 * j, K, vec);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            float a[8];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                a[2 * h] = i4_bf16_low(w[h]) * f;
                a[2 * h + 1] = i4_bf16_high(w[h]) * f;
            }
            dst[j * 32] = i4_operand(a);
            sum += ((a[0] + a[1]) + (a[2] + a[3])) + ((a[4] + a[5]) + (a[6] + a[7]));
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (t == 0) xsum[gi * 8 * NT + m] = sum * I4_UNIT;               // as the products with codes are
    }
    __syncthreads();
    const uint32_t odd_rows = s_odd;
    float back[NT][2];                                                   // what brings the sums of rows 2t, 2t + 1 back
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int e;
            i4_factor(__uint_as_float(min(s_most[nt * 8 + 2 * t + h], I4L_ODD - 1)), e);
            back[nt][h] = i4_pow2(e - 14 + 24);
        }

    // ---- the sums of a finished pass that this block finishes: a warp per unit and block of 8 rows of x
    auto finish = [&](int p) {
        for (int i = warp; i < owned * NT; i += I4L_WARPS) {
            const int nt = i % NT, w = (i / NT) * ranks + rank, u = (p * I4L_WARPS + w) * n_cl + cl;
            if (w >= I4L_WARPS || u >= units) continue;
            const float4* src = sums + (p & 1) * half + (size_t)(i / NT) * ranks * RT * NT * 32 + lane;
            float4 v[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
                for (int c = 0; c < ranks; ++c) {
                    const float4 a = src[((c * RT + r) * NT + nt) * 32];
                    v[r].x += a.x, v[r].y += a.y, v[r].z += a.z, v[r].w += a.w;
                }
            }
            auto put = [&](int m, int n, float value) {
                if (m >= M || n >= (GLU ? N / 2 : N)) return;
                if (out_f32) reinterpret_cast<float*>(out)[(size_t)m * ld_out + n] = value;
                else reinterpret_cast<bf16*>(out)[(size_t)m * ld_out + n] = __float2bfloat16_rn(value);
            };
            const int m = nt * 8 + 2 * t;
            if (GLU) {
                const int n = u * 16 + g;
                put(m, n, glu_unit(v[0].x, v[RT - 1].x, unit));
                put(m + 1, n, glu_unit(v[0].y, v[RT - 1].y, unit));
                put(m, n + 8, glu_unit(v[0].z, v[RT - 1].z, unit));
                put(m + 1, n + 8, glu_unit(v[0].w, v[RT - 1].w, unit));
            } else {
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int n = (u * RT + r) * 16 + g;
                    put(m, n, v[r].x), put(m + 1, n, v[r].y), put(m, n + 8, v[r].z), put(m + 1, n + 8, v[r].w);
                }
            }
        }
    };

    int slot = 0;
    for (int p = 0; p < passes; ++p) {
        const int u = unit_of(p);
        float y[RT][NT][4];
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[r][nt][e] = 0.f;
        if (u < units) {
            for (int gi = 0; gi < G; ++gi) {
                issue();
                asm volatile("cp.async.wait_group %0;\n" ::"n"(DEPTH - 1) : "memory");
                __syncwarp();                                            // a tile's steps come with other lanes' copies
                uint4 c[RT][2];
                uint32_t mg[RT], mg8[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const unsigned char* tile = my_ring + (slot * RT + r) * I4_TILE;
                    c[r][0] = *reinterpret_cast<const uint4*>(tile + lane * 16);
                    c[r][1] = *reinterpret_cast<const uint4*>(tile + 512 + lane * 16);
                    mg[r] = *reinterpret_cast<const uint32_t*>(tile + 1024 + g * 4);
                    mg8[r] = *reinterpret_cast<const uint32_t*>(tile + 1024 + g * 4 + 32);
                }
                slot = slot + 1 == DEPTH ? 0 : slot + 1;
                float z[RT][NT][4], zl[RT][NT][4];                       // two chains of products
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) z[r][nt][e] = zl[r][nt][e] = 0.f;
                const uint4* fr = reinterpret_cast<const uint4*>(frag + (size_t)gi * NT * 2048) + lane;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4 b[NT];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) b[nt] = fr[(nt * 4 + j) * 32];
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const uint32_t w0 = j == 0 ? c[r][0].x : j == 1 ? c[r][0].y : j == 2 ? c[r][0].z : c[r][0].w;
                        const uint32_t w1 = j == 0 ? c[r][1].x : j == 1 ? c[r][1].y : j == 2 ? c[r][1].z : c[r][1].w;
                        const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            i4_mma(z[r][nt], w0 & I4_NEAR, w1 & I4_NEAR, w0 & I4_FAR, w1 & I4_FAR, b[nt].x, b[nt].y);
                            i4_mma(zl[r][nt], v0 & I4_NEAR, v1 & I4_NEAR, v0 & I4_FAR, v1 & I4_FAR, b[nt].z, b[nt].w);
                        }
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float2 xs = *reinterpret_cast<const float2*>(xsum + gi * 8 * NT + nt * 8 + 2 * t);
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        const float s = i4_bf16_low(mg[r]), s8 = i4_bf16_low(mg8[r]);
                        const float l = i4_bf16_high(mg[r]), l8 = i4_bf16_high(mg8[r]);
                        y[r][nt][0] = fmaf(l, xs.x, fmaf(s, z[r][nt][0] + zl[r][nt][0], y[r][nt][0]));
                        y[r][nt][1] = fmaf(l, xs.y, fmaf(s, z[r][nt][1] + zl[r][nt][1], y[r][nt][1]));
                        y[r][nt][2] = fmaf(l8, xs.x, fmaf(s8, z[r][nt][2] + zl[r][nt][2], y[r][nt][2]));
                        y[r][nt][3] = fmaf(l8, xs.y, fmaf(s8, z[r][nt][3] + zl[r][nt][3], y[r][nt][3]));
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) y[r][nt][e] *= back[nt][e & 1];
            // rows of x with numbers that no power of two brings into range: multiply-adds, as for any float32 product
            for (uint32_t left = odd_rows; left; left &= left - 1) {
                const int m = __ffs((int)left) - 1;
                for (int r = 0; r < RT; ++r) {
                    const int rt = min(row_tile(u, r), row_tiles - 1);
                    for (int o = 0; o < 16; ++o) {
                        float v = 0.f;
                        for (int gi = 0; gi < G; ++gi) {
                            const unsigned char* tile = tiles + ((size_t)rt * groups + g0 + gi) * I4_TILE;
                            const uint32_t meta = __ldg(reinterpret_cast<const uint32_t*>(tile + 1024 + o * 4));
                            for (int kk = lane; kk < I4_GROUP_W; kk += 32) {
                                const int k = (g0 + gi) * I4_GROUP_W + kk;
                                const uint32_t two = tile[(o >> 3) * 512 + ((o & 7) * 4 + (kk >> 5)) * 16 + ((kk & 31) >> 1)];
                                const float q = (float)((two >> (4 * (kk & 1))) & 15);
                                if (k < K) v = fmaf(fmaf(i4_bf16_low(meta), q, i4_bf16_high(meta)), to_f32(x[(size_t)m * K + k]), v);
                            }
                        }
                        v = warp_sum(v);
#pragma unroll
                        for (int rr = 0; rr < RT; ++rr)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    if (rr == r && nt * 8 + 2 * t + (e & 1) == m && g + 8 * (e >> 1) == o) y[rr][nt][e] = v;
                    }
                }
            }
        }
        asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
        if (p > 0) finish(p - 1);                                        // its sums are complete, and those of pass p - 2 done with
        if (u < units) {
            float4* dst = cluster.map_shared_rank(sums, warp % ranks) + (p & 1) * half + ((size_t)(warp / ranks) * ranks + rank) * RT * NT * 32 + lane;
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    dst[(r * NT + nt) * 32] = make_float4(y[r][nt][0], y[r][nt][1], y[r][nt][2], y[r][nt][3]);
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    finish(passes - 1);
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
}

// ------------------------------------------------------------------------------------------------ host
#include <mutex>
#include <vector>
namespace {
struct Residency { const void* kernel; int device, ranks; size_t smem; int clusters; };
std::mutex g_residency_mutex;
std::vector<Residency> g_residency;
}
// How many clusters of `ranks` CTAs of this kernel the current device holds at once (looked up once).
static int resident_clusters(const void* kernel, cudaLaunchConfig_t* cfg, int ranks, size_t smem, int* clusters) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) { gi_set_error("gi_int4_linear: %s", cudaGetErrorString(e)); return (int)e; }
    std::lock_guard<std::mutex> lock(g_residency_mutex);
    for (const Residency& r : g_residency)
        if (r.kernel == kernel && r.device == dev && r.ranks == ranks && r.smem == smem) { *clusters = r.clusters; return 0; }
    cfg->gridDim = dim3(ranks);
    e = cudaOccupancyMaxActiveClusters(clusters, kernel, cfg);
    if (e != cudaSuccess) { gi_set_error("gi_int4_linear: clusters of %d: %s", ranks, cudaGetErrorString(e)); return (int)e; }
    if (*clusters < 1) { gi_set_error("gi_int4_linear: no cluster of %d blocks with %zu bytes of shared memory fits this GPU", ranks, smem); return GI_ERR_ARGUMENT; }
    g_residency.push_back({kernel, dev, ranks, smem, *clusters});
    return 0;
}

template <int NT, int RT, bool GLU, int SLOTS>
static int launch_int4_linear(const bf16* x, const unsigned char* tiles, void* out, int out_f32, int M, int N, int K, int ranks,
                              GluShape unit, long long ld_out, cudaStream_t stream) {
    const int groups = (K - 1) / I4_GROUP_W + 1;
    const int slice = (groups + ranks - 1) / ranks;
    const int row_tiles = (N + 15) / 16, units = GLU ? row_tiles / 2 : (row_tiles + RT - 1) / RT;
    const size_t smem = (size_t)I4L_WARPS * SLOTS * I4_TILE + 2ull * ((I4L_WARPS + ranks - 1) / ranks) * ranks * RT * NT * 512 +
                        (size_t)slice * NT * 2048 + (size_t)slice * 8 * NT * 4;
    GI_REQUIRE(smem <= 226 * 1024, "gi_int4_linear: %d inputs are too many for %d rows", K, M);
    auto kernel = int4_linear_kernel<NT, RT, GLU, SLOTS>;
    if (int rc = gi_reserve_smem((const void*)kernel, smem, "gi_int4_linear")) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(I4L_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (int rc = resident_clusters((const void*)kernel, &cfg, ranks, smem, &clusters)) return rc;
    if (clusters > units) clusters = units;
    cfg.gridDim = dim3((unsigned)(clusters * ranks));
    cfg.numAttrs = gi_pdl_enabled() ? 2 : 1;
    const int vec = K % 8 == 0 && (uintptr_t)x % 16 == 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, x, tiles, out, out_f32, M, N, K, groups, slice, units, vec, unit, ld_out);
    if (e != cudaSuccess) { gi_set_error("gi_int4_linear: launch: %s", cudaGetErrorString(e)); return (int)e; }
    return gi_check_launch("gi_int4_linear");
}

// out [M, N] with rows ld_out apart = x [M, K] . W^T for 1 to 16 rows.  glu: W holds a gate's outputs and as many of an up,
// each a multiple of 16, and out [M, N / 2] is their gated unit.  ranks: blocks that share K (0: chosen here).
extern "C" int gi_int4_linear(const void* x, const void* tiles, void* out, int out_dtype, long long ld_out, int M, int N, int K,
                              int glu, int kind, float alpha, float gate_max, float up_limit, float up_shift, int ranks,
                              void* stream) {
    GI_REQUIRE(M >= 1 && M <= 16, "gi_int4_linear: %d rows; this kernel takes 1 to 16", M);
    GI_REQUIRE(N > 0 && K > 0 && N < (1 << 30) && K < (1 << 30), "gi_int4_linear: a weight of %d x %d", N, K);
    GI_REQUIRE((uintptr_t)tiles % 16 == 0, "gi_int4_linear: the tiles must start on 16 bytes");
    GI_REQUIRE(out_dtype == GI_DTYPE_BF16 || out_dtype == GI_DTYPE_F32, "gi_int4_linear: output dtype %d", out_dtype);
    GI_REQUIRE(!glu || (N % 32 == 0 && kind >= 0 && kind <= 2 && up_limit >= 0.f),
               "gi_int4_linear: a gated unit %d of %d outputs (halves must be multiples of 16)", kind, N);
    GI_REQUIRE(ld_out >= (glu ? N / 2 : N), "gi_int4_linear: output rows %lld apart hold no %d columns", ld_out, glu ? N / 2 : N);
    GI_REQUIRE(ranks >= 0 && ranks <= 8, "gi_int4_linear: a cluster of %d blocks; 1 to 8 are possible", ranks);
    const int groups = (K - 1) / I4_GROUP_W + 1;
    if (ranks == 0) ranks = groups < 8 ? (groups < 2 ? 1 : groups / 2) : 8;
    const GluShape unit = {kind, alpha, gate_max, up_limit, up_shift};
    const bf16* xp = (const bf16*)x;
    const unsigned char* tp = (const unsigned char*)tiles;
    const int f32 = out_dtype == GI_DTYPE_F32;
    cudaStream_t s = (cudaStream_t)stream;
#define GI_I4(NT, RT, GLU, SLOTS) launch_int4_linear<NT, RT, GLU, SLOTS>(xp, tp, out, f32, M, N, K, ranks, unit, ld_out, s)
    if (M <= 8) return glu ? GI_I4(1, 2, true, 8) : GI_I4(1, 1, false, 8);
    return glu ? GI_I4(2, 2, true, 6) : GI_I4(2, 1, false, 6);
#undef GI_I4
}
