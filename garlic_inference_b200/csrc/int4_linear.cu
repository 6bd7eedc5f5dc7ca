// y = x W^T for a weight in 4 bits (layout: int4_weight.cu) and 1 to 16 rows of bfloat16 x: decode steps.
//
//   y[m, n] = sum over groups g of 128 inputs:  step[n, g] * sum_k q[n, k] x[m, k]  +  low[n, g] * sum_k x[m, k]
//
// bound by reading W once, 0.53 bytes a number, which leaves an SM 46 cycles for a tile (16 outputs x 128 inputs, 1,088 bytes).  16 outputs
// are the 16 rows of mma.sync m16n8k16, rows of x its 8 columns; the sums over q run on the tensor cores with the codes
// as they are (int4.cuh), step and low join in float32 once per group.
//
//  * K is cut over the blocks of a cluster, and a block's slice into parts where it has few rows of tiles: a warp sums one part of
//    one row of tiles in registers, after the other, and no warp waits for another.
//  * A warp's tiles come by bulk copies, `sg` groups (4, or 2) at a time, into a ring of its own, asked for by four warps that do nothing else (a
//    lane a ring: done by the multiplying warps it took a sixth of their time, and one warp for all 16 rings came too late with every
//    second copy); one lane waits (32 lanes at a barrier take 700 cycles, one 75).  W is nobody's output: in a recorded step the rings
//    fill before the kernel waits for the one that makes x.  Otherwise, where W is more than the rings hold, half a copy
//    goes ahead of x and the others follow when x is here: behind 18 MB of W, x took 3.5 us.
//  * A block turns its slice of x into operand fragments in shared memory once, scaled by a power of two per row and group.
//  * Sums go to the block of the cluster that finishes the row, 16 bytes at a time by stores that count on that block's barrier as they
//    land; it adds them in a fixed order: the same bits from run to run.
//
// Instructions that a launch runs only once cost about 20 cycles each: they come from the instruction cache's next level, for all
// warps alike.  So what is not the loop over tiles is kept small and rolled up, above all the conversion of x (unrolled for 32 inputs a
// lane it took 2.8 us of a launch), and counts that need divisions come from the host.
//
// The product itself is 81 instructions a tile, 33 to 38 cycles of 16 warps (measured on tiles that stay in shared memory; 46 of the 81 are
// on the integer pipe, 23 cycles).  What else was tried around it, 8 x 4096 x 24576 with a gated unit: 16-byte copies by all lanes into
// rings, 26 us (2.4 us to issue 120 KB an SM); tiles straight into registers, two ahead in 32 warps or four in 16, 21 us; warps that own a group
// of inputs and meet once a unit to add up, or leave that to warps of their own, 18 to 22 us.
#include "int4.cuh"
#include "glu.cuh"
#include "tcgen05.cuh"

#define I4L_ODD 0x79800000u        // bits of 2^116: sums of rows with such numbers are not scaled back in float32
#define I4L_STAGES 2               // copies a warp has in flight or in use
#define I4L_COPIERS 4              // warps that ask for copies
#define I4L_ERR_COPY 95            // a copy of W did not land
#define I4L_ERR_SUMS 96            // another block's sums did not arrive
#define I4L_POLLS (1 << 22)        // of a copying lane for room; a poll that fails takes some tens of cycles
#define I4L_ERR_ROOM 97            // a place in a ring was not given back

__device__ __forceinline__ void i4l_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// 16 bytes into shared memory of a block of the cluster (`where`, `bar`: addresses there), counted on its barrier as they land
__device__ __forceinline__ void i4l_send(uint32_t where, const float (&v)[4], uint32_t bar) {
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];"
                 ::"r"(where), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t i4l_remote(uint32_t address, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(address), "r"(rank));
    return r;
}
// A barrier's phase, asked for by one lane of the warp (32 asking at once take 700 cycles, one 75); bounded.  One that gives up
// says so and goes on.
__device__ __forceinline__ void i4l_wait(void* bar, uint32_t parity, volatile int* abort, int* error_flag, int code) {
    if ((threadIdx.x & 31) == 0 && !t5_bar_wait(bar, parity, abort)) {
        *abort = 1;
        atomicExch(error_flag, code);
    }
    __syncwarp();
}

// The end of a warp that gave up a wait: what is on its way into the block's shared memory lands before the block leaves (again with a limit).
// First its ring's copies; the copying lane leaves 1 + their number in `left`.  Then other blocks' sums: those blocks' waits are bounded
// too, and the barrier of the cluster counts who has left, so behind it all sums are under way and the count of bytes says when they are here.
__device__ __noinline__ void i4l_leave(volatile int* left, uint64_t* full, uint64_t* arrived, bool owned, bool cluster) {
    const bool first = (threadIdx.x & 31) == 0;
    int never = 0;
    if (first) {
        int n = 0;
        for (int i = 0; i < I4L_POLLS && n == 0; ++i) n = *left;
        for (int j = max(0, n - 1 - I4L_STAGES); j < n - 1; ++j) t5_bar_wait(&full[j % I4L_STAGES], (j / I4L_STAGES) & 1, &never);
    }
    __syncwarp();
    if (cluster) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    if (first && owned) t5_bar_wait(arrived, 0, &never);
    __syncwarp();
}

// Eight consecutive inputs of a row of x from k on, zeros beyond K.  vec: K is a multiple of 8 and x starts on 16 bytes.
__device__ __noinline__ uint4 i4l_load8_plain(const bf16* row, int k, int K) {
    uint32_t w[4];
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = k + 2 * i < K ? *reinterpret_cast<const uint16_t*>(row + k + 2 * i) : 0;
        const uint32_t b = k + 2 * i + 1 < K ? *reinterpret_cast<const uint16_t*>(row + k + 2 * i + 1) : 0;
        w[i] = a | (b << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Row m of x times output o of a row of tiles over groups g_first .. g_end - 1, multiply-adds in float32: for rows with
// numbers that no power of two brings into range.  The whole warp; every lane gets the sum.
__device__ __noinline__ float i4l_long_way(const bf16* x, const unsigned char* row, int m, int o, int g_first, int g_end, int K) {
    const int lane = threadIdx.x & 31;
    float v = 0.f;
    for (int gi = g_first; gi < g_end; ++gi) {
        const unsigned char* tile = row + (size_t)gi * I4_TILE;
        const uint32_t meta = __ldg(reinterpret_cast<const uint32_t*>(tile + I4_TILE_CODES + o * 4));
        for (int kk = lane; kk < I4_GROUP_W; kk += 32) {
            const int k = gi * I4_GROUP_W + kk;
            const uint32_t two = tile[(o >> 3) * 512 + ((o & 7) * 4 + (kk >> 5)) * 16 + ((kk & 31) >> 1)];
            const float q = (float)((two >> (4 * (kk & 1))) & 15);
            if (k < K) v = fmaf(fmaf(i4_bf16_low(meta), q, i4_bf16_high(meta)), to_f32(x[(size_t)m * K + k]), v);
        }
    }
    return warp_sum(v);
}

// NT: blocks of 8 rows of x.
template <int NT, int WARPS, bool GLU>
__global__ void __launch_bounds__((WARPS + I4L_COPIERS) * 32, 1)
int4_linear_kernel(const bf16* __restrict__ x, const unsigned char* __restrict__ tiles, void* __restrict__ out, int out_f32,
                   int M, int N, int K, int groups, int slice, int log_parts, int units, int units_each, int units_left, int vec,
                   int x_first, int hold, int sg, GluShape act, long long ld_out, int* __restrict__ error_flag) {
    gi_pdl_launch_dependents();
    extern __shared__ __align__(16) unsigned char i4_smem[];
    __shared__ __align__(8) uint64_t s_full[WARPS][I4L_STAGES], s_room[WARPS][I4L_STAGES], s_arrived, s_x;
    __shared__ uint32_t s_odd;                                           // rows of x that are summed the long way
    __shared__ int s_abort, s_left[WARPS];                               // 1 + the copies of a ring, when its lane has left
    constexpr int R = GLU ? 2 : 1;                                       // rows of tiles of a unit
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
    // blocks of a cluster lie along y and share K; cluster cl has units cl, cl + n_cl, ..: units_each, and one more of the first units_left
    const int rank = blockIdx.y, ranks = gridDim.y, n_cl = gridDim.x, cl = blockIdx.x;
    const int g0 = rank * slice, G = max(0, min(slice, groups - g0));    // this block's groups
    const int my_units = units_each + (cl < units_left ? 1 : 0), my_rows = my_units * R, owned = my_units > rank ? (my_units - rank + ranks - 1) / ranks : 0;
    // warp w: part w mod parts of the slice, rows w / parts, + stride, .. of the cluster's
    const int parts = 1 << log_parts, stride = WARPS >> log_parts;
    auto begin_of = [&](int w) { return ((w & (parts - 1)) * G) >> log_parts; };
    auto end_of = [&](int w) { return (((w & (parts - 1)) + 1) * G) >> log_parts; };
    auto row_of = [&](int i) { return GLU ? (i >> 1) * n_cl + cl + (i & 1) * units : i * n_cl + cl; };
    const uint32_t row_bytes = (uint32_t)groups * I4_TILE;

    // ---- x: item i is rows 2 (i mod 4 NT), + 1 of group i / (4 NT); half a warp has a row, a lane 8 inputs
    const int half = lane >> 4, chunk = lane & 15;
    auto load_x = [&](int i) {
        const int m = (i % (4 * NT)) * 2 + half, k = (g0 + i / (4 * NT)) * I4_GROUP_W + chunk * 8;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (i < G * 4 * NT && m < M) {
            if (!vec) v = i4l_load8_plain(x + (size_t)m * K, k, K);
            else if (k < K) v = __ldg(reinterpret_cast<const uint4*>(x + (size_t)m * K + k));
        }
        return v;
    };
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (x_first && warp < WARPS) raw = load_x(warp);                     // no kernel before this one is still to write x
    if (warp == WARPS) {
        if (lane < WARPS) {
            s_left[lane] = 0;
#pragma unroll
            for (int i = 0; i < I4L_STAGES; ++i) t5_bar_init(&s_full[lane][i], 1), t5_bar_init(&s_room[lane][i], 1);
        }
        if (lane == 0) {
            t5_bar_init(&s_arrived, 1);
            t5_bar_init(&s_x, WARPS);
            s_odd = 0, s_abort = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        if (lane == 0) t5_bar_expect(&s_arrived, owned * R * ranks * parts * NT * 512);
        __syncwarp();
    }
    __syncthreads();                                                     // the barriers and s_odd are there
    if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");       // waited for before sums are sent
    if (warp >= WARPS) {
        // ================================================================ the copying warps: a lane fills a ring
        const int w = (warp - WARPS) + lane * I4L_COPIERS, ga = begin_of(w), gb = end_of(w);
        int row = w >> log_parts, gi = ga, slot = 0, round = 0;
        bool left = w < WARPS && gb > ga && row < my_rows;
        const unsigned char* const base = tiles + (size_t)g0 * I4_TILE;
        const uint32_t ring = t5_smem(i4_smem) + w * (I4L_STAGES * sg * I4_TILE);
        auto copy = [&](int from, int to) {                              // groups from .. to - 1 of the next copy's; the first part says how many come
            const int count = min(sg, gb - gi), last = min(to, count);
            const uint32_t bar = t5_smem(&s_full[w][slot]);
            if (from == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(count * I4_TILE) : "memory");
            if (last > from)
                i4l_copy(ring + (slot * sg + from) * I4_TILE, base + (size_t)row_of(row) * row_bytes + (gi + from) * I4_TILE, (last - from) * I4_TILE, bar);
        };
        int from = 0;
        if (hold) {
            if (left) copy(0, sg / 2);
            from = sg / 2;
            i4l_wait(&s_x, 0, &s_abort, error_flag, I4L_ERR_ROOM);
        }
        for (int spin = 0; left; ++spin) {                               // the lanes go their own ways
            if (round == 0 || t5_bar_test(&s_room[w][slot], (round - 1) & 1)) {
                copy(from, sg);
                from = 0, spin = 0, gi += sg;
                if (gi >= gb) {
                    gi = ga, row += stride;
                    left = row < my_rows;
                }
                if (++slot == I4L_STAGES) slot = 0, ++round;
            } else if (spin > I4L_POLLS || *(volatile int*)&s_abort) {      // bounded: the warps that wait for these copies give up too
                s_abort = 1;
                atomicExch(error_flag, I4L_ERR_ROOM);
                break;
            }
        }
        if (w < WARPS) *(volatile int*)&s_left[w] = 1 + round * I4L_STAGES + slot;
        return;
    }
    gi_pdl_wait();
    if (!x_first) raw = load_x(warp);
    const int part = warp & (parts - 1), ga = begin_of(warp), gb = end_of(warp);
    unsigned char* const ring = i4_smem + warp * (I4L_STAGES * sg * I4_TILE);
    // units that this block finishes [unit][row][block that sends, part][NT][32][4] | fragments of x [slice][NT][4][32] | [slice][8 NT] of
    // what brings sums back and times the sum of x
    float4* sums = reinterpret_cast<float4*>(i4_smem + WARPS * I4L_STAGES * sg * I4_TILE);
    uint4* frag = reinterpret_cast<uint4*>(sums + (size_t)((units_each + (units_left ? 1 : 0) + ranks - 1) / ranks) * R * ranks * parts * NT * 32);
    float2* xmeta = reinterpret_cast<float2*>(frag + (size_t)slice * NT * 128);
    if (warp >= G * 4 * NT && lane == 0) t5_bar_arrive(&s_x);
#pragma unroll 1
    for (int i = warp; i < G * 4 * NT; i += WARPS) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t most = 0;                                               // of |x| as bits: ordered like the numbers, NaN above all
#pragma unroll
        for (int h = 0; h < 4; ++h) most = max(most, max((w[h] & 0x7FFFu) << 16, w[h] & 0x7FFF0000u));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        if (i == warp && lane == 0) t5_bar_arrive(&s_x);                 // this warp's first x is here
        const bool odd = most >= I4L_ODD;                                // 2^116 and more, infinite or NaN
        int e;
        const float scale = i4_factor(odd ? 0.f : __uint_as_float(most), e);
        float a[8], sum = 0.f;
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            a[2 * h] = odd ? 0.f : i4_bf16_low(w[h]) * scale;
            a[2 * h + 1] = odd ? 0.f : i4_bf16_high(w[h]) * scale;
            sum += a[2 * h] + a[2 * h + 1];
        }
        const int gi = i / (4 * NT), m = (i % (4 * NT)) * 2 + half;
        frag[((gi * NT + (m >> 3)) * 4 + (chunk & 3)) * 32 + (m & 7) * 4 + (chunk >> 2)] = i4_operand(a);
        raw = load_x(i + WARPS);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (chunk == 0) {
            const float back = i4_pow2(e - 14);
            xmeta[gi * 8 * NT + m] = make_float2(back * 16777216.f, back * sum);      // codes count in 2^-24
            if (odd) atomicOr(&s_odd, 1u << m);
        }
    }
    asm volatile("bar.sync 1, %0;\n" ::"n"(WARPS * 32) : "memory");      // the multiplying warps: all of x is there
    if (ranks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    const uint32_t odd_rows = s_odd;

    // ---- the products
    int row = warp >> log_parts;
    float y[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) y[nt][e] = 0.f;
    auto close_row = [&]() {                                             // the row's sums go where they are finished
#pragma unroll 1
        for (uint32_t left = odd_rows; left; left &= left - 1) {
            const int m = __ffs((int)left) - 1;
            const unsigned char* at = tiles + (size_t)row_of(row) * row_bytes;
#pragma unroll 1
            for (int o = 0; o < 16; ++o) {
                const float v = i4l_long_way(x, at, m, o, g0 + ga, g0 + gb, K);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (nt * 8 + 2 * t4 + (e & 1) == m && g + 8 * (e >> 1) == o) y[nt][e] = v;
            }
        }
        const int unit = row / R, owner = unit % ranks;
        const uint32_t at = t5_smem(sums + ((((size_t)(unit / ranks) * R + row % R) * ranks + rank) * parts + part) * NT * 32 + lane);
        const uint32_t to = ranks > 1 ? i4l_remote(at, owner) : at, bar = ranks > 1 ? i4l_remote(t5_smem(&s_arrived), owner) : t5_smem(&s_arrived);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            i4l_send(to + nt * 512, y[nt], bar);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[nt][e] = 0.f;
        }
    };
    int slot = 0;
    uint32_t phase = 0;
#pragma unroll 1
    for (; row < my_rows; row += stride) {
#pragma unroll 1
        for (int gi = ga; gi < gb; gi += 2) {
            const int in = (gi - ga) & (sg - 1);                     // place in the copy
            if (in == 0) i4l_wait(&s_full[warp][slot], phase, &s_abort, error_flag, I4L_ERR_COPY);
            // two groups side by side; of a last one alone the second's steps and low values are taken as zeros
            const unsigned char* tile = ring + (slot * sg + in) * I4_TILE;
            const bool two = gi + 1 < gb;
            uint4 c[2][2];
            uint32_t meta[2][2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                c[r][0] = *reinterpret_cast<const uint4*>(tile + r * I4_TILE + lane * 16);
                c[r][1] = *reinterpret_cast<const uint4*>(tile + r * I4_TILE + 512 + lane * 16);
                meta[r][0] = *reinterpret_cast<const uint32_t*>(tile + r * I4_TILE + I4_TILE_CODES + g * 4);
                meta[r][1] = *reinterpret_cast<const uint32_t*>(tile + r * I4_TILE + I4_TILE_CODES + 32 + g * 4);
            }
            if (!two) meta[1][0] = meta[1][1] = 0;
            const uint4* fr[2] = {frag + gi * (NT * 128) + lane, frag + (two ? gi + 1 : gi) * (NT * 128) + lane};
            float z[2][NT][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const uint32_t w0 = j == 0 ? c[r][0].x : j == 1 ? c[r][0].y : j == 2 ? c[r][0].z : c[r][0].w;
                    const uint32_t w1 = j == 0 ? c[r][1].x : j == 1 ? c[r][1].y : j == 2 ? c[r][1].z : c[r][1].w;
                    const uint32_t v0 = w0 >> 8, v1 = w1 >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint4 b = fr[r][(nt * 4 + j) * 32];
                        if (j == 0) i4_mma_first(z[r][nt], w0 & I4_NEAR, w1 & I4_NEAR, w0 & I4_FAR, w1 & I4_FAR, b.x, b.y);
                        else i4_mma(z[r][nt], w0 & I4_NEAR, w1 & I4_NEAR, w0 & I4_FAR, w1 & I4_FAR, b.x, b.y);
                        i4_mma(z[r][nt], v0 & I4_NEAR, v1 & I4_NEAR, v0 & I4_FAR, v1 & I4_FAR, b.z, b.w);
                    }
                }
            if (in == sg - 2 || gi + 2 >= gb) {                      // the copy's last two
                __syncwarp();                                            // every lane has read it: its place is filled again
                if (lane == 0) t5_bar_arrive(&s_room[warp][slot]);
                slot ^= 1;
                if (slot == 0) phase ^= 1;
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float s = i4_bf16_low(meta[r][0]), s8 = i4_bf16_low(meta[r][1]), l = i4_bf16_high(meta[r][0]), l8 = i4_bf16_high(meta[r][1]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float4 xm = *reinterpret_cast<const float4*>(xmeta + ((two ? gi + r : gi) * NT + nt) * 8 + 2 * t4);
                    // z < 4 and xm.x < 2^126: their product is finite, a step times xm.x need not be
                    y[nt][0] = fmaf(l, xm.y, fmaf(s, xm.x * z[r][nt][0], y[nt][0]));
                    y[nt][1] = fmaf(l, xm.w, fmaf(s, xm.z * z[r][nt][1], y[nt][1]));
                    y[nt][2] = fmaf(l8, xm.y, fmaf(s8, xm.x * z[r][nt][2], y[nt][2]));
                    y[nt][3] = fmaf(l8, xm.w, fmaf(s8, xm.z * z[r][nt][3], y[nt][3]));
                }
            }
        }
        close_row();
    }

    // ---- the units that this block finishes, a warp each, when all their sums are here (the block stays until then: nobody sends to one
    // that has gone)
    if (owned) {
        i4l_wait(&s_arrived, 0, &s_abort, error_flag, I4L_ERR_SUMS);
        for (int i = warp; i < owned * NT; i += WARPS) {
            const int u = (i / NT * ranks + rank) * n_cl + cl, nt = i % NT;
            float4 v[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                v[r] = make_float4(0.f, 0.f, 0.f, 0.f);
                const float4* from = sums + (((size_t)(i / NT) * R + r) * ranks * parts * NT + nt) * 32 + lane;
#pragma unroll 4
                for (int k = 0; k < ranks * parts; ++k) {
                    const float4 a = from[k * NT * 32];
                    v[r].x += a.x, v[r].y += a.y, v[r].z += a.z, v[r].w += a.w;
                }
            }
            const float value[4] = {v[0].x, v[0].y, v[0].z, v[0].w}, up[4] = {v[R - 1].x, v[R - 1].y, v[R - 1].z, v[R - 1].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int m = nt * 8 + 2 * t4 + (e & 1), n = u * 16 + g + 8 * (e >> 1);
                if (m >= M || n >= (GLU ? N / 2 : N)) continue;
                const float a = GLU ? glu_unit(value[e], up[e], act) : value[e];
                if (out_f32) reinterpret_cast<float*>(out)[(size_t)m * ld_out + n] = a;
                else reinterpret_cast<bf16*>(out)[(size_t)m * ld_out + n] = __float2bfloat16_rn(a);
            }
        }
    }
    if (*(volatile int*)&s_abort) i4l_leave(&s_left[warp], s_full[warp], &s_arrived, owned > 0, ranks > 1);
}

// ------------------------------------------------------------------------------------------------ host
#include <atomic>
#define I4L_DEVICES 64
#define I4L_WARPS 16
#define I4L_SMEM (214 * 1024)      // of an SM's 227 KB: what a product may take
// Clusters of 1 to 8 blocks, one to an SM, that a B200 was seen to hold at once.  They differ a little from device to device (45 of 3, 26
// of 5, 22 of 6, 15 of 7 on another): the cut, and so the order of the sums, is chosen with these, that a result has the same bits on all.
static const int i4l_b200[9] = {0, 148, 74, 48, 33, 28, 21, 18, 15};
// What the current device holds, asked for once a device: how many are launched, and so what a product's sums take in shared memory.  Where
// there is no device to ask (sizes worked out on a host), the numbers above.
struct Int4Held { int clusters[9]; };
static int clusters_held(Int4Held* held) {
    static std::atomic<int> seen[I4L_DEVICES][9];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) {
        cudaGetLastError();
        for (int r = 0; r <= 8; ++r) held->clusters[r] = i4l_b200[r];
        return 0;
    }
    // every instance of the kernel has the same threads, and takes more than half an SM's shared memory: one stands for all
    auto kernel = int4_linear_kernel<1, I4L_WARPS, false>;
    held->clusters[0] = 0;
    for (int r = 1; r <= 8; ++r) {
        int n = dev < I4L_DEVICES ? seen[dev][r].load(std::memory_order_relaxed) : 0;
        if (n == 0) {
            if (int rc = gi_reserve_smem((const void*)kernel, 224 * 1024, "gi_int4_linear")) return rc;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1, r), cfg.blockDim = dim3((I4L_WARPS + I4L_COPIERS) * 32), cfg.dynamicSmemBytes = I4L_SMEM;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1, attr[0].val.clusterDim.y = r, attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr, cfg.numAttrs = 1;
            const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, (const void*)kernel, &cfg);
            if (e != cudaSuccess) { gi_set_error("gi_int4_linear: clusters of %d: %s", r, cudaGetErrorString(e)); return (int)e; }
            if (n < 1) n = -1;                                           // none fits: that number of blocks is not taken
            if (dev < I4L_DEVICES) seen[dev][r].store(n, std::memory_order_relaxed);
        }
        held->clusters[r] = n;
    }
    return 0;
}

// How a product is cut: blocks that share K, parts that a block's warps take of its slice, groups of a copy; ranks 0: it does not fit.
struct Int4Cut { int ranks, parts, sg; };
static size_t smem_of(int ranks, int parts, int sg, int groups, int units, int clusters, int nt, int rows_of_unit) {
    return (size_t)I4L_WARPS * I4L_STAGES * sg * I4_TILE + (size_t)((groups + ranks - 1) / ranks) * nt * (2048 + 64) +
           (size_t)(((units + clusters - 1) / clusters + ranks - 1) / ranks) * rows_of_unit * ranks * parts * nt * 512;
}
// The cut whose busiest warp has the least to do: tiles to multiply, rows of tiles to hand over (as long as a tile), pairs of rows of x to
// convert (two tiles), sums of a row to add up (an eighth); an even number of blocks, or one (clusters of 3 or 5 left a recorded step's SMs idle: 28 us where
// 4 took 16).  Best and chosen, us: 8 x 4096 x 4096 6.9 in 4 blocks and 2 parts, chosen; 8 x 12288 x 4096 11.8 in 6 and 1, chosen; 8 x 4096 x 24576 gated 16.1 in 4 and 1, chosen.
static Int4Cut cut_of(int M, int N, int K, int glu, int ranks, int parts, const Int4Held& held) {
    const int groups = (K - 1) / I4_GROUP_W + 1, row_tiles = (N + 15) / 16, units = glu ? row_tiles / 2 : row_tiles, nt = M > 8 ? 2 : 1, R = glu ? 2 : 1;
    Int4Cut cut = {0, 0, 0};
    long long best = -1;
    for (int r = 1; r <= 8; ++r) {
        if (ranks ? r != ranks : (r > 1 && r % 2)) continue;
        if (r > groups || held.clusters[r] < 1) continue;
        const int slice = (groups + r - 1) / r, clusters = units < held.clusters[r] ? units : held.clusters[r],
                  rows = R * ((units + i4l_b200[r] - 1) / i4l_b200[r]);
        for (int p = 1; p <= 16 && p <= slice; p *= 2) {
            if (parts && p != parts) continue;
            const int sg = smem_of(r, p, 4, groups, units, clusters, nt, R) <= I4L_SMEM && nt == 1 ? 4 : 2;
            if (smem_of(r, p, sg, groups, units, clusters, nt, R) > I4L_SMEM) continue;
            const int stride = I4L_WARPS / p;
            const long long turns = (rows + stride - 1) / stride;
            const long long cost = 8 * (turns * ((slice + p - 1) / p + 1) + 2 * ((slice * 4 * nt + I4L_WARPS - 1) / I4L_WARPS)) + r * p;
            if (best < 0 || cost < best) best = cost, cut = {r, p, sg};
        }
    }
    return cut;
}

template <int NT, bool GLU>
static int launch_int4_linear(const bf16* x, const unsigned char* tiles, void* out, int out_f32, int M, int N, int K, Int4Cut cut,
                              const Int4Held& held, GluShape act, long long ld_out, int* error_flag, cudaStream_t stream) {
    const int groups = (K - 1) / I4_GROUP_W + 1, row_tiles = (N + 15) / 16, units = GLU ? row_tiles / 2 : row_tiles;
    auto kernel = int4_linear_kernel<NT, I4L_WARPS, GLU>;
    constexpr int WARPS = I4L_WARPS, R = GLU ? 2 : 1;
    const int pick = cut.ranks, pick_parts = cut.parts, slice = (groups + pick - 1) / pick;
    int log_parts = 0;
    while ((1 << log_parts) < pick_parts) ++log_parts;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3((WARPS + I4L_COPIERS) * 32);
    cfg.dynamicSmemBytes = 160 * 1024;                                   // more than half an SM's: one block each
    cfg.stream = stream;
    if (int rc = gi_reserve_smem((const void*)kernel, 224 * 1024, "gi_int4_linear")) return rc;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1;
    attr[0].val.clusterDim.y = pick;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const int clusters = units < held.clusters[pick] ? units : held.clusters[pick];
    const size_t smem = smem_of(pick, pick_parts, cut.sg, groups, units, clusters, NT, R);
    if (smem > cfg.dynamicSmemBytes) cfg.dynamicSmemBytes = smem;
    cfg.gridDim = dim3(clusters, pick);
    cfg.numAttrs = gi_pdl_enabled() ? 2 : 1;
    const int vec = K % 8 == 0 && (uintptr_t)x % 16 == 0;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, x, tiles, out, out_f32, M, N, K, groups, slice, log_parts, units, units / clusters, units % clusters,
                                       vec, gi_pdl_enabled() ? 0 : 1,
                                       !gi_pdl_enabled() && (size_t)row_tiles * groups * I4_TILE > (size_t)148 * WARPS * I4L_STAGES * cut.sg * I4_TILE, cut.sg, act,
                                       ld_out, error_flag);
    if (e != cudaSuccess) { gi_set_error("gi_int4_linear: launch: %s", cudaGetErrorString(e)); return (int)e; }
    return gi_check_launch("gi_int4_linear");
}

// out [M, N] with rows ld_out apart = x [M, K] . W^T for 1 to 16 rows.  glu: W holds a gate's outputs and as many of an up,
// each a multiple of 16, and out [M, N / 2] is their gated unit.  ranks, parts: blocks that share K, and parts that
// a block's warps take of its slice (0: chosen here).
extern "C" int gi_int4_linear(const void* x, const void* tiles, void* out, int out_dtype, long long ld_out, int M, int N, int K,
                              int glu, int kind, float alpha, float gate_max, float up_limit, float up_shift, int ranks, int parts,
                              int* error_flag, void* stream) {
    GI_REQUIRE(M >= 1 && M <= 16, "gi_int4_linear: %d rows; this kernel takes 1 to 16", M);
    GI_REQUIRE(N > 0 && K > 0 && N < (1 << 30) && K < (1 << 30), "gi_int4_linear: a weight of %d x %d", N, K);
    GI_REQUIRE((uintptr_t)tiles % 16 == 0, "gi_int4_linear: the tiles must start on 16 bytes");
    GI_REQUIRE(out_dtype == GI_DTYPE_BF16 || out_dtype == GI_DTYPE_F32, "gi_int4_linear: output dtype %d", out_dtype);
    GI_REQUIRE(!glu || (N % 32 == 0 && kind >= 0 && kind <= 2 && up_limit >= 0.f),
               "gi_int4_linear: a gated unit %d of %d outputs (halves must be multiples of 16)", kind, N);
    GI_REQUIRE(ld_out >= (glu ? N / 2 : N), "gi_int4_linear: output rows %lld apart hold no %d columns", ld_out, glu ? N / 2 : N);
    GI_REQUIRE(ranks >= 0 && ranks <= 8, "gi_int4_linear: a cluster of %d blocks; 1 to 8 are possible", ranks);
    GI_REQUIRE(parts >= 0 && parts <= 16, "gi_int4_linear: %d parts; 1, 2, 4, 8 or 16 are possible", parts);
    GI_REQUIRE(error_flag != nullptr, "gi_int4_linear: an error flag on the device is required");
    const GluShape unit = {kind, alpha, gate_max, up_limit, up_shift};
    const bf16* xp = (const bf16*)x;
    const unsigned char* tp = (const unsigned char*)tiles;
    const int f32 = out_dtype == GI_DTYPE_F32;
    cudaStream_t s = (cudaStream_t)stream;
    Int4Held held;
    if (int rc = clusters_held(&held)) return rc;
    const Int4Cut cut = cut_of(M, N, K, glu, ranks, parts, held);
    GI_REQUIRE(cut.ranks > 0, "gi_int4_linear: %d x %d is too large for %d rows (in %d blocks, %d parts)", N, K, M, ranks, parts);
#define GI_I4(NT, GLU) launch_int4_linear<NT, GLU>(xp, tp, out, f32, M, N, K, cut, held, unit, ld_out, error_flag, s)
    if (M <= 8) return glu ? GI_I4(1, true) : GI_I4(1, false);
    return glu ? GI_I4(2, true) : GI_I4(2, false);
#undef GI_I4
}

// Whether gi_int4_linear takes a product of these sizes on the current device: 1 or 0, or -1 if the device could not be asked.
extern "C" int gi_int4_linear_takes(int M, int N, int K, int glu) {
    Int4Held held;
    if (clusters_held(&held)) return -1;
    return M >= 1 && M <= 16 && N > 0 && K > 0 && N < (1 << 30) && K < (1 << 30) && (!glu || N % 32 == 0) && cut_of(M, N, K, glu, 0, 0, held).ranks > 0;
}
// What gi_int4_linear counts on: clusters of 1 to 8 blocks that the current device holds at once.
extern "C" int gi_int4_linear_held(int ranks) {
    Int4Held held;
    return ranks < 1 || ranks > 8 || clusters_held(&held) ? -1 : held.clusters[ranks];
}
