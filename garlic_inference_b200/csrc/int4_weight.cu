// Weights in 4 bits: made from, and turned back into, 16 or 32 bits (the product that reads them: int4_linear.cu).
//
// A weight [N, K] lies in tiles of 16 outputs x 128 inputs, [ceil(N / 16), ceil(K / 128), 1088] bytes, inputs fastest, so that
// what a block streams (one row of tiles, any range of inputs) is contiguous.  In a tile: two pieces of 512 bytes (outputs 0-7
// and 8-15), in each 8 outputs x 4 quarters of 32 inputs x 16 bytes, which is the order in which the 32 lanes of a warp hold the
// product's first operand, 16 bytes each; then (step, low) of the 16 outputs.  What a tile holds beyond N or K is zeros.
//
// Both kernels are bound by the 16- or 32-bit side: 2 or 4 bytes a number against 0.53.  Neither lets its successor start early: products ask
// for their weight before they wait for the kernel in front, and here that kernel writes it.
#include "int4.cuh"

// A warp per (output, group of 128): 4 consecutive inputs a lane.
template <typename T>
__global__ void __launch_bounds__(256)
int4_quantize_weight_kernel(const T* __restrict__ w, long long ld, unsigned char* __restrict__ tiles, int N, int K, long long items,
                            int groups) {
    gi_pdl_start_alone();
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (item >= items) return;
    const int lane = threadIdx.x & 31;
    const int gk = (int)(item % groups);
    const long long n = item / groups;                                   // up to the next multiple of 16 beyond N
    const int k0 = gk * I4_GROUP_W + lane * 4;
    float x[4], mn = INFINITY, mx = -INFINITY;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = n < N && k0 + i < K;
        x[i] = in ? to_f32(w[n * ld + k0 + i]) : 0.f;
        if (in) {
            finite = finite && fabsf(x[i]) <= 3.402823466e38f;
            mn = fminf(mn, x[i]);
            mx = fmaxf(mx, x[i]);
        }
    }
    mx = warp_max(mx);
    mn = -warp_max(-mn);
    finite = __all_sync(0xffffffffu, finite);
    float step = 0.f, low = 0.f;
    if (n < N) i4_step_low(mn, mx, finite, step, low);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n < N && k0 + i < K) bits |= i4_code(x[i], step, low) << (4 * i);
    unsigned char* tile = tiles + ((n >> 4) * groups + gk) * I4_TILE;
    const int r = (int)(n & 15);
    // 2 bytes of the lane's 4 numbers: quarter lane / 8, byte 2 (lane mod 8) in it
    *reinterpret_cast<uint16_t*>(tile + (r >> 3) * 512 + ((r & 7) * 4 + (lane >> 3)) * 16 + (lane & 7) * 2) = (uint16_t)bits;
    if (lane == 0) *reinterpret_cast<uint32_t*>(tile + I4_TILE_CODES + r * 4) = i4_meta(step, low);
}

// Eight inputs of eight outputs (a piece of a tile) a thread, so that a warp writes 512 bytes of a row at once; out [rows, K] holds outputs
// n0 .. n0 + rows - 1.  Bound by writing.
template <typename T>
__global__ void __launch_bounds__(256)
int4_dequantize_weight_kernel(const unsigned char* __restrict__ tiles, T* __restrict__ out, int n0, int rows, int K, int groups, int vec) {
    gi_pdl_start_alone();
    const int word = blockIdx.x * 256 + threadIdx.x, group = word >> 4, k0 = word * 8;      // eight inputs
    if (k0 >= K) return;
    const int piece = blockIdx.y + (n0 >> 3);
    const unsigned char* tile = tiles + ((size_t)(piece >> 1) * groups + group) * I4_TILE;
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(tile + (piece & 1) * 512) + (word & 15);
    const uint32_t* meta = reinterpret_cast<const uint32_t*>(tile + I4_TILE_CODES) + (piece & 1) * 8;
    uint32_t c[8], m[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) c[r] = __ldg(codes + r * 16), m[r] = __ldg(meta + r);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const int row = piece * 8 + r - n0;
        if (row < 0 || row >= rows) continue;
        const float step = i4_bf16_low(m[r]), low = i4_bf16_high(m[r]);
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf(step, (float)((c[r] >> (4 * i)) & 15), low);
        T* dst = out + (size_t)row * K + k0;
        if (vec) {                                                       // K is a multiple of 8
            if (sizeof(T) == 2) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<__nv_bfloat162*>(&w[i]) = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
                store4_act(dst, make_float4(v[0], v[1], v[2], v[3]));
                store4_act(dst + 4, make_float4(v[4], v[5], v[6], v[7]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k0 + i < K) dst[i] = from_f32<T>(v[i]);
        }
    }
}

extern "C" int gi_int4_quantize_weight(const void* w, int dtype, long long ld, void* tiles, int N, int K, void* stream) {
    GI_REQUIRE(N > 0 && K > 0 && ld >= K, "gi_int4_quantize_weight: a weight of %d x %d with rows %lld apart", N, K, ld);
    GI_REQUIRE((uintptr_t)tiles % 16 == 0, "gi_int4_quantize_weight: the tiles must start on 16 bytes");
    const int groups = (K - 1) / I4_GROUP_W + 1;
    const long long items = ((long long)(N - 1) / 16 + 1) * 16 * groups, blocks = (items + 7) / 8;
    GI_REQUIRE(blocks < 2147483647LL, "gi_int4_quantize_weight: %lld groups are too many", items);
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == GI_DTYPE_F32)
        gi_launch(int4_quantize_weight_kernel<float>, dim3((unsigned)blocks), dim3(256), 0, s, (const float*)w, ld, (unsigned char*)tiles, N, K, items, groups);
    else if (dtype == GI_DTYPE_BF16)
        gi_launch(int4_quantize_weight_kernel<bf16>, dim3((unsigned)blocks), dim3(256), 0, s, (const bf16*)w, ld, (unsigned char*)tiles, N, K, items, groups);
    else GI_REQUIRE(false, "gi_int4_quantize_weight: dtype %d", dtype);
    return gi_check_launch("gi_int4_quantize_weight");
}

extern "C" int gi_int4_dequantize_weight(const void* tiles, void* out, int dtype, int n0, int rows, int N, int K, void* stream) {
    GI_REQUIRE(N > 0 && K > 0 && n0 >= 0 && rows > 0 && rows <= N - n0,
               "gi_int4_dequantize_weight: outputs %d .. %d of a weight of %d x %d", n0, n0 + rows - 1, N, K);
    GI_REQUIRE((uintptr_t)tiles % 16 == 0, "gi_int4_dequantize_weight: the tiles must start on 16 bytes");
    const int groups = (K - 1) / I4_GROUP_W + 1;
    const dim3 grid((K + 2047) / 2048, ((n0 + rows + 7) >> 3) - (n0 >> 3));      // eight rows a block
    GI_REQUIRE(grid.y <= 65535, "gi_int4_dequantize_weight: %d outputs at a time are too many", rows);
    const int vec = K % 8 == 0 && (uintptr_t)out % 16 == 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == GI_DTYPE_F32)
        gi_launch(int4_dequantize_weight_kernel<float>, grid, dim3(256), 0, s, (const unsigned char*)tiles, (float*)out, n0, rows, K, groups, vec);
    else if (dtype == GI_DTYPE_BF16)
        gi_launch(int4_dequantize_weight_kernel<bf16>, grid, dim3(256), 0, s, (const unsigned char*)tiles, (bf16*)out, n0, rows, K, groups, vec);
    else GI_REQUIRE(false, "gi_int4_dequantize_weight: dtype %d", dtype);
    return gi_check_launch("gi_int4_dequantize_weight");
}
