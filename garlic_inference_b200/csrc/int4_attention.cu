// Attention over a cache in 4 bits (layout: int4_rows.cu) for single tokens and for a few tokens of a sequence:
//
//   o = softmax_j(q . k_j * scale) v_j,   k_j, v_j = step * code + low per 64 numbers of a head
//
// over the keys j <= position of the query's own sequence (and j > position - window), query head h reading key/value head
// h / (n_q / n_kv).  Bound by reading the cache once, 0.56 bytes a number: on a B200 that leaves each SM 200 cycles for
// 32 keys of 128, so unpacking has to be short.  Codes therefore go to the tensor cores as they are (int4.cuh), with keys
// and output numbers as the 16-wide side of mma.sync m16n8k16 and the queries as its 8 columns:
//
//   scores^T [16 keys x 8] = codes of K [16 x 64] . q^T,  then  step_j * that + low_j * sum(q),  per group of 64
//   out^T [16 numbers x 8] += codes of V^T [16 x 16 keys] . (p_j * step_j)^T,   and  sum_j p_j * low_j beside it
//
// q goes in exactly (a scaled f16), p_j * step_j rounded to the 11 significant bits of an f16, scaled by a power of two that
// follows the largest step so far; a probability of 2^-20 of the largest still has all of them, 2^-10 with a step 2^10 below the
// largest.  From the first 16 keys on whose steps lie further apart, every column has a scale of its own, so that no key, seen or not, takes
// bits from others.  Everything else is float32, but for what int4.cuh says of the sums in an instruction.
// The transposition that the second product needs of V (its 16-wide side runs along a row of the cache) is ldmatrix's, on half words of
// four numbers; that of the probabilities is movmatrix.
//
//  * A block is one run of tokens, one key/value head, one block of 8 NT columns (token, query head of the group) and one
//    slice of the keys.  Its 4 warps take 32 keys each, in turn, through a queue of their own (cp.async, three chunks deep), 16 at a time, and
//    are merged in shared memory at the end; up to 8 slices are a cluster that joins itself, others are joined by a second kernel.
//  * The reference of the softmax is moved only when a score lies 2^8 above it, and the scale of the steps only when one leaves its range:
//    one vote a step instead of reductions and products over all sums.  What is rare (steps far apart, values that are not finite) has a
//    branch of its own, which shortened the common path by 9 instructions.
//  * What runs once a block is kept small and rolled up: such instructions come from the instruction cache's next level at about 20 cycles each.
//
// Measured, 8 key/value heads of 128, nothing in L2: one sequence of 131,000 keys 45.5 us in 74 slices (3.3 TB/s; 335 instructions for 16 keys of a
// head at 2.2 a cycle and SM, 80 of them unpacking, 16 warps an SM), 8 of 2,048 14.8 us, 64 of 500 18.3 us, 48 of 1 to 8,000 61 us.
#include "int4.cuh"

#include <type_traits>

#define I4A_WARPS 4
#define I4A_THREADS (I4A_WARPS * 32)
#define I4A_KEYS 32                // keys of a chunk
#define I4A_STAGES 3
#define I4A_LOG2E 1.4426950408889634f

struct Int4Cache {
    const unsigned char *k, *v;    // codes
    const unsigned char *km, *vm;  // steps and low values
};

__device__ __forceinline__ void i4a_cp(void* smem, const void* gmem, bool valid, std::integral_constant<int, 16>) {
    const int bytes = valid ? 16 : 0;                                    // 0 source bytes: zero-filled
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void i4a_cp(void* smem, const void* gmem, bool valid, std::integral_constant<int, 8>) {
    const int bytes = valid ? 8 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void i4a_cp(void* smem, const void* gmem, bool valid, std::integral_constant<int, 4>) {
    const int bytes = valid ? 4 : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"((uint32_t)__cvta_generic_to_shared(smem)), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint32_t i4a_transpose(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float i4a_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

template <int D> struct Int4Chunk {
    static constexpr int G = D / I4_GROUP_KV;                            // groups of a row
    static constexpr int ROW = D / 2, CODES = I4A_KEYS * ROW, META = I4A_KEYS * G * 4;
    static constexpr int BYTES = 2 * (CODES + META);
    static constexpr int PIECES = ROW / 16;                              // 16-byte pieces of a row
};
// Where piece c of row r lies in a chunk: eight rows' pieces of one number cover all banks
template <int D> __device__ __forceinline__ int i4a_piece(int r, int c) {
    return r * Int4Chunk<D>::ROW + (D == 128 ? c ^ ((r >> 1) & 3) : c ^ ((r >> 2) & 1)) * 16;
}
// Four 8 x 8 matrices of half words, as they are or transposed; a lane gives the address of a row of 16 bytes
__device__ __forceinline__ void i4a_matrix(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void i4a_matrix_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
#define I4A_SLACK 8.f              // a score may lie this far (in powers of two) above the reference
#define I4A_STEP_TOP 6             // the largest step so far is scaled to [2^6, 2^7): times 2^8 it stays below f16's largest number
#define I4A_STEP_RANGE 10          // steps down to 2^-10 of it share its scale
#define I4A_STEP_MOST 30           // the scale follows steps up to 2^31, so that sums of larger ones and of those near 1 are both float32 numbers

// Where the warps of a block meet: [warp][column][D + 4] sums, [warp][column] maximum and weight, then the block's own maximum and weight of a
// column; its sums lie in the first warp's place.
template <int D, int NT> struct Int4Meet {
    static constexpr int COLS = 8 * NT, LD = D + 4, ML = I4A_WARPS * COLS * LD, OWN = ML + I4A_WARPS * COLS * 2, FLOATS = OWN + COLS * 2;
};
__device__ __forceinline__ uint32_t i4a_remote(const void* p, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return r;
}
__device__ __forceinline__ void i4a_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Slices whose blocks are a cluster: each adds up its share of the columns' numbers, in the order of the slices, out of the others' shared memory
template <int D, int NT, typename Row>
__device__ __forceinline__ void i4a_join(bf16* __restrict__ out, int n_cols, int split, int n_splits, Row result_row) {
    typedef Int4Meet<D, NT> M;
    extern __shared__ __align__(16) unsigned char i4a_smem[];
    const float* const meet = reinterpret_cast<const float*>(i4a_smem);
    __syncwarp();
    i4a_cluster_sync();                                                        // the blocks' sums are there
    const int items = n_cols * (D / 4);
#pragma unroll 1
    for (int i = items * split / n_splits + threadIdx.x; i < items * (split + 1) / n_splits; i += I4A_THREADS) {
        const int cc = i / (D / 4), d4 = (i % (D / 4)) * 4;
        float m[8], l[8], most = -INFINITY;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            m[r] = -INFINITY;
            if (r < n_splits) asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m[r]), "=f"(l[r]) : "r"(i4a_remote(meet + M::OWN + cc * 2, r)) : "memory");
            most = fmaxf(most, m[r]);
        }
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            if (m[r] == -INFINITY) continue;                                   // no such slice, or it saw no key
            float4 v;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(i4a_remote(meet + cc * M::LD + d4, r)) : "memory");
            const float f = i4a_exp2(m[r] - most);
            acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
            L = fmaf(f, l[r], L);
        }
        const float inv = L == 0.f ? 0.f : 1.f / L;
        store4_act(out + result_row(cc) * D + d4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    }
    __syncwarp();
    i4a_cluster_sync();                                                        // the others have read this block's
}

// Columns col0 .. of a run (rows row0 .. row0 + rows - 1 of q, at positions pos0 ..) over slice `split` of its keys, by a whole block.
template <int D, int NT>
__device__ __forceinline__ void i4a_columns(const bf16* __restrict__ q, const Int4Cache& cache, const int* __restrict__ table, bf16* __restrict__ out,
                                            float* __restrict__ part_o, float* __restrict__ part_ml, int slot, int row0, int rows, int pos0, int col0,
                                            int kvh, int split, int n_q, int n_kv, int n_slots, int max_pages, int page_size, int n_pages, int window,
                                            float scale_log2, int n_splits, int group, int whole, int* __restrict__ status) {
    typedef Int4Chunk<D> C;
    constexpr int G = C::G, COLS = 8 * NT;
    extern __shared__ __align__(16) unsigned char i4a_smem[];
    // the queries as operand fragments [column block][group, word][lane], what brings a column's scores back, its sums per group: in the
    // last stage of the first warp's ring, which is filled only once all have read them.  Beyond the rings they would cost the fourth
    // block of an SM (4 x 55,296 bytes of 233,472, a kilobyte a block taken)
    static_assert(NT * 2 * G * 512 + (1 + G) * COLS * 4 <= C::BYTES, "the fragments' place");
    uint4* const s_frag = reinterpret_cast<uint4*>(i4a_smem + (I4A_STAGES - 1) * C::BYTES);
    float* const s_back = reinterpret_cast<float*>(s_frag + NT * 2 * G * 32);
    float* const s_sum = s_back + COLS;                                        // [G][COLS]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n_cols = min(rows * group - col0, COLS);                         // columns: (token, head of the group)
    auto token_of = [&](int c) { return rows == 1 ? 0 : (col0 + c) / group; };
    auto result_row = [&](int c) {                                             // row of the result that column c is: (token, query head)
        const int tok = token_of(c);
        return (size_t)(row0 + tok) * n_q + kvh * group + (col0 + c - tok * group);
    };
    const int first = pos0 + token_of(0), hi = pos0 + token_of(n_cols - 1);    // positions of the block's tokens
    bool ok = slot >= 0;
    if (ok && (pos0 < 0 || slot >= n_slots || hi / page_size >= max_pages)) {
        if (threadIdx.x == 0) atomicExch(status, 4);
        ok = false;
    }
    const int lo = window > 0 ? max(0, first - window + 1) : 0;
    const int chunk0 = lo / I4A_KEYS, n_chunks = hi / I4A_KEYS - chunk0 + 1;
    const int per = max((n_chunks + n_splits - 1) / n_splits, 2 * I4A_WARPS);   // fewer chunks do not pay for a block's start
    const int c_begin = chunk0 + split * per, c_end = chunk0 + min(n_chunks, (split + 1) * per);
    if (!ok || c_begin >= c_end) {
        if (n_splits > 1 && !part_ml) {
            if (threadIdx.x < n_cols) *reinterpret_cast<float2*>(reinterpret_cast<float*>(i4a_smem) + Int4Meet<D, NT>::OWN + threadIdx.x * 2) = make_float2(-INFINITY, 0.f);
            i4a_join<D, NT>(out, n_cols, split, n_splits, result_row);
        } else if (n_splits > 1) {
            for (int i = threadIdx.x; i < n_cols; i += I4A_THREADS) {
                float* ml = part_ml + (result_row(i) * n_splits + split) * 2;
                ml[0] = -INFINITY, ml[1] = 0.f;
            }
        } else {
            for (int i = threadIdx.x; i < n_cols * D; i += I4A_THREADS) out[result_row(i / D) * D + i % D] = __float2bfloat16_rn(0.f);
        }
        return;
    }
    const int* bt = table + (size_t)slot * max_pages;

    // ---- the warp's queue: chunk c_begin + warp + 4 i
    unsigned char* ring = i4a_smem + warp * I4A_STAGES * C::BYTES;
    constexpr int ROWS = 32 / C::PIECES;                                       // rows that a copy of the warp takes
    const int my_r = lane / C::PIECES, my_dst = i4a_piece<D>(my_r, lane % C::PIECES);      // of the first copy; others lie ROWS rows on
    int next = c_begin + warp, slot_in = 0;
    int page_next = whole >= 0 && next < c_end ? __ldg(bt + (next * I4A_KEYS >> whole)) : -1;      // asked for one chunk ahead
    bool unmapped = false;
    auto issue = [&]() {
        if (next < c_end) {
            const int j0 = next * I4A_KEYS, here = hi - j0 + 1;                // rows of the chunk that exist
            unsigned char* dst = ring + slot_in * C::BYTES;
            if (whole >= 0) {                                                  // a chunk lies in one page: its rows are contiguous
                const int page = page_next;
                if (next + I4A_WARPS < c_end) page_next = __ldg(bt + (j0 + I4A_WARPS * I4A_KEYS >> whole));
                const bool mapped = page >= 0 && page < n_pages;
                unmapped |= !mapped;
                const int rows_here = mapped ? here : 0;
                const size_t row = mapped ? ((size_t)page * n_kv + kvh) * page_size + (j0 & (page_size - 1)) : 0;
                const unsigned char *k = cache.k + row * C::ROW + lane * 16, *v = cache.v + row * C::ROW + lane * 16;
                const unsigned char *km = cache.km + (row + lane) * (G * 4), *vm = cache.vm + (row + lane) * (G * 4);
                unsigned char *to = dst + my_dst, *mto = dst + 2 * C::CODES + lane * G * 4;
                if (rows_here >= I4A_KEYS) {
#pragma unroll
                    for (int i = 0; i < C::PIECES; ++i) {
                        i4a_cp(to + i * 512, k + i * 512, true, std::integral_constant<int, 16>());
                        i4a_cp(to + C::CODES + i * 512, v + i * 512, true, std::integral_constant<int, 16>());
                    }
                    i4a_cp(mto, km, true, std::integral_constant<int, G * 4>());
                    i4a_cp(mto + C::META, vm, true, std::integral_constant<int, G * 4>());
                } else {                                                       // rows that do not exist are zeros, and read nowhere
#pragma unroll 1
                    for (int i = 0; i < C::PIECES; ++i) {
                        const bool in = i * ROWS + my_r < rows_here;
                        i4a_cp(to + i * 512, in ? k + i * 512 : cache.k, in, std::integral_constant<int, 16>());
                        i4a_cp(to + C::CODES + i * 512, in ? v + i * 512 : cache.v, in, std::integral_constant<int, 16>());
                    }
                    const bool in = lane < rows_here;
                    i4a_cp(mto, in ? km : cache.km, in, std::integral_constant<int, G * 4>());
                    i4a_cp(mto + C::META, in ? vm : cache.vm, in, std::integral_constant<int, G * 4>());
                }
            } else {
                const int lp = (j0 + lane) / page_size;                        // this lane's row of the chunk
                long long row = -1;
                if (lane < here) {                                             // then lp is within the table
                    const int page = __ldg(bt + lp);
                    if (page >= 0 && page < n_pages) row = ((long long)page * n_kv + kvh) * page_size + (j0 + lane - lp * page_size);
                    else unmapped |= j0 + lane >= lo;                          // pages behind the window may have been given back
                }
#pragma unroll 1
                for (int i = 0; i < C::PIECES; ++i) {
                    const long long at = __shfl_sync(0xffffffffu, row, i * ROWS + my_r);
                    const size_t off = at < 0 ? 0 : (size_t)at * C::ROW + lane % C::PIECES * 16;
                    i4a_cp(dst + my_dst + i * 512, cache.k + off, at >= 0, std::integral_constant<int, 16>());
                    i4a_cp(dst + C::CODES + my_dst + i * 512, cache.v + off, at >= 0, std::integral_constant<int, 16>());
                }
                const size_t m = row < 0 ? 0 : (size_t)row * G * 4;
                i4a_cp(dst + 2 * C::CODES + lane * G * 4, cache.km + m, row >= 0, std::integral_constant<int, G * 4>());
                i4a_cp(dst + 2 * C::CODES + C::META + lane * G * 4, cache.vm + m, row >= 0, std::integral_constant<int, G * 4>());
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");                 // an empty group when nothing is left
        next += I4A_WARPS;
        slot_in = slot_in + 1 == I4A_STAGES ? 0 : slot_in + 1;
    };
#pragma unroll 1
    for (int i = 0; i < I4A_STAGES - 1; ++i) issue();

    // ---- the queries as operand fragments: a thread has 8 numbers of a column
    constexpr int CHUNKS = D / 8;
#pragma unroll 1
    for (int i = threadIdx.x; i < COLS * CHUNKS; i += I4A_THREADS) {           // whole warps, and the threads of a column, go on or stop together
        const int c = i / CHUNKS, k = i % CHUNKS;
        const uint4 raw = c < n_cols ? __ldg(reinterpret_cast<const uint4*>(q + result_row(c) * D + k * 8)) : make_uint4(0, 0, 0, 0);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) most = max(most, max((w[e] & 0x7FFFu) << 16, w[e] & 0x7FFF0000u));
#pragma unroll
        for (int o = CHUNKS / 2; o > 0; o >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        int ex;
        const float f = i4_factor(__uint_as_float(min(most, 0x7F7F0000u)), ex);
        float a[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            a[2 * e] = i4_bf16_low(w[e]) * f;
            a[2 * e + 1] = i4_bf16_high(w[e]) * f;
            sum += a[2 * e] + a[2 * e + 1];
        }
        // numbers 32 h + 8 t .. of group k / 8: word h of lane (column, t)
        s_frag[((c >> 3) * 2 * G + (k >> 2)) * 32 + (c & 7) * 4 + (k & 3)] = i4_operand(a);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if ((k & 7) == 0) s_sum[(k >> 3) * COLS + c] = sum * I4_UNIT;
        // codes are multiples of 2^-24 to the tensor cores; a query with a number that is not finite has no scores
        if (k == 0) s_back[c] = most > 0x7F7FFFFFu ? __uint_as_float(0x7FC00000u) : i4_pow2(ex) * 1024.f * scale_log2;
    }
    __syncthreads();
    uint4 qf[NT][2 * G];
    float qsum[NT][G][2], cscale[NT][2], m[NT][2], use[NT][2], limit[NT][2], l[NT][2], off_sum[NT][G][2], o[G * 4][NT][4];      // of columns 2t, 2t + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 2 * G; ++i) qf[nt][i] = s_frag[(nt * 2 * G + i) * 32 + lane];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            cscale[nt][e] = s_back[nt * 8 + 2 * t + e];
            m[nt][e] = limit[nt][e] = -INFINITY;
            use[nt][e] = l[nt][e] = 0.f;                                       // the reference; 0 while no key was seen
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                qsum[nt][gr][e] = s_sum[gr * COLS + nt * 8 + 2 * t + e];
                off_sum[nt][gr][e] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < G * 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
    }
    // What scales the largest step so far (of those below 2^31) to [2^6, 2^7): 2^(6 - e), e its exponent; 0 while there is none.  A step
    // shares this scale if it lies in [2^(e - 10), 2^(e + 1)).  Negative once some step did not: sums of columns that see only small ones
    // then want the scale of their own that the branch for such keys gives them, to the end of the slice.
    float vscale[G];
    auto step_exp = [&](int gr) { return vscale[gr] == 0.f ? -113 : I4A_STEP_TOP + 127 - (int)(__float_as_uint(fabsf(vscale[gr])) >> 23); };
#pragma unroll
    for (int gr = 0; gr < G; ++gr) vscale[gr] = 0.f;

    uint32_t matrix[G];                                                        // this lane's row of the four matrices of a group, K's and V's
#pragma unroll
    for (int gr = 0; gr < G; ++gr) matrix[gr] = (uint32_t)i4a_piece<D>(((lane >> 3) & 1) * 8 + (lane & 7), gr * 2 + (lane >> 4));
    __syncthreads();                                                           // the fragments are read: their place may be filled
    int slot_out = 0;
    for (int c = c_begin + warp; c < c_end; c += I4A_WARPS) {
        issue();
        asm volatile("cp.async.wait_group %0;\n" ::"n"(I4A_STAGES - 1) : "memory");
        __syncwarp();
        const unsigned char* const chunk = ring + slot_out * C::BYTES;
        slot_out = slot_out + 1 == I4A_STAGES ? 0 : slot_out + 1;
#pragma unroll 1
        for (int half16 = 0; half16 < 2; ++half16) {
            const int j0 = c * I4A_KEYS + half16 * 16;
            if (j0 > hi) break;
            const uint32_t sK = (uint32_t)__cvta_generic_to_shared(chunk) + half16 * 16 * C::ROW;
            const unsigned char* sKM = chunk + 2 * C::CODES + (half16 * 16 + g) * G * 4;
            const unsigned char* sVM = sKM + C::META;
            // ---- scores of 16 keys, in powers of two
            float s[NT][4], z[G][NT][4];
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                uint32_t w[4];                                                 // rows g, g + 8 of numbers 8 t .., then of 32 + 8 t ..
                i4a_matrix(w, sK + matrix[gr]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a0 = w[2 * h], a1 = w[2 * h + 1], c0 = a0 >> 8, c1 = a1 >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint4 b = qf[nt][gr * 2 + h];
                        if (h == 0) i4_mma_first(z[gr][nt], a0 & I4_NEAR, a1 & I4_NEAR, a0 & I4_FAR, a1 & I4_FAR, b.x, b.y);
                        else i4_mma(z[gr][nt], a0 & I4_NEAR, a1 & I4_NEAR, a0 & I4_FAR, a1 & I4_FAR, b.x, b.y);
                        i4_mma(z[gr][nt], c0 & I4_NEAR, c1 & I4_NEAR, c0 & I4_FAR, c1 & I4_FAR, b.z, b.w);
                    }
                }
            }
            float vs[G][2], vo[G][2];                                          // steps and low values of this lane's two values per group
            bool moved = false;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t km[G], vm[G];
                const int at = half * 8 * (G * 4);
                if (G == 2) {
                    const uint2 a = *reinterpret_cast<const uint2*>(sKM + at), b = *reinterpret_cast<const uint2*>(sVM + at);
                    km[0] = a.x, km[G - 1] = a.y, vm[0] = b.x, vm[G - 1] = b.y;
                } else {
                    km[0] = *reinterpret_cast<const uint32_t*>(sKM + at), vm[0] = *reinterpret_cast<const uint32_t*>(sVM + at);
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = 0.f;
#pragma unroll
                        for (int gr = 0; gr < G; ++gr)
                            v = fmaf(i4_bf16_low(km[gr]), z[gr][nt][half * 2 + e], fmaf(i4_bf16_high(km[gr]), qsum[nt][gr][e], v));
                        s[nt][half * 2 + e] = fmaf(v, cscale[nt][e], -use[nt][e]);      // above the reference
                    }
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    vs[gr][half] = i4_bf16_low(vm[gr]);
                    vo[gr][half] = i4_bf16_high(vm[gr]);
                }
            }
            // ---- keys that a column does not see, and values there that are not finite
            const bool edge = j0 + 15 > first || (window > 0 && j0 <= hi - window);
            bool odd = false;
            if (edge) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + g + (e >> 1) * 8, cc = nt * 8 + 2 * t + (e & 1), p = cc < n_cols ? pos0 + token_of(cc) : -1;
                        if (j > p || (window > 0 && j <= p - window)) s[nt][e] = -INFINITY;
                    }
#pragma unroll
                for (int half = 0; half < 2; ++half) {                         // what no column sees has no value
                    const int j = j0 + g + half * 8;
                    if (j > hi || (window > 0 && j <= first - window))
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) vs[gr][half] = vo[gr][half] = 0.f;
                }
#pragma unroll
                for (int gr = 0; gr < G; ++gr) odd |= !(vs[gr][0] <= 3.4e38f) || !(vs[gr][1] <= 3.4e38f) || !(fabsf(vo[gr][0]) <= 3.4e38f) || !(fabsf(vo[gr][1]) <= 3.4e38f);
                odd = __any_sync(0xffffffffu, odd);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) moved |= s[nt][e] > limit[nt][e & 1];
#pragma unroll
            for (int gr = 0; gr < G; ++gr)
                moved |= !(fabsf(vs[gr][0] * vscale[gr] - 64.f) <= 63.9375f) || !(fabsf(vs[gr][1] * vscale[gr] - 64.f) <= 63.9375f);      // [2^-4, 2^7)
            // ---- a new reference for the columns' sums, or a new scale for the steps
            bool apart = false;                                                // steps of more than one range
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    const uint32_t b0 = __float_as_uint(vs[gr][0]), b1 = __float_as_uint(vs[gr][1]);      // never negative; NaN and infinities aside
                    const uint32_t most = __reduce_max_sync(0xffffffffu, max(b0 < 0x7F800000u ? b0 : 0u, b1 < 0x7F800000u ? b1 : 0u));
                    const int before = step_exp(gr), e = max(max(min((int)(most >> 23) - 127, I4A_STEP_MOST), -112), before);
                    const float grow = before < -112 ? 0.f : i4a_exp2((float)(before - e));      // nothing summed up yet: 0 times 0
                    auto outside = [&](uint32_t b) { return b != 0 && b < 0x7F800000u && (b >> 23) - (uint32_t)(e - I4A_STEP_RANGE + 127) > I4A_STEP_RANGE; };
                    const bool far = vscale[gr] < 0.f || (before >= -112 && e - before > I4A_STEP_RANGE) || outside(b0) || outside(b1);
                    const bool any = __any_sync(0xffffffffu, far);
                    vscale[gr] = any ? -i4_pow2(I4A_STEP_TOP - e) : i4_pow2(I4A_STEP_TOP - e);
                    apart |= any;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[gr * 4 + i][nt][x] *= grow;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(s[nt][e], s[nt][e + 2]);
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                        const float m_new = fmaxf(m[nt][e], mx + use[nt][e]), corr = m_new == -INFINITY ? 1.f : i4a_exp2(m[nt][e] - m_new);
                        const float to = m_new == -INFINITY ? 0.f : m_new;
                        s[nt][e] += use[nt][e] - to, s[nt][e + 2] += use[nt][e] - to;
                        m[nt][e] = m_new, use[nt][e] = to;
                        limit[nt][e] = m_new == -INFINITY ? -INFINITY : I4A_SLACK;
                        l[nt][e] *= corr;
#pragma unroll
                        for (int gr = 0; gr < G; ++gr) off_sum[nt][gr][e] *= corr;
#pragma unroll
                        for (int i = 0; i < G * 4; ++i) o[i][nt][e] *= corr, o[i][nt][e + 2] *= corr;
                    }
            }
            auto probabilities = [&]() {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s[nt][e] = i4a_exp2(s[nt][e]);
                        s[nt][e + 2] = i4a_exp2(s[nt][e + 2]);
                        l[nt][e] += s[nt][e] + s[nt][e + 2];
                    }
            };
            auto offsets = [&](int gr, int half, int nt) {
                const float p0 = s[nt][half * 2], p1 = s[nt][half * 2 + 1];
                off_sum[nt][gr][0] += p0 == 0.f ? 0.f : p0 * vo[gr][half];
                off_sum[nt][gr][1] += p1 == 0.f ? 0.f : p1 * vo[gr][half];
            };
            // ---- steps far apart, or values that are not finite: what a column does not see stays out, and every column has a scale of
            // its own, so that its largest probability times step lies in [2^14, 2^15)
            if (apart || odd) {
                probabilities();
#pragma unroll
                for (int gr = 0; gr < G; ++gr)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) offsets(gr, 0, nt), offsets(gr, 1, nt);
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
                    const uint32_t b0 = __float_as_uint(vs[gr][0]), b1 = __float_as_uint(vs[gr][1]);
                    const uint32_t most = __reduce_max_sync(0xffffffffu, max(b0 < 0x7F800000u ? b0 : 0u, b1 < 0x7F800000u ? b1 : 0u));
                    const int e = min(max((int)(most >> 23) - 127, -112), 126);
                    const float down = i4_pow2(-e), up = i4a_exp2((float)(I4A_STEP_TOP + e - step_exp(gr)));
                    uint32_t w[4];
                    i4a_matrix_trans(w, sK + C::CODES + matrix[gr]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float x[2][2], back[2];                                // [half][column]
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float p0 = s[nt][c], p1 = s[nt][2 + c];
                            x[0][c] = p0 == 0.f ? 0.f : p0 * (vs[gr][0] * down), x[1][c] = p1 == 0.f ? 0.f : p1 * (vs[gr][1] * down);
                            float top = fmaxf(x[0][c], x[1][c]);               // NaN aside
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                            int ex;
                            const float f = i4_factor(top, ex);
                            x[0][c] *= f, x[1][c] *= f;
                            back[c] = i4_pow2(ex - 14) * up;
                        }
                        const uint32_t k0 = i4a_transpose(i4_f16x2(x[0][0], x[0][1])), k8 = i4a_transpose(i4_f16x2(x[1][0], x[1][1]));
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t a = w[i & 2] >> (i & 1) * 8, d = w[(i & 2) + 1] >> (i & 1) * 8;
                            float z[4];
                            i4_mma_first(z, a & I4_NEAR, a & I4_FAR, d & I4_NEAR, d & I4_FAR, k0, k8);
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[gr * 4 + i][nt][r] = fmaf(z[r], back[r & 1], o[gr * 4 + i][nt][r]);
                        }
                    }
                }
                continue;
            }
            probabilities();
            // ---- out^T += codes of V^T . (p step)^T
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                uint32_t b[NT][2];                                             // second operand: keys of rows 0-7 and 8-15
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float step = vs[gr][half] * vscale[gr];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float p0 = s[nt][half * 2], p1 = s[nt][half * 2 + 1];
                        off_sum[nt][gr][0] = fmaf(p0, vo[gr][half], off_sum[nt][gr][0]);
                        off_sum[nt][gr][1] = fmaf(p1, vo[gr][half], off_sum[nt][gr][1]);
                        b[nt][half] = i4a_transpose(i4_f16x2(p0 * step, p1 * step));
                    }
                }
                // half words of numbers 4 g .. of keys 2 t, 2 t + 1; of keys 8 on; of numbers 32 + 4 g ..
                uint32_t w[4];
                i4a_matrix_trans(w, sK + C::CODES + matrix[gr]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a = w[2 * h], d = w[2 * h + 1], a8 = a >> 8, d8 = d >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        i4_mma(o[gr * 4 + 2 * h][nt], a & I4_NEAR, a & I4_FAR, d & I4_NEAR, d & I4_FAR, b[nt][0], b[nt][1]);
                        i4_mma(o[gr * 4 + 2 * h + 1][nt], a8 & I4_NEAR, a8 & I4_FAR, d8 & I4_NEAR, d8 & I4_FAR, b[nt][0], b[nt][1]);
                    }
                }
            }
        }
        __syncwarp();                                                          // every lane is done with the slot that is filled next
    }
    if (unmapped) atomicExch(status, 5);

    // ---- the warps meet
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();
    typedef Int4Meet<D, NT> M;
    constexpr int LD = M::LD;
    float* so = reinterpret_cast<float*>(i4a_smem);
    float* sml = so + M::ML;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int cc = nt * 8 + 2 * t + e;
            float sum = l[nt][e];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
                float f = off_sum[nt][gr][e];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) f += __shfl_xor_sync(0xffffffffu, f, x);
                // 2^(e - 6) for the steps' scale, 2^24 for the codes', in two factors of which neither overflows
                const float back = vscale[gr] == 0.f ? 0.f : i4_pow2(step_exp(gr));
                float* dst = so + (warp * COLS + cc) * LD + gr * 64 + 4 * g;
#pragma unroll
                for (int i = 0; i < 4; ++i) {                                  // numbers four bits up count 16 times
                    dst[(i >> 1) * 32 + (i & 1) * 2] = fmaf(o[gr * 4 + i][nt][e] * 262144.f, back, f);
                    dst[(i >> 1) * 32 + (i & 1) * 2 + 1] = fmaf(o[gr * 4 + i][nt][e + 2] * 16384.f, back, f);
                }
            }
            if (g == 0) {
                // a sum that is NaN (a key, a query that is not finite) keeps its place whatever the reference is
                sml[(warp * COLS + cc) * 2] = sum == sum ? m[nt][e] : 0.f;
                sml[(warp * COLS + cc) * 2 + 1] = sum;
            }
        }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < n_cols * (D / 4); i += I4A_THREADS) {
        const int cc = i / (D / 4), d4 = (i % (D / 4)) * 4;
        float most = -INFINITY;
#pragma unroll
        for (int w = 0; w < I4A_WARPS; ++w) most = fmaxf(most, sml[(w * COLS + cc) * 2]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll 1
        for (int w = 0; w < I4A_WARPS; ++w) {
            const float mw = sml[(w * COLS + cc) * 2];
            if (mw == -INFINITY) continue;                                     // saw no key
            const float f = i4a_exp2(mw - most);
            const float4 v = *reinterpret_cast<const float4*>(so + (w * COLS + cc) * LD + d4);
            acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
            L = fmaf(f, sml[(w * COLS + cc) * 2 + 1], L);
        }
        const size_t row = result_row(cc);
        if (n_splits == 1) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            store4_act(out + row * D + d4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        } else if (!part_ml) {
            *reinterpret_cast<float4*>(so + cc * LD + d4) = acc;               // the first warp's, read by this thread alone
            if (d4 == 0) *reinterpret_cast<float2*>(so + M::OWN + cc * 2) = make_float2(most, L);
        } else {
            *reinterpret_cast<float4*>(part_o + (row * n_splits + split) * D + d4) = acc;
            if (d4 == 0) *reinterpret_cast<float2*>(part_ml + (row * n_splits + split) * 2) = make_float2(most, L);
        }
    }
    if (n_splits > 1 && !part_ml) i4a_join<D, NT>(out, n_cols, split, n_splits, result_row);
}

// The run of a block: slot, first row, rows, position of the first row; without runs, run i is the single token i.  False: there is none.
__device__ __forceinline__ bool i4a_run(const int4* __restrict__ runs, const int* __restrict__ tok_pos, const int* __restrict__ tok_slot, int run,
                                        int n_rows, int4& r, int* status) {
    if (!runs) {
        r = make_int4(tok_slot[run], run, 1, tok_pos[run]);
        return true;
    }
    r = runs[run];
    if (r.z <= 0) return false;
    if (r.y >= 0 && r.z <= n_rows && r.y <= n_rows - r.z && r.w <= 2147483647 - r.z) return true;
    if (threadIdx.x == 0 && status) atomicExch(status, 4);
    return false;
}

template <int D, int NT>
__global__ void __launch_bounds__(I4A_THREADS, NT == 1 ? 4 : 3)
int4_attention_kernel(const bf16* __restrict__ q, Int4Cache cache, const int* __restrict__ table, const int4* __restrict__ runs,
                      const int* __restrict__ tok_pos, const int* __restrict__ tok_slot, bf16* __restrict__ out,
                      float* __restrict__ part_o, float* __restrict__ part_ml, int n_rows, int n_q, int n_kv, int n_slots, int max_pages,
                      int page_size, int n_pages, int window, float scale_log2, int n_splits, int group, int whole, int* __restrict__ status) {
    gi_pdl_start();
    int4 r;
    if (!i4a_run(runs, tok_pos, tok_slot, blockIdx.z, n_rows, r, status)) return;
    const int split = blockIdx.x % n_splits, step = gridDim.x / n_splits * (8 * NT);
#pragma unroll 1
    for (int col0 = blockIdx.x / n_splits * (8 * NT); col0 < r.z * group; col0 += step) {
        if (col0 >= step) __syncthreads();                                     // the last columns' sums are read
        i4a_columns<D, NT>(q, cache, table, out, part_o, part_ml, r.x, r.y, r.z, r.w, col0, blockIdx.y, split, n_q, n_kv, n_slots, max_pages,
                           page_size, n_pages, window, scale_log2, n_splits, group, whole, status);
    }
}

// Joins the slices of a row (token, query head): warp w takes slices w, w + 4 ..; the sums of the four warps meet in shared memory.  A block
// goes through its run's rows, gridDim.y apart.
template <int D>
__global__ void __launch_bounds__(128)
int4_attention_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, const int4* __restrict__ runs,
                           bf16* __restrict__ out, int n_rows, int n_q, int n_splits) {
    constexpr int V = D / 32, AHEAD = 4;                                       // numbers of a lane; slices whose loads are in flight
    __shared__ float s_o[4][D], s_l[4];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    gi_pdl_start();
    int4 r = make_int4(0, blockIdx.z, 1, 0);
    if (runs && !i4a_run(runs, nullptr, nullptr, blockIdx.z, n_rows, r, nullptr)) return;
#pragma unroll 1
    for (int tok = blockIdx.y; tok < r.z; tok += gridDim.y) {
        const size_t row = (size_t)(r.y + tok) * n_q + blockIdx.x;
        const float* ml = part_ml + row * n_splits * 2;
        const float* o = part_o + row * n_splits * D + lane * V;
        float M = -INFINITY;
        for (int s = lane; s < n_splits; s += 32) M = fmaxf(M, ml[2 * s]);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
        float acc[V], L = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = 0.f;
#pragma unroll 1
        for (int s0 = warp; s0 < n_splits; s0 += 4 * AHEAD) {
            float m[AHEAD], v[AHEAD][V];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int s = s0 + 4 * j;
                m[j] = s < n_splits ? ml[2 * s] : -INFINITY;
                if (m[j] != -INFINITY) {                                           // an empty slice wrote no output
                    L = fmaf(i4a_exp2(m[j] - M), ml[2 * s + 1], L);
#pragma unroll
                    for (int i = 0; i < V; i += 2) *reinterpret_cast<float2*>(&v[j][i]) = *reinterpret_cast<const float2*>(o + (size_t)s * D + i);
                }
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (m[j] != -INFINITY) {
                    const float f = i4a_exp2(m[j] - M);
#pragma unroll
                    for (int i = 0; i < V; ++i) acc[i] = fmaf(f, v[j][i], acc[i]);
                }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) s_o[warp][lane * V + i] = acc[i];
        if (lane == 0) s_l[warp] = L;
        __syncthreads();
        if (threadIdx.x < D) {
            const float sum = s_l[0] + s_l[1] + s_l[2] + s_l[3], v = s_o[0][threadIdx.x] + s_o[1][threadIdx.x] + s_o[2][threadIdx.x] + s_o[3][threadIdx.x];
            out[row * D + threadIdx.x] = __float2bfloat16_rn(sum == 0.f ? 0.f : v / sum);
        }
        __syncthreads();
    }
}

// runs [n_runs, 4], or none: every token is a sequence of its own.  With n_splits > 1 the
// up to 8 slices without part_o and part_ml are a cluster and join
// themselves; otherwise they lie in part_o [tokens, n_q, n_splits, d] and part_ml [tokens, n_q, n_splits, 2], and a second kernel joins them.
extern "C" int gi_int4_attention(const void* q, const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta,
                                 const int* table, const int* runs, int n_runs, int n_rows, const int* tok_pos, const int* tok_slot,
                                 void* out, float* part_o, float* part_ml, int n_q, int n_kv, int d, int n_slots, int max_pages,
                                 int page_size, int n_pages, int window, float scale, int n_splits, int* status, void* stream) {
    GI_REQUIRE(d == 64 || d == 128, "gi_int4_attention: heads of %d; 64 and 128 are possible", d);
    GI_REQUIRE(n_kv > 0 && n_q > 0 && n_q % n_kv == 0 && n_kv <= 65535, "gi_int4_attention: %d query heads over %d key/value heads", n_q, n_kv);
    GI_REQUIRE(n_runs >= 0 && n_runs <= 65535 && n_rows >= (runs ? 0 : n_runs) && n_rows <= 1 << 24,
               "gi_int4_attention: %d runs of %d rows", n_runs, n_rows);
    GI_REQUIRE(page_size > 0 && max_pages > 0 && n_slots > 0 && window >= 0, "gi_int4_attention: page and table sizes must be positive");
    GI_REQUIRE(n_splits >= 1 && n_splits <= 256 && (part_o != nullptr) == (part_ml != nullptr) && (n_splits <= 8 || part_o), "gi_int4_attention: %d slices", n_splits);
    GI_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_meta % 8 == 0 &&
               (uintptr_t)v_meta % 8 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)part_o % 16 == 0 && (uintptr_t)runs % 16 == 0,
               "gi_int4_attention: operands must start on 16 bytes");
    if (n_runs == 0 || n_rows == 0) return 0;
    const Int4Cache cache = {(const unsigned char*)k_codes, (const unsigned char*)v_codes, (const unsigned char*)k_meta, (const unsigned char*)v_meta};
    int whole = -1;                                                            // pages of 2^whole rows, chunks within a page; -1: any other
    for (int i = 5; i < 31; ++i) if (page_size == 1 << i) whole = i;
    const int group = n_q / n_kv;
    const long long cols = ((long long)n_rows * group + n_runs - 1) / n_runs;   // of a run, on average
    const int nt = cols > 8 ? 2 : 1;
    const long long col_tiles = (cols + 8 * nt - 1) / (8 * nt);
    GI_REQUIRE(col_tiles * n_splits < 2147483647LL, "gi_int4_attention: %d rows in %d runs are too many", n_rows, n_runs);
#define GI_I4A(DD, NN)                                                                                                               \
    {                                                                                                                                \
        size_t smem = (size_t)I4A_WARPS * I4A_STAGES * Int4Chunk<DD>::BYTES;                                                         \
        const size_t meet = (size_t)Int4Meet<DD, NN>::FLOATS * 4;                                                                     \
        if (meet > smem) smem = meet;                                                                                                \
        if (int rc = gi_reserve_smem((const void*)int4_attention_kernel<DD, NN>, smem, "gi_int4_attention")) return rc;              \
        cudaLaunchConfig_t cfg = {};                                                                                                 \
        cfg.gridDim = dim3((unsigned)(col_tiles * n_splits), n_kv, n_runs), cfg.blockDim = dim3(I4A_THREADS);                        \
        cfg.dynamicSmemBytes = smem, cfg.stream = (cudaStream_t)stream;                                                              \
        cudaLaunchAttribute attr[2];                                                                                                 \
        attr[0].id = cudaLaunchAttributeClusterDimension;                                                                            \
        attr[0].val.clusterDim.x = part_o ? 1 : n_splits, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;                   \
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;                                                             \
        attr[1].val.programmaticStreamSerializationAllowed = 1;                                                                      \
        cfg.attrs = attr, cfg.numAttrs = gi_pdl_enabled() ? 2 : 1;                                                                   \
        cudaLaunchKernelEx(&cfg, int4_attention_kernel<DD, NN>, (const bf16*)q, cache, table, (const int4*)runs, tok_pos, tok_slot,  \
                           (bf16*)out, part_o, part_ml, n_rows, n_q, n_kv, n_slots, max_pages, page_size, n_pages, window,           \
                           scale * I4A_LOG2E, n_splits, group, whole, status);                                                       \
    }
    if (d == 64) { if (nt == 1) GI_I4A(64, 1) else GI_I4A(64, 2) }
    else { if (nt == 1) GI_I4A(128, 1) else GI_I4A(128, 2) }
#undef GI_I4A
    if (int rc = gi_check_launch("gi_int4_attention")) return rc;
    if (!part_o || n_splits == 1) return 0;
    const int per = runs ? (n_rows + n_runs - 1) / n_runs : 1;
    const dim3 joins(n_q, per < 65535 ? per : 65535, n_runs);
    if (d == 64) gi_launch(int4_attention_join_kernel<64>, joins, dim3(128), 0, (cudaStream_t)stream, part_o, part_ml, (const int4*)runs, (bf16*)out, n_rows, n_q, n_splits);
    else gi_launch(int4_attention_join_kernel<128>, joins, dim3(128), 0, (cudaStream_t)stream, part_o, part_ml, (const int4*)runs, (bf16*)out, n_rows, n_q, n_splits);
    return gi_check_launch("gi_int4_attention (slices)");
}
