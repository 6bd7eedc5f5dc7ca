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
// follows the largest step so far; a probability of 2^-29 of the largest still has all of them.  Everything else is float32.
// The transposition that the second product needs of V (its 16-wide side runs along a row of the cache) is two byte permutes
// for two keys' words; that of the probabilities is movmatrix.
//
//  * A block is one run of tokens, one key/value head, one block of 8 NT columns (token, query head of the group) and one
//    slice of the keys.  Its 4 warps take 32 keys each, in turn, through a queue of their own (cp.async, three chunks deep), and
//    are merged in shared memory at the end; slices are merged by gi_attention_decode_combine, or there is one only.
//  * In a chunk, row r of the 16 x 32 tile is key perm(r), so that the reads of K (8 rows x 4 pieces of 8 bytes) and of V (4 rows x 8 words)
//    touch every bank once.
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
// Where piece c of row r lies in a chunk: with rows of 64 bytes the pieces of every other pair of rows change places, so that four
// rows whose numbers differ mod 4 cover all banks with any one group
template <int D> __device__ __forceinline__ int i4a_piece(int r, int c) {
    return r * Int4Chunk<D>::ROW + (D == 128 ? c ^ (((r >> 1) & 1) << 1) : c) * 16;
}

// runs[i] = {slot, first row, rows, position of the first row}; without runs, run i is the single token i.
template <int D, int NT>
__global__ void __launch_bounds__(I4A_THREADS, NT == 1 ? 4 : 2)
int4_attention_kernel(const bf16* __restrict__ q, Int4Cache cache, const int* __restrict__ table, const int4* __restrict__ runs,
                      const int* __restrict__ tok_pos, const int* __restrict__ tok_slot, bf16* __restrict__ out,
                      float* __restrict__ part_o, float* __restrict__ part_ml, int n_q, int n_kv, int n_slots, int max_pages,
                      int page_size, int n_pages, int window, float scale_log2, int n_splits, int col_tiles, int* __restrict__ status) {
    typedef Int4Chunk<D> C;
    constexpr int G = C::G, COLS = 8 * NT;
    gi_pdl_start();
    extern __shared__ __align__(16) unsigned char i4a_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % n_splits, ct = blockIdx.x / n_splits, kvh = blockIdx.y, run = blockIdx.z;
    const int group = n_q / n_kv;

    int slot, row0, rows, pos0;
    if (runs) {
        const int4 r = runs[run];
        slot = r.x, row0 = r.y, rows = r.z, pos0 = r.w;
    } else {
        slot = tok_slot[run], row0 = run, rows = 1, pos0 = tok_pos[run];
    }
    const int col0 = ct * COLS, n_cols = min(rows * group - col0, COLS);       // columns of this block: (token, head of the group)
    if (n_cols <= 0) return;
    auto result_row = [&](int c) {                                             // row of the result that column c is: (token, query head)
        const int col = col0 + c;
        return (size_t)(row0 + col / group) * n_q + kvh * group + col % group;
    };
    const int first = pos0 + col0 / group, hi = pos0 + (col0 + n_cols - 1) / group;       // positions of the block's tokens
    bool ok = slot >= 0;
    if (ok && (pos0 < 0 || slot >= n_slots || hi / page_size >= max_pages)) {
        if (threadIdx.x == 0) atomicExch(status, 4);
        ok = false;
    }
    const int lo = window > 0 ? max(0, first - window + 1) : 0;
    const int chunk0 = lo / I4A_KEYS, n_chunks = hi / I4A_KEYS - chunk0 + 1;
    const int per = (n_chunks + n_splits - 1) / n_splits;
    const int c_begin = chunk0 + split * per, c_end = chunk0 + min(n_chunks, (split + 1) * per);
    if (!ok || c_begin >= c_end) {
        for (int i = threadIdx.x; i < n_cols; i += I4A_THREADS)
            if (n_splits > 1) {
                float* ml = part_ml + (result_row(i) * n_splits + split) * 2;
                ml[0] = -INFINITY, ml[1] = 0.f;
            }
        if (n_splits == 1)
            for (int i = threadIdx.x; i < n_cols * D; i += I4A_THREADS) out[result_row(i / D) * D + i % D] = __float2bfloat16_rn(0.f);
        return;
    }
    const int* bt = table + (size_t)slot * max_pages;

    // ---- the warp's queue: chunk c_begin + warp + 4 i
    unsigned char* ring = i4a_smem + warp * I4A_STAGES * C::BYTES;
    const bool whole = page_size % I4A_KEYS == 0;                              // a chunk lies in one page
    int next = c_begin + warp, slot_in = 0;
    bool unmapped = false;
    auto issue = [&]() {
        if (next < c_end) {
            const int j = next * I4A_KEYS + lane, lp = j / page_size;          // this lane's row of the chunk
            int page = -1;
            if (j <= hi) {                                                     // then lp is within the table
                page = __ldg(bt + lp);
                if (page < 0 || page >= n_pages) page = -1, unmapped = true;
            }
            const long long row = page < 0 ? -1 : ((long long)page * n_kv + kvh) * page_size + (j - lp * page_size);
            unsigned char* dst = ring + slot_in * C::BYTES;
            const long long base = __shfl_sync(0xffffffffu, row, 0);
            constexpr int ROWS = 32 / C::PIECES;                               // rows that a copy of the warp takes
#pragma unroll
            for (int i = 0; i < C::PIECES; ++i) {
                const int r = i * ROWS + lane / C::PIECES, c = lane % C::PIECES;
                long long at;
                if (whole) at = next * I4A_KEYS + r <= hi && base >= 0 ? base + r : -1;
                else at = __shfl_sync(0xffffffffu, row, r);
                const size_t off = at < 0 ? 0 : (size_t)at * C::ROW + c * 16;
                i4a_cp(dst + i4a_piece<D>(r, c), cache.k + off, at >= 0, std::integral_constant<int, 16>());
                i4a_cp(dst + C::CODES + i4a_piece<D>(r, c), cache.v + off, at >= 0, std::integral_constant<int, 16>());
            }
            const size_t moff = row < 0 ? 0 : (size_t)row * G * 4;
            i4a_cp(dst + 2 * C::CODES + lane * G * 4, cache.km + moff, row >= 0, std::integral_constant<int, G * 4>());
            i4a_cp(dst + 2 * C::CODES + C::META + lane * G * 4, cache.vm + moff, row >= 0, std::integral_constant<int, G * 4>());
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");                 // an empty group when nothing is left
        next += I4A_WARPS;
        slot_in = slot_in + 1 == I4A_STAGES ? 0 : slot_in + 1;
    };
#pragma unroll
    for (int i = 0; i < I4A_STAGES - 1; ++i) issue();

    // ---- the queries as operand fragments: lane (g, t) holds, of column g, numbers 16 t .. 16 t + 15 of every group
    uint4 qf[NT][2 * G];                                                       // of its two words each
    float qsum[NT][G][2], cscale[NT][2];                                       // of columns 2t, 2t + 1
    int pcol[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int c = nt * 8 + g;
        const bool live = c < n_cols;
        uint4 raw[G][2];
        uint32_t most = 0;
#pragma unroll
        for (int gr = 0; gr < G; ++gr)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                raw[gr][h] = live ? __ldg(reinterpret_cast<const uint4*>(q + result_row(c) * D + gr * 64 + t * 16 + h * 8)) : make_uint4(0, 0, 0, 0);
                const uint32_t w[4] = {raw[gr][h].x, raw[gr][h].y, raw[gr][h].z, raw[gr][h].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) most = max(most, max((w[e] & 0x7FFFu) << 16, w[e] & 0x7FFF0000u));
            }
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
        int ex;
        const float f = i4_factor(__uint_as_float(min(most, 0x7F7F0000u)), ex);
        // a query with a number that is not finite has no scores
        const float back = most > 0x7F7FFFFFu ? __uint_as_float(0x7FC00000u) : i4_pow2(ex) * 1024.f * scale_log2;
        float sum[G];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            sum[gr] = 0.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t w[4] = {raw[gr][h].x, raw[gr][h].y, raw[gr][h].z, raw[gr][h].w};
                float a[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    a[2 * e] = i4_bf16_low(w[e]) * f;
                    a[2 * e + 1] = i4_bf16_high(w[e]) * f;
                    sum[gr] += a[2 * e] + a[2 * e + 1];
                }
                qf[nt][gr * 2 + h] = i4_operand(a);
            }
            sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 1);
            sum[gr] += __shfl_xor_sync(0xffffffffu, sum[gr], 2);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int from = (2 * t + e) * 4;                                  // a lane that holds column 2t + e
#pragma unroll
            for (int gr = 0; gr < G; ++gr) qsum[nt][gr][e] = __shfl_sync(0xffffffffu, sum[gr], from) * I4_UNIT;
            cscale[nt][e] = __shfl_sync(0xffffffffu, back, from);
            const int cc = nt * 8 + 2 * t + e;
            pcol[nt][e] = cc < n_cols ? pos0 + (col0 + cc) / group : -1;       // no key is at or before -1
        }
    }

    float o[G * 4][NT][4], off_sum[NT][G][2], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < G * 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][nt][e] = 0.f;
#pragma unroll
        for (int gr = 0; gr < G; ++gr) off_sum[nt][gr][0] = off_sum[nt][gr][1] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
    }
    int vexp[G];                                                               // exponent that the steps of V are scaled by: their largest so far lands in [2^14, 2^15)
#pragma unroll
    for (int gr = 0; gr < G; ++gr) vexp[gr] = -113;

    const int perm = (0x57463120 >> (4 * g)) & 7;                              // row g of a tile is this key, row g + 8 eight behind
    const int kv0 = (0x57463120 >> (8 * t)) & 7, kv1 = (0x57463120 >> (8 * t + 4)) & 7;   // rows 2t, 2t + 1
    int slot_out = 0;
    for (int c = c_begin + warp; c < c_end; c += I4A_WARPS) {
        issue();
        asm volatile("cp.async.wait_group %0;\n" ::"n"(I4A_STAGES - 1) : "memory");
        __syncwarp();
        const unsigned char* sK = ring + slot_out * C::BYTES;
        const unsigned char* sV = sK + C::CODES;
        const unsigned char* sKM = sV + C::CODES;
        const unsigned char* sVM = sKM + C::META;
        slot_out = slot_out + 1 == I4A_STAGES ? 0 : slot_out + 1;
        const int j0 = c * I4A_KEYS;

        // ---- scores of 32 keys, in powers of two
        float s[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
            const int r = mt * 16 + perm;
            float z[G][NT][4];
#pragma unroll
            for (int gr = 0; gr < G; ++gr) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) z[gr][nt][e] = 0.f;
                const uint2 w0 = *reinterpret_cast<const uint2*>(sK + i4a_piece<D>(r, gr * 2 + (t >> 1)) + (t & 1) * 8);
                const uint2 w1 = *reinterpret_cast<const uint2*>(sK + i4a_piece<D>(r + 8, gr * 2 + (t >> 1)) + (t & 1) * 8);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t a0 = h ? w0.y : w0.x, a1 = h ? w1.y : w1.x, c0 = a0 >> 8, c1 = a1 >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const uint4 b = qf[nt][gr * 2 + h];
                        i4_mma(z[gr][nt], a0 & I4_NEAR, a1 & I4_NEAR, a0 & I4_FAR, a1 & I4_FAR, b.x, b.y);
                        i4_mma(z[gr][nt], c0 & I4_NEAR, c1 & I4_NEAR, c0 & I4_FAR, c1 & I4_FAR, b.z, b.w);
                    }
                }
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t meta[G];
#pragma unroll
                for (int gr = 0; gr < G; ++gr) meta[gr] = *reinterpret_cast<const uint32_t*>(sKM + (r + 8 * half) * G * 4 + gr * 4);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float v = 0.f;
#pragma unroll
                        for (int gr = 0; gr < G; ++gr)
                            v = fmaf(i4_bf16_low(meta[gr]), z[gr][nt][half * 2 + e], fmaf(i4_bf16_high(meta[gr]), qsum[nt][gr][e], v));
                        s[mt][nt][half * 2 + e] = v * cscale[nt][e];
                    }
            }
        }
        // ---- keys that a column does not see
        const bool edge = j0 + I4A_KEYS - 1 > first || (window > 0 && j0 <= hi - window);
        if (edge) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = j0 + mt * 16 + perm + (e >> 1) * 8, p = pcol[nt][e & 1];
                        if (j > p || (window > 0 && j <= p - window)) s[mt][nt][e] = -INFINITY;
                    }
        }
        // ---- running maximum, probabilities
        float corr[NT][2];
        bool moved = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float mx = fmaxf(fmaxf(s[0][nt][e], s[0][nt][e + 2]), fmaxf(s[1][nt][e], s[1][nt][e + 2]));
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                const float m_new = fmaxf(m[nt][e], mx), use = m_new == -INFINITY ? 0.f : m_new;
                moved |= m_new > m[nt][e];
                corr[nt][e] = i4a_exp2(m[nt][e] - use);
                m[nt][e] = m_new;
                float sum = 0.f;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        float& v = s[mt][nt][half * 2 + e];
                        v = i4a_exp2(v - use);
                        sum += v;
                    }
                l[nt][e] = l[nt][e] * corr[nt][e] + sum;
            }
        // ---- steps and offsets of this lane's four values per group; a larger step changes the scale of what is summed up
        float vs[G][2][2], vo[G][2][2];                                        // [tile][row g, g + 8]
        float grow[G];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
            uint32_t most = 0;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t meta = *reinterpret_cast<const uint32_t*>(sVM + (mt * 16 + perm + 8 * half) * G * 4 + gr * 4);
                    vs[gr][mt][half] = i4_bf16_low(meta);
                    vo[gr][mt][half] = i4_bf16_high(meta);
                    const uint32_t bits = meta << 16;                          // steps are never negative
                    most = max(most, bits < 0x7F800000u ? bits : 0u);
                }
            most = __reduce_max_sync(0xffffffffu, most);
            const int e = max((int)(most >> 23) - 127, -112);
            grow[gr] = 1.f;
            if (e > vexp[gr]) {                                                // the same for the whole warp
                grow[gr] = vexp[gr] < -112 ? 0.f : i4a_exp2((float)(vexp[gr] - e));      // nothing summed up yet: 0 times 0
                vexp[gr] = e;
                moved = true;
            }
            const float vscale = i4_pow2(14 - vexp[gr]);
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) vs[gr][mt][0] *= vscale, vs[gr][mt][1] *= vscale;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int gr = 0; gr < G; ++gr) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float f = corr[nt][e & 1] * grow[gr];
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[gr * 4 + i][nt][e] *= f;
                    }
                    off_sum[nt][gr][0] *= corr[nt][0];
                    off_sum[nt][gr][1] *= corr[nt][1];
                }
        }
        // ---- out^T += codes of V^T . (p step)^T
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint32_t b[NT][2];                                             // second operand: keys of rows 0-7 and 8-15
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const float p0 = s[mt][nt][half * 2], p1 = s[mt][nt][half * 2 + 1];
                        float x0 = p0 * vs[gr][mt][half], x1 = p1 * vs[gr][mt][half], f0 = p0 * vo[gr][mt][half], f1 = p1 * vo[gr][mt][half];
                        if (edge) {                                            // a value that is not finite does not reach the columns that do not see it
                            if (p0 == 0.f) x0 = f0 = 0.f;
                            if (p1 == 0.f) x1 = f1 = 0.f;
                        }
                        off_sum[nt][gr][0] += f0;
                        off_sum[nt][gr][1] += f1;
                        b[nt][half] = i4a_transpose(i4_f16x2(x0, x1));
                    }
                // words of numbers 8 g .. 8 g + 7 of the keys of rows 2t, 2t + 1, 2t + 8, 2t + 9
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int r = mt * 16 + (i & 1 ? kv1 : kv0) + (i >> 1) * 8;
                    w[i] = *reinterpret_cast<const uint32_t*>(sV + i4a_piece<D>(r, gr * 2 + (g >> 2)) + (g & 3) * 4);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {                                  // numbers 0-3 of the eight, then 4-7, of two keys each
                    const uint32_t a = __byte_perm(w[0], w[1], h ? 0x7632 : 0x5410), c = __byte_perm(w[2], w[3], h ? 0x7632 : 0x5410);
                    const uint32_t a8 = a >> 8, c8 = c >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        i4_mma(o[gr * 4 + 2 * h][nt], a & I4_NEAR, a & I4_FAR, c & I4_NEAR, c & I4_FAR, b[nt][0], b[nt][1]);
                        i4_mma(o[gr * 4 + 2 * h + 1][nt], a8 & I4_NEAR, a8 & I4_FAR, c8 & I4_NEAR, c8 & I4_FAR, b[nt][0], b[nt][1]);
                    }
                }
            }
        }
        __syncwarp();                                                          // every lane is done with the slot that is filled next
    }
    if (unmapped) atomicExch(status, 5);

    // ---- the warps meet: [warp][column][D + 4] outputs, then [warp][column] maximum and sum
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");
    __syncthreads();
    constexpr int LD = D + 4;
    float* so = reinterpret_cast<float*>(i4a_smem);
    float* sml = so + I4A_WARPS * COLS * LD;
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
                // 2^(vexp - 14) for the steps' scale, 2^24 for the codes', in two factors of which neither overflows
                const float back = vexp[gr] < -112 ? 0.f : i4_pow2(vexp[gr]);
                float* dst = so + (warp * COLS + cc) * LD + gr * 64 + 8 * g;
#pragma unroll
                for (int i = 0; i < 4; ++i) {                                  // numbers four bits up count 16 times
                    dst[2 * i] = fmaf(o[gr * 4 + i][nt][e] * 1024.f, back, f);
                    dst[2 * i + 1] = fmaf(o[gr * 4 + i][nt][e + 2] * 64.f, back, f);
                }
            }
            if (g == 0) {
                // a sum that is NaN (a key, a query that is not finite) keeps its place whatever the maximum is
                sml[(warp * COLS + cc) * 2] = sum == sum ? m[nt][e] : 0.f;
                sml[(warp * COLS + cc) * 2 + 1] = sum;
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < n_cols * (D / 4); i += I4A_THREADS) {
        const int cc = i / (D / 4), d4 = (i % (D / 4)) * 4;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < I4A_WARPS; ++w) M = fmaxf(M, sml[(w * COLS + cc) * 2]);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < I4A_WARPS; ++w) {
            const float mw = sml[(w * COLS + cc) * 2];
            if (mw == -INFINITY) continue;                                     // saw no key
            const float f = i4a_exp2(mw - M);
            const float4 v = *reinterpret_cast<const float4*>(so + (w * COLS + cc) * LD + d4);
            acc.x = fmaf(f, v.x, acc.x), acc.y = fmaf(f, v.y, acc.y), acc.z = fmaf(f, v.z, acc.z), acc.w = fmaf(f, v.w, acc.w);
            L = fmaf(f, sml[(w * COLS + cc) * 2 + 1], L);
        }
        const size_t row = result_row(cc);
        if (n_splits == 1) {
            const float inv = L == 0.f ? 0.f : 1.f / L;
            store4_act(out + row * D + d4, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        } else {
            *reinterpret_cast<float4*>(part_o + (row * n_splits + split) * D + d4) = acc;
            if (d4 == 0) {
                part_ml[(row * n_splits + split) * 2] = M;
                part_ml[(row * n_splits + split) * 2 + 1] = L == L ? L : 1.f;       // then the sums are NaN, and stay so
            }
        }
    }
}

// runs [n_runs, 4] (first token of the longest: most_rows), or none: every token is a sequence of its own.  With n_splits > 1 the
// result is left in part_o [tokens, n_q, n_splits, d] and part_ml [tokens, n_q, n_splits, 2] for gi_attention_decode_combine.
extern "C" int gi_int4_attention(const void* q, const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta,
                                 const int* table, const int* runs, int n_runs, int most_rows, const int* tok_pos, const int* tok_slot,
                                 void* out, float* part_o, float* part_ml, int n_q, int n_kv, int d, int n_slots, int max_pages,
                                 int page_size, int n_pages, int window, float scale, int n_splits, int* status, void* stream) {
    GI_REQUIRE(d == 64 || d == 128, "gi_int4_attention: heads of %d; 64 and 128 are possible", d);
    GI_REQUIRE(n_kv > 0 && n_q > 0 && n_q % n_kv == 0 && n_kv <= 65535, "gi_int4_attention: %d query heads over %d key/value heads", n_q, n_kv);
    GI_REQUIRE(n_runs >= 0 && n_runs <= 65535 && most_rows >= 1, "gi_int4_attention: %d runs of up to %d tokens", n_runs, most_rows);
    GI_REQUIRE(page_size > 0 && max_pages > 0 && n_slots > 0 && window >= 0, "gi_int4_attention: page and table sizes must be positive");
    GI_REQUIRE(n_splits >= 1 && n_splits <= 256 && (n_splits == 1 || (part_o && part_ml)), "gi_int4_attention: %d slices", n_splits);
    GI_REQUIRE((uintptr_t)q % 16 == 0 && (uintptr_t)k_codes % 16 == 0 && (uintptr_t)v_codes % 16 == 0 && (uintptr_t)k_meta % 8 == 0 &&
               (uintptr_t)v_meta % 8 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)part_o % 16 == 0 && (uintptr_t)runs % 16 == 0,
               "gi_int4_attention: operands must start on 16 bytes");
    if (n_runs == 0) return 0;
    const Int4Cache cache = {(const unsigned char*)k_codes, (const unsigned char*)v_codes, (const unsigned char*)k_meta, (const unsigned char*)v_meta};
    const long long cols = (long long)most_rows * (n_q / n_kv);
    const int nt = cols > 8 ? 2 : 1;
    const long long col_tiles = (cols + 8 * nt - 1) / (8 * nt);
    GI_REQUIRE(col_tiles * n_splits < 2147483647LL, "gi_int4_attention: runs of %d tokens are too long", most_rows);
#define GI_I4A(DD, NN)                                                                                                               \
    {                                                                                                                                \
        size_t smem = (size_t)I4A_WARPS * I4A_STAGES * Int4Chunk<DD>::BYTES;                                                         \
        const size_t meet = (size_t)I4A_WARPS * 8 * NN * (DD + 4 + 2) * 4;                                                           \
        if (meet > smem) smem = meet;                                                                                                \
        if (int rc = gi_reserve_smem((const void*)int4_attention_kernel<DD, NN>, smem, "gi_int4_attention")) return rc;              \
        gi_launch(int4_attention_kernel<DD, NN>, dim3((unsigned)(col_tiles * n_splits), n_kv, n_runs), dim3(I4A_THREADS), smem,      \
                  (cudaStream_t)stream, (const bf16*)q, cache, table, (const int4*)runs, tok_pos, tok_slot, (bf16*)out, part_o,      \
                  part_ml, n_q, n_kv, n_slots, max_pages, page_size, n_pages, window, scale * I4A_LOG2E, n_splits, (int)col_tiles,   \
                  status);                                                                                                           \
    }
    if (d == 64) { if (nt == 1) GI_I4A(64, 1) else GI_I4A(64, 2) }
    else { if (nt == 1) GI_I4A(128, 1) else GI_I4A(128, 2) }
#undef GI_I4A
    return gi_check_launch("gi_int4_attention");
}
