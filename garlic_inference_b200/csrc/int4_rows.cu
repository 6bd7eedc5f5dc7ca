// The key/value cache in 4 bits: new rows in, rows out.
//
// Pages are codes [pages, heads, page size, d / 2] bytes and meta [pages, heads, page size, d / 64] words (step, low as two
// bfloat16): a row of d numbers takes d / 2 + d / 16 bytes, 4.5 bits a number.  A group of 64 numbers of a head has one step:
//   low = min,  step = (max - min) / 15 rounded up to bfloat16,  q = round((x - low) / step) in 0 .. 15
// so that a number comes back within half a step.  Writing gives a group to 8 lanes, 8 numbers each (16 bytes of a bfloat16 row, 4 of codes);
// reading gives it to 4 lanes, 16 numbers each (8 bytes of codes, 32 of the result).  All are bound by the 16-bit side (2 bytes a number
// against 0.56), a step of a few tokens by the launch.
#include "int4.cuh"

#define I4R_THREADS 256
#define I4R_ROPE_WARPS 4

struct Int4Pool { unsigned char* codes; uint32_t* meta; };

// Where a token's rows of the cache are: the page and the row in it.  0, or what is wrong with the position (1) or the page (2).
__device__ __forceinline__ int i4r_place(int pos, int slot, const int* __restrict__ table, int n_slots, int max_pages, int page_size, int n_pages,
                                         long long& page, int& row) {
    const int lp = pos / page_size;
    if (pos < 0 || lp >= max_pages || slot >= n_slots) return 1;
    page = table[(size_t)slot * max_pages + lp];
    if (page < 0 || page >= n_pages) return 2;
    row = pos - lp * page_size;
    return 0;
}

// Keys and values of the step's tokens into their pages; k and v: a token's heads k_hs (v_hs) numbers apart, tokens k_ts (v_ts) apart.
template <typename T>
__global__ void __launch_bounds__(I4R_THREADS)
int4_append_kernel(const T* __restrict__ k, long long k_ts, long long k_hs, const T* __restrict__ v, long long v_ts, long long v_hs,
                   Int4Pool kp, Int4Pool vp, const int* __restrict__ table, const int* __restrict__ tok_pos,
                   const int* __restrict__ tok_slot, int n_kv, int groups, int n_slots, int max_pages, int page_size, int n_pages,
                   int vec, int* __restrict__ status) {
    gi_pdl_launch_dependents();
    const int at_group = (blockIdx.y * blockDim.x + threadIdx.x) >> 3, l = threadIdx.x & 7, tok = blockIdx.x;      // group: of keys, then of values
    const bool live = at_group < 2 * n_kv * groups;                      // 8 lanes alike; others of the warp may differ
    const bool values = at_group >= n_kv * groups;
    const int of_kind = values ? at_group - n_kv * groups : at_group, head = of_kind / groups, grp = of_kind - head * groups;
    // positions, slots and the block table are set before the step's first kernel: read before the wait
    long long page = 0;
    int row = 0;
    const int pos = tok_pos[tok], slot = tok_slot[tok];
    const int bad = slot < 0 ? 0 : i4r_place(pos, slot, table, n_slots, max_pages, page_size, n_pages, page, row);
    gi_pdl_wait();
    if (bad && live && l == 0) atomicExch(status, bad);
    const bool there = live && slot >= 0 && !bad;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (there) {
        const T* src = (values ? v + tok * v_ts + head * v_hs : k + tok * k_ts + head * k_hs) + grp * I4_GROUP_KV + l * 8;
        if (vec) {
            const float4 f = load4_act(src), h = load4_act(src + 4);
            x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w, x[4] = h.x, x[5] = h.y, x[6] = h.z, x[7] = h.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = to_f32(src[i]);
        }
    }
    float mn = x[0], mx = x[0];
    int odd = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mn = fminf(mn, x[i]), mx = fmaxf(mx, x[i]);
        odd |= !(fabsf(x[i]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        odd |= __shfl_xor_sync(0xffffffffu, odd, o);
    }
    if (!there) return;
    float step, low;
    i4_step_low(mn, mx, !odd, step, low);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) bits |= i4_code(x[i], step, low) << (4 * i);
    const Int4Pool pool = values ? vp : kp;
    const size_t at = (((size_t)page * n_kv + head) * page_size + row) * groups + grp;
    reinterpret_cast<uint32_t*>(pool.codes)[at * 8 + l] = bits;
    if (l == 0) pool.meta[at] = i4_meta(step, low);
}

// What the attention layers do to the joined projection qkv [tokens, (n_q + 2 n_kv) d] before the cache: RMSNorm over each head of q and k
// (with weights), rotation of the first rotary_dim numbers by cos/sin [positions, rotary_dim / 2] (number i with i + rotary_dim / 2), q
// rounded to q_out [tokens, n_q, d], k (float32, not rounded before) and v into their pages.  A warp takes a head of a token.
template <int EPL>
__global__ void __launch_bounds__(I4R_ROPE_WARPS * 32)
int4_qk_norm_rope_append_kernel(const bf16* __restrict__ qkv, bf16* __restrict__ q_out, Int4Pool kp, Int4Pool vp, const void* __restrict__ q_w,
                                const void* __restrict__ k_w, int w_dtype, float eps, const float* __restrict__ cos_t,
                                const float* __restrict__ sin_t, int rotary_dim, const int* __restrict__ tok_pos,
                                const int* __restrict__ tok_slot, const int* __restrict__ table, int n_q, int n_kv, int n_slots,
                                int max_pages, int page_size, int n_pages, int max_positions, int heads_here, int* __restrict__ status) {
    constexpr int d = EPL * 32, LANES = I4_GROUP_KV / EPL;              // lanes of a group
    __shared__ float s_head[I4R_ROPE_WARPS][d];
    gi_pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tok = blockIdx.x, h = blockIdx.y * I4R_ROPE_WARPS + warp;
    const int half = rotary_dim / 2;
    const bool is_q = h < n_q, is_v = h >= n_q + n_kv;
    // positions, slots, the block table and the rotation table are set before the step's first kernel: read before the wait
    const int pos = tok_pos[tok], slot = is_q ? 0 : tok_slot[tok];
    long long page = 0;
    int row = 0, bad = 0;
    if (!is_q && slot >= 0) bad = i4r_place(pos, slot, table, n_slots, max_pages, page_size, n_pages, page, row);
    if (!bad && !is_v && (pos < 0 || pos >= max_positions)) bad = 3;
    gi_pdl_wait();                                                      // by every block, whatever it finds: the next kernel's start rests on it
    if (h >= heads_here || slot < 0) return;
    if (bad) {
        if (lane == 0) atomicExch(status, bad);
        return;
    }
    float x[EPL];
    const bf16* src = qkv + ((size_t)tok * (n_q + 2 * n_kv) + h) * d + lane * EPL;
#pragma unroll
    for (int e = 0; e < EPL; e += 2) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(src + e);
        x[e] = i4_bf16_low(w), x[e + 1] = i4_bf16_high(w);
    }
    if (!is_v) {
        const void* w = is_q ? q_w : k_w;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) ss += x[e] * x[e];
            const float inv = rsqrtf(warp_sum(ss) / (float)d + eps);
#pragma unroll
            for (int e = 0; e < EPL; ++e) x[e] = x[e] * inv * load_w(w, w_dtype, lane * EPL + e);
        }
#pragma unroll
        for (int e = 0; e < EPL; ++e) s_head[warp][lane * EPL + e] = x[e];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const int i = lane * EPL + e;
            if (i < rotary_dim) {
                const int j = i < half ? i : i - half;
                const float c = cos_t[(size_t)pos * half + j], s = sin_t[(size_t)pos * half + j], other = s_head[warp][i < half ? i + half : j];
                x[e] = i < half ? x[e] * c - other * s : x[e] * c + other * s;
            }
        }
    }
    if (is_q) {
        bf16* dst = q_out + ((size_t)tok * n_q + h) * d + lane * EPL;
#pragma unroll
        for (int e = 0; e < EPL; e += 2) *reinterpret_cast<__nv_bfloat162*>(dst + e) = __floats2bfloat162_rn(x[e], x[e + 1]);
        return;
    }
    float mn = x[0], mx = x[0], step, low;
    int odd = 0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        mn = fminf(mn, x[e]), mx = fmaxf(mx, x[e]);
        odd |= !(fabsf(x[e]) <= 3.402823466e38f);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        odd |= __shfl_xor_sync(0xffffffffu, odd, o);
    }
    i4_step_low(mn, mx, !odd, step, low);
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < EPL; ++e) bits |= i4_code(x[e], step, low) << (4 * e);
    const Int4Pool pool = is_v ? vp : kp;
    const size_t at = (((size_t)page * n_kv + (h - n_q - (is_v ? n_kv : 0))) * page_size + row) * (d / I4_GROUP_KV) + lane / LANES;
    if (EPL == 4) reinterpret_cast<uint16_t*>(pool.codes)[at * 16 + lane % LANES] = (uint16_t)bits;
    else pool.codes[at * 32 + lane % LANES] = (unsigned char)bits;
    if (lane % LANES == 0) pool.meta[at] = i4_meta(step, low);
}

// 16 numbers
template <typename T>
__device__ __forceinline__ void i4r_unpack(T* dst, uint2 bits, uint32_t meta) {
    const float step = i4_bf16_low(meta), low = i4_bf16_high(meta);
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
        const uint32_t b = (i < 8 ? bits.x : bits.y) >> (4 * (i & 7));
        store4_act(dst + i, make_float4(fmaf(step, (float)(b & 15), low), fmaf(step, (float)((b >> 4) & 15), low),
                                        fmaf(step, (float)((b >> 8) & 15), low), fmaf(step, (float)((b >> 12) & 15), low)));
    }
}
__device__ __forceinline__ void i4r_unpack(bf16* dst, uint2 bits, uint32_t meta) {
    const float step = i4_bf16_low(meta), low = i4_bf16_high(meta);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t b = h ? bits.y : bits.x;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<__nv_bfloat162*>(&w[i]) = __floats2bfloat162_rn(fmaf(step, (float)((b >> (8 * i)) & 15), low), fmaf(step, (float)((b >> (8 * i + 4)) & 15), low));
        reinterpret_cast<uint4*>(dst)[h] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// What the pages hold of the listed tokens: out [tokens, n_kv, d], zeros for padding and where no page is mapped.
template <typename T>
__global__ void __launch_bounds__(I4R_THREADS)
int4_read_kernel(Int4Pool pool, T* __restrict__ out, const int* __restrict__ table, const int* __restrict__ tok_pos,
                 const int* __restrict__ tok_slot, int n_kv, int groups, int n_slots, int max_pages, int page_size, int n_pages,
                 int items, int* __restrict__ status) {
    gi_pdl_start();
    const int item = blockIdx.x * I4R_THREADS + threadIdx.x;
    if (item >= items) return;
    const int l = item & 3, head_group = item >> 2, per = n_kv * groups, tok = head_group / per, of_tok = head_group - tok * per;
    const int head = of_tok / groups, grp = of_tok - head * groups;
    long long page;
    int row;
    uint2 bits = make_uint2(0, 0);
    uint32_t meta = 0;
    const int pos = tok_pos[tok], slot = tok_slot[tok];
    const int bad = slot < 0 ? 0 : i4r_place(pos, slot, table, n_slots, max_pages, page_size, n_pages, page, row);
    if (bad && l == 0) atomicExch(status, bad);
    if (slot >= 0 && !bad) {
        const size_t at = (((size_t)page * n_kv + head) * page_size + row) * groups + grp;
        bits = reinterpret_cast<const uint2*>(pool.codes)[at * 4 + l];
        meta = pool.meta[at];
    }
    i4r_unpack(out + (size_t)item * 16, bits, meta);
}

// Blocks of 64 positions of the step's sequences, each number rounded to bfloat16 (which holds whatever a step and a low value make, next to
// any other; the prompt kernel's operands are that), as pages of their own, [blocks, n_kv, 64, d], for the prompt kernel on
// tensor memory, and their block table [n_slots, max_blocks]: block i holds positions 64 b .. of the slot that blocks[i] =
// {slot, b} names.  Positions without a page are zeros, as are those behind the table's last column; one that a run sees is reported.  runs_out: the
// runs, those that name a slot, rows or positions that do not exist as empty ones (the prompt kernel takes them as they are).
__global__ void __launch_bounds__(I4R_THREADS)
int4_gather_kernel(Int4Pool kp, Int4Pool vp, bf16* __restrict__ k_out, bf16* __restrict__ v_out, int* __restrict__ out_table,
                   const int2* __restrict__ blocks, const int4* __restrict__ runs, int4* __restrict__ runs_out, int n_runs, int n_rows,
                   const int* __restrict__ table, int n_kv, int groups, int n_slots, int max_pages, int max_blocks, int page_size,
                   int n_pages, int window, int* __restrict__ status) {
    gi_pdl_start();
    auto run_there = [&](int4 r) {
        return r.x < n_slots && r.y >= 0 && r.z <= 128 && r.z <= n_rows && r.y <= n_rows - r.z && r.w >= 0 && r.w <= 2147483647 - 128 &&
               (r.w + r.z - 1) / page_size < max_pages;
    };
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < n_runs; i += I4R_THREADS) {
            int4 r = runs[i];
            const bool there = run_there(r);
            if (r.x >= 0 && r.z > 0 && !there) atomicExch(status, 4);
            if (r.x < 0 || r.z <= 0 || !there) r = make_int4(-1, 0, 0, 0);
            runs_out[i] = r;
        }
    const int2 b = blocks[blockIdx.x];
    const bool ok = b.x >= 0 && b.x < n_slots && b.y >= 0 && b.y < max_blocks;
    if (blockIdx.y == 0 && threadIdx.x == 0) {
        if (ok) out_table[(size_t)b.x * max_blocks + b.y] = blockIdx.x;
        else atomicExch(status, 1);
    }
    const int head = blockIdx.y >> 1;
    const Int4Pool pool = blockIdx.y & 1 ? vp : kp;
    bf16* out = (blockIdx.y & 1 ? v_out : k_out) + ((size_t)blockIdx.x * n_kv + head) * 64 * groups * I4_GROUP_KV;
    // 64 rows x groups x 4 lanes: the lanes of a warp lie in 8 or 4 rows of a page, or of two
    for (int i = threadIdx.x; i < 64 * groups * 4; i += I4R_THREADS) {
        const int l = i & 3, of_row = i >> 2, r = of_row / groups, grp = of_row - r * groups, pos = b.y * 64 + r, lp = pos / page_size;
        uint2 bits = make_uint2(0, 0);
        uint32_t meta = 0;
        if (ok && lp < max_pages) {
            const int page = __ldg(table + (size_t)b.x * max_pages + lp);
            if (page >= 0 && page < n_pages) {
                const size_t at = (((size_t)page * n_kv + head) * page_size + (pos - lp * page_size)) * groups + grp;
                bits = reinterpret_cast<const uint2*>(pool.codes)[at * 4 + l];
                meta = pool.meta[at];
            } else if (blockIdx.y == 0 && l == 0 && grp == 0) {                // of the first head's keys: is it one that a run sees?
                for (int j = 0; j < n_runs; ++j) {
                    const int4 r = runs[j];
                    if (r.x == b.x && r.z > 0 && run_there(r) && pos < r.w + r.z && (window == 0 || pos > r.w - window)) {
                        atomicExch(status, 5);
                        break;
                    }
                }
            }
        }
        i4r_unpack(out + (size_t)i * 16, bits, meta);
    }
}

// Listed rows of a matrix, 16 bytes a piece, into a dense one (put: from it), for the short sequences of a step.  A row that does not exist is reported:
// zeros are taken for it, and it is put nowhere.
__global__ void __launch_bounds__(I4R_THREADS)
int4_move_rows_kernel(uint4* __restrict__ matrix, uint4* __restrict__ some, const int* __restrict__ rows, int n, int pieces, int put,
                      int* __restrict__ status) {
    gi_pdl_start();
    const int row = rows[blockIdx.x];
    const bool there = row >= 0 && row < n;
    if (!there && threadIdx.x == 0) atomicExch(status, 4);
    uint4* const at = matrix + (size_t)(there ? row : 0) * pieces;
    uint4* const to = some + (size_t)blockIdx.x * pieces;
    for (int i = threadIdx.x; i < pieces; i += I4R_THREADS) {
        if (!put) to[i] = there ? at[i] : make_uint4(0, 0, 0, 0);
        else if (there) at[i] = to[i];
    }
}

static int check_pool(const char* who, const void* codes, const void* meta, int n_kv, int d, int page_size, int max_pages, int n_slots) {
    GI_REQUIRE(n_kv > 0 && d > 0 && d % I4_GROUP_KV == 0 && d <= 1024, "%s: %d heads of %d; heads are multiples of 64 numbers", who, n_kv, d);
    GI_REQUIRE(page_size > 0 && max_pages > 0 && n_slots > 0, "%s: page and table sizes must be positive", who);
    GI_REQUIRE((uintptr_t)codes % 16 == 0 && (uintptr_t)meta % 16 == 0, "%s: pages must start on 16 bytes", who);
    return 0;
}

extern "C" int gi_int4_append(const void* k, long long k_ts, long long k_hs, const void* v, long long v_ts, long long v_hs, int dtype,
                              void* k_codes, void* k_meta, void* v_codes, void* v_meta, const int* table, const int* tok_pos,
                              const int* tok_slot, int n_tokens, int n_kv, int d, int n_slots, int max_pages, int page_size,
                              int n_pages, int* status, void* stream) {
    if (int rc = check_pool("gi_int4_append", k_codes, k_meta, n_kv, d, page_size, max_pages, n_slots)) return rc;
    if (int rc = check_pool("gi_int4_append", v_codes, v_meta, n_kv, d, page_size, max_pages, n_slots)) return rc;
    GI_REQUIRE(n_tokens >= 0, "gi_int4_append: %d tokens", n_tokens);
    if (n_tokens == 0) return 0;
    const int groups = d / I4_GROUP_KV;
    const int lanes = n_kv * 2 * groups * 8, threads = lanes < I4R_THREADS ? lanes + 31 & ~31 : I4R_THREADS;
    GI_REQUIRE(n_kv <= 32768, "gi_int4_append: %d heads", n_kv);
    const size_t eight = dtype == GI_DTYPE_F32 ? 32 : 16;                // bytes of eight numbers
    const int vec = (uintptr_t)k % eight == 0 && (uintptr_t)v % eight == 0 && k_ts % 8 == 0 && k_hs % 8 == 0 && v_ts % 8 == 0 && v_hs % 8 == 0;
    const Int4Pool kp = {(unsigned char*)k_codes, (uint32_t*)k_meta}, vp = {(unsigned char*)v_codes, (uint32_t*)v_meta};
    cudaStream_t s = (cudaStream_t)stream;
#define GI_APPEND(T)                                                                                                                 \
    gi_launch(int4_append_kernel<T>, dim3(n_tokens, (lanes + threads - 1) / threads), dim3(threads), 0, s, (const T*)k, k_ts, k_hs, (const T*)v, v_ts,    \
              v_hs, kp, vp, table, tok_pos, tok_slot, n_kv, groups, n_slots, max_pages, page_size, n_pages, vec, status)
    if (dtype == GI_DTYPE_F32) GI_APPEND(float);
    else if (dtype == GI_DTYPE_BF16) GI_APPEND(bf16);
    else GI_REQUIRE(false, "gi_int4_append: dtype %d", dtype);
#undef GI_APPEND
    return gi_check_launch("gi_int4_append");
}

extern "C" int gi_int4_qk_norm_rope_append(const void* qkv, void* q_out, void* k_codes, void* k_meta, void* v_codes, void* v_meta,
                                           const void* q_w, const void* k_w, int w_dtype, float eps, const float* cos_t,
                                           const float* sin_t, int rotary_dim, const int* tok_pos, const int* tok_slot, const int* table,
                                           int n_tokens, int n_q, int n_kv, int d, int n_slots, int max_pages, int page_size,
                                           int n_pages, int max_positions, int append, int* status, void* stream) {
    const char* who = "gi_int4_qk_norm_rope_append";
    if (int rc = check_pool(who, k_codes, k_meta, n_kv, d, page_size, max_pages, n_slots)) return rc;
    if (int rc = check_pool(who, v_codes, v_meta, n_kv, d, page_size, max_pages, n_slots)) return rc;
    GI_REQUIRE(d == 64 || d == 128, "%s: heads of %d; 64 and 128 are possible", who, d);
    GI_REQUIRE(n_tokens >= 0 && n_q > 0 && (long long)n_q + 2LL * n_kv <= 65535 * I4R_ROPE_WARPS, "%s: %d tokens, %d query heads", who, n_tokens, n_q);
    GI_REQUIRE(rotary_dim >= 0 && rotary_dim <= d && rotary_dim % 2 == 0, "%s: rotary_dim %d must be even and at most %d", who, rotary_dim, d);
    GI_REQUIRE((q_w == nullptr) == (k_w == nullptr), "%s: q and k norm weights go together", who);
    GI_REQUIRE((uintptr_t)qkv % 4 == 0 && (uintptr_t)q_out % 4 == 0, "%s: qkv and q must start on 4 bytes", who);
    if (n_tokens == 0) return 0;
    const int heads_here = append ? n_q + 2 * n_kv : n_q;
    const Int4Pool kp = {(unsigned char*)k_codes, (uint32_t*)k_meta}, vp = {(unsigned char*)v_codes, (uint32_t*)v_meta};
    const dim3 grid(n_tokens, (heads_here + I4R_ROPE_WARPS - 1) / I4R_ROPE_WARPS);
#define GI_ROPE4(EPL)                                                                                                                \
    gi_launch(int4_qk_norm_rope_append_kernel<EPL>, grid, dim3(I4R_ROPE_WARPS * 32), 0, (cudaStream_t)stream, (const bf16*)qkv,      \
              (bf16*)q_out, kp, vp, q_w, k_w, w_dtype, eps, cos_t, sin_t, rotary_dim, tok_pos, tok_slot, table, n_q, n_kv, n_slots,  \
              max_pages, page_size, n_pages, max_positions, heads_here, status)
    if (d == 64) GI_ROPE4(2);
    else GI_ROPE4(4);
#undef GI_ROPE4
    return gi_check_launch(who);
}

extern "C" int gi_int4_read(const void* codes, const void* meta, void* out, int dtype, const int* table, const int* tok_pos,
                            const int* tok_slot, int n_tokens, int n_kv, int d, int n_slots, int max_pages, int page_size, int n_pages,
                            int* status, void* stream) {
    if (int rc = check_pool("gi_int4_read", codes, meta, n_kv, d, page_size, max_pages, n_slots)) return rc;
    GI_REQUIRE(n_tokens >= 0 && (uintptr_t)out % 16 == 0, "gi_int4_read: %d tokens, the output must start on 16 bytes", n_tokens);
    if (n_tokens == 0) return 0;
    const int groups = d / I4_GROUP_KV;
    GI_REQUIRE((long long)n_tokens * n_kv * groups * 4 < 2147483647LL - I4R_THREADS, "gi_int4_read: too many (token, head) pairs");
    const int items = n_tokens * n_kv * groups * 4, blocks = (items + I4R_THREADS - 1) / I4R_THREADS;
    const Int4Pool pool = {(unsigned char*)codes, (uint32_t*)meta};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == GI_DTYPE_F32)
        gi_launch(int4_read_kernel<float>, dim3(blocks), dim3(I4R_THREADS), 0, s, pool, (float*)out, table, tok_pos, tok_slot, n_kv, groups, n_slots, max_pages, page_size, n_pages, items, status);
    else if (dtype == GI_DTYPE_BF16)
        gi_launch(int4_read_kernel<bf16>, dim3(blocks), dim3(I4R_THREADS), 0, s, pool, (bf16*)out, table, tok_pos, tok_slot, n_kv, groups, n_slots, max_pages, page_size, n_pages, items, status);
    else GI_REQUIRE(false, "gi_int4_read: dtype %d", dtype);
    return gi_check_launch("gi_int4_read");
}

extern "C" int gi_int4_move_rows(void* matrix, void* some, const int* rows, int n_some, int n, long long row_bytes, int put, int* status,
                                 void* stream) {
    GI_REQUIRE(n_some >= 0 && n >= 0 && row_bytes > 0 && row_bytes % 16 == 0 && row_bytes / 16 < (1 << 30) && (uintptr_t)matrix % 16 == 0 &&
               (uintptr_t)some % 16 == 0, "gi_int4_move_rows: %d of %d rows of %lld bytes; rows must start on 16", n_some, n, row_bytes);
    if (n_some == 0) return 0;
    gi_launch(int4_move_rows_kernel, dim3((unsigned)n_some), dim3(I4R_THREADS), 0, (cudaStream_t)stream, (uint4*)matrix, (uint4*)some, rows, n,
              (int)(row_bytes / 16), put, status);
    return gi_check_launch("gi_int4_move_rows");
}

extern "C" int gi_int4_gather(const void* k_codes, const void* k_meta, const void* v_codes, const void* v_meta, void* k_out, void* v_out,
                              int* out_table, const int* blocks, int n_blocks, const int* runs, int* runs_out, int n_runs, int n_rows, const int* table, int n_kv, int d, int n_slots,
                              int max_pages, int max_blocks, int page_size, int n_pages, int window, int* status, void* stream) {
    if (int rc = check_pool("gi_int4_gather", k_codes, k_meta, n_kv, d, page_size, max_pages, n_slots)) return rc;
    if (int rc = check_pool("gi_int4_gather", v_codes, v_meta, n_kv, d, page_size, max_pages, n_slots)) return rc;
    GI_REQUIRE(n_blocks >= 0 && max_blocks > 0 && n_kv <= 32767 && (uintptr_t)blocks % 8 == 0 && (uintptr_t)k_out % 16 == 0 && (uintptr_t)v_out % 16 == 0,
               "gi_int4_gather: %d blocks of %d heads; blocks must start on 8 bytes, the pages on 16", n_blocks, n_kv);
    GI_REQUIRE(window >= 0, "gi_int4_gather: a window of %d", window);
    GI_REQUIRE(n_blocks > 0 && n_runs >= 0 && n_rows >= 0 && (uintptr_t)runs % 16 == 0 && (uintptr_t)runs_out % 16 == 0,
               "gi_int4_gather: %d runs over %d blocks; runs must start on 16 bytes", n_runs, n_blocks);
    const Int4Pool kp = {(unsigned char*)k_codes, (uint32_t*)k_meta}, vp = {(unsigned char*)v_codes, (uint32_t*)v_meta};
    gi_launch(int4_gather_kernel, dim3((unsigned)n_blocks, (unsigned)(2 * n_kv)), dim3(I4R_THREADS), 0, (cudaStream_t)stream, kp, vp, (bf16*)k_out,
              (bf16*)v_out, out_table, (const int2*)blocks, (const int4*)runs, (int4*)runs_out, n_runs, n_rows, table, n_kv, d / I4_GROUP_KV, n_slots, max_pages, max_blocks, page_size,
              n_pages, window, status);
    return gi_check_launch("gi_int4_gather");
}
