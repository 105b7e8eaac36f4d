// Log probabilities of given tokens, with the entropy of their rows and the likeliest alternatives.
//
// A row of logits x (not a number counts as minus infinity):
//   m = max x,  s = sum exp(x - m),  u = sum exp(x - m) (x - m);
//   logprob = (x[token] - m) - ln s,  lse = m + ln s,  entropy = -sum p ln p = ln s - u / s,
// and the k largest logits, the first id first among equals, as (x - m) - ln s.  All three sums are kept over any part of a
// row in one pass, the maximum as it is so far; two parts join as
//   m = max(m1, m2),  f_i = exp(m_i - m),  s = sum f_i s_i,  u = sum f_i (u_i + (m_i - m) s_i).
// A row with nothing above minus infinity has no distribution: its log probabilities are minus infinity, its entropy is 0.
// A row with plus infinity has entropy NaN and log probabilities x - inf.  A token outside the vocabulary has minus infinity.
//
// The reference takes the same numbers from whole rows on the host (crates/airun-core/src/sample.rs:128-140, :489-503).
#include "common.cuh"

typedef unsigned long long u64;

#define TOP_MAX 128

// ------------------------------------------------------------------ parts of a row
struct Part { float m, s, u; };

__device__ __forceinline__ Part join(const Part& a, const Part& b) {
    const float m = fmaxf(a.m, b.m);
    // (both empty: the differences are not numbers, and the bound makes them terms of zero)
    const float da = fmaxf(a.m - m, -200.0f), db = fmaxf(b.m - m, -200.0f), fa = __expf(da), fb = __expf(db);
    return {m, fa * a.s + fb * b.s, fa * fmaf(da, a.s, a.u) + fb * fmaf(db, b.s, b.u)};
}

// A part whose maximum so far becomes `m`, larger than before.
__device__ __forceinline__ void raise_max(Part& p, float m) {
    const float d = fmaxf(p.m - m, -200.0f), f = __expf(d);
    p.u = f * fmaf(d, p.s, p.u);
    p.s *= f;
    p.m = m;
}

// One logit below or at the maximum so far.  Minus infinity, NaN and what is 200 below the maximum add exp(-200) = 0.
__device__ __forceinline__ void add_logit(Part& p, float x) {
    const float d = fmaxf(x - p.m, -200.0f), e = __expf(d);
    p.s += e;
    p.u = fmaf(e, d, p.u);
}

__device__ __forceinline__ Part warp_join(Part p) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        p = join(p, Part{__shfl_xor_sync(0xffffffffu, p.m, o), __shfl_xor_sync(0xffffffffu, p.s, o), __shfl_xor_sync(0xffffffffu, p.u, o)});
    return p;
}

// The joined part of the block's threads, in thread 0's warp.  `sh` holds one Part a warp.
template <int NT> __device__ __forceinline__ Part block_join(Part p, Part* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    p = warp_join(p);
    __syncthreads();
    if (lane == 0) sh[warp] = p;
    __syncthreads();
    if (warp == 0) p = warp_join(lane < NT / 32 ? sh[lane] : Part{-INFINITY, 0.0f, 0.0f});
    return p;
}

__device__ __forceinline__ float log_prob(const Part& p, float ln_s, float x) {
    if (!(x > -INFINITY) || p.m == -INFINITY) return -INFINITY;
    return p.m == INFINITY ? x - p.m : (x - p.m) - ln_s;
}

// ------------------------------------------------------------------ the k largest of many
// A logit and its id as one number: larger logits first, among equals the lower id first; 0 is no logit.  -0 counts as 0.
__device__ __forceinline__ u64 key_of(float x, int id) {
    if (x != x) x = -INFINITY;
    unsigned b = __float_as_uint(x + 0.0f);
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((u64)b << 32) | (u64)(0xFFFFFFFFu - (unsigned)id);
}
__device__ __forceinline__ float key_logit(u64 k) {
    const unsigned b = (unsigned)(k >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ int key_id(u64 k) { return (int)(0xFFFFFFFFu - (unsigned)(k & 0xFFFFFFFFull)); }

template <int NT> struct TopShared {
    static constexpr int CAP = NT >= 256 ? 4096 : 2048;       // keys of the list
    u64 group[NT];
    u64 list[CAP];
    u64 top[TOP_MAX];
    u64 cut;
    int count;
};

// The k largest of all threads' keys, in order, in sh.top (0 beyond the last).  The threads' keys are all different; `best` is a
// thread's largest (0: it has none) and each(f) calls f on every key of the thread, or on all that can be as large as `cut`.
// The k-th largest of the maxima of groups of threads is a lower bound of the k-th largest of all, and close to it when
// there are twice as many groups as wanted keys: about k to 2 k keys reach it.  Those are listed and each counts the larger ones.
// A group is as many lanes as leave 2 k groups; equal logits in every place, whose keys fall with the id, then list
// k groups' first vectors: 4,096 keys at the most.  A list longer than `few` is cut again in the same way.
template <int NT, typename Each>
__device__ __forceinline__ void select_top(TopShared<NT>& sh, u64 best, int k, Each each) {
    constexpr int CAP = TopShared<NT>::CAP, MINE = CAP / NT;
    const int tid = threadIdx.x;
    int g = 32;
    while (g > 1 && NT / g < 2 * k) g >>= 1;
    const int groups = NT / g;
    auto find_cut = [&](u64 b) {
        for (int o = 1; o < g; o <<= 1) {
            const u64 other = __shfl_xor_sync(0xffffffffu, b, o);
            b = other > b ? other : b;
        }
        __syncthreads();
        if (tid % g == 0) sh.group[tid / g] = b;
        if (tid == 0) { sh.cut = 1; sh.count = 0; }
        __syncthreads();
        if (tid < groups) {
            const u64 mine = sh.group[tid];
            int larger = 0;
#pragma unroll 8
            for (int j = 0; j < groups; ++j) larger += sh.group[j] > mine;
            if (larger == k - 1 && mine != 0) sh.cut = mine;
        }
        __syncthreads();
        return sh.cut;
    };
    auto push = [&](u64 key) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < CAP) sh.list[at] = key;
    };
    u64 cut = find_cut(best);
    if (best >= cut) each(cut, [&](u64 key) { if (key >= cut) push(key); });
    for (int i = tid; i < k; i += NT) sh.top[i] = 0;
    __syncthreads();
    int n = sh.count;
    if (n > CAP) {
        // more keys reach the bound than the list holds (large logits that repeat at the threads' stride): one after the other
        u64 below = ~0ull;
        for (int i = 0; i < k; ++i) {
            u64 b = 0;
            if (best != 0) each(1ull, [&](u64 key) { if (key < below && key > b) b = key; });
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const u64 other = __shfl_xor_sync(0xffffffffu, b, o);
                b = other > b ? other : b;
            }
            __syncthreads();
            if ((tid & 31) == 0) sh.group[tid >> 5] = b;
            __syncthreads();
            b = 0;
            for (int w = 0; w < NT / 32; ++w) b = sh.group[w] > b ? sh.group[w] : b;
            if (tid == 0) sh.top[i] = b;
            below = b;
            if (b == 0) break;                                   // (the same for all threads)
        }
        __syncthreads();
        return;
    }
    const int few = 2 * k > 128 ? 2 * k : 128;
    for (int round = 0; round < 4 && n > few; ++round) {
        u64 mine[MINE], b = 0;
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            mine[i] = tid + i * NT < n ? sh.list[tid + i * NT] : 0;
            b = mine[i] > b ? mine[i] : b;
        }
        cut = find_cut(b);                                       // (its first barrier: every thread has read its keys)
#pragma unroll
        for (int i = 0; i < MINE; ++i) if (mine[i] >= cut) push(mine[i]);
        __syncthreads();
        const int now = sh.count;
        if (now >= n) break;
        n = now;
    }
    for (int i = tid; i < n; i += NT) {
        const u64 mine = sh.list[i];
        int larger = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) larger += sh.list[j] > mine;
        if (larger < k) sh.top[larger] = mine;
    }
    __syncthreads();
}

// ------------------------------------------------------------------ from logits
struct TokenParams {
    const void* logits;
    long long ld;
    int held, V;                       // rows and columns of the buffer
    const int32_t* rows;               // the rows that are asked for, or null: 0 .. n - 1
    const int32_t* tokens;
    float *logprob, *entropy, *lse;    // [n] (entropy, lse: or null)
    int k;
    int32_t* top_ids;                  // [n][k]
    float* top_logprobs;
    int* err;
};

template <typename T> struct Pack;
template <> struct Pack<float> {
    static constexpr int N = 4;
    float4 v;
    __device__ __forceinline__ float at(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    uint4 v;
    __device__ __forceinline__ float at(int i) const {
        const unsigned w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
        return __uint_as_float((i & 1) ? (w & 0xFFFF0000u) : (w << 16));
    }
};

// A cluster of C blocks a row (C = 1: a block).  The row's 16-byte vectors are dealt to the blocks in turn ranges and, inside, to
// the threads in batches of U: a thread's elements come by ascending id.  The few elements ahead of the first
// 16-byte boundary and behind the last belong to the first block's first threads and the last block's first threads.
template <typename T, int NT, bool CLUSTER>
__global__ __launch_bounds__(NT) void token_logprobs_kernel(const TokenParams p, int n_parts) {
    pdl_trigger();
    constexpr int VEC = Pack<T>::N, U = 4;
    __shared__ TopShared<NT> top;
    __shared__ Part s_parts[32];
    __shared__ Part s_mine;
    const int tid = threadIdx.x;
    const int part = CLUSTER ? (int)cluster_rank() : 0, parts = CLUSTER ? n_parts : 1;
    const int r = CLUSTER ? blockIdx.x / parts : blockIdx.x;
    pdl_wait();
    const int at = p.rows ? p.rows[r] : r;
    const int token = p.tokens[r];
    const bool there = at >= 0 && at < p.held;
    if (!there && tid == 0 && part == 0 && p.err) atomicOr(p.err, AIRUN_DEV_BAD_ROW);
    const int V = there ? p.V : 0;
    const T* row = (const T*)p.logits + (size_t)(there ? at : 0) * p.ld;
    const float given = part == 0 && token >= 0 && token < V ? to_f32<T>(row[token]) : -INFINITY;

    const int lead = min(V, (int)((16 - ((uintptr_t)row & 15)) % 16 / sizeof(T)));
    const int vecs = (V - lead) / VEC, tail = lead + vecs * VEC;
    const int v0 = (int)((long long)vecs * part / parts), v1 = (int)((long long)vecs * (part + 1) / parts);
    const int n_batches = (v1 - v0 + U * NT - 1) / (U * NT);
    const Pack<T>* from = reinterpret_cast<const Pack<T>*>(row + lead);
    // the element ahead of the vectors that is this thread's, and the one behind them
    const int ahead = part == 0 && tid < lead ? tid : -1, behind = part == parts - 1 && tid < V - tail ? tail + tid : -1;

    Part mine = {-INFINITY, 0.0f, 0.0f};
    float second = -INFINITY;                                    // largest of the batches but the one with the maximum
    int best_batch = -1;
    if (ahead >= 0) {
        const float x = to_f32<T>(row[ahead]);
        if (x > mine.m) mine.m = x;
        add_logit(mine, x);
        second = mine.m;                                         // (its own key is looked at below)
    }
    for (int b = 0; b < n_batches; ++b) {
        Pack<T> x[U];
        const int first = v0 + b * U * NT + tid;
#pragma unroll
        for (int i = 0; i < U; ++i) if (first + i * NT < v1) x[i] = from[first + i * NT];
        float most = -INFINITY;
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (first + i * NT < v1)
#pragma unroll
                for (int j = 0; j < VEC; ++j) most = fmaxf(most, x[i].at(j));
        if (most > mine.m) {
            if (best_batch >= 0) second = mine.m;
            raise_max(mine, most);
            best_batch = b;
        } else {
            second = fmaxf(second, most);
        }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (first + i * NT < v1)
#pragma unroll
                for (int j = 0; j < VEC; ++j) add_logit(mine, x[i].at(j));
    }
    if (behind >= 0) {
        const float x = to_f32<T>(row[behind]);
        if (x > mine.m) raise_max(mine, x);
        add_logit(mine, x);
    }

    if (p.k > 0) {
        auto vectors = [&](int b, auto f) {
            const int first = v0 + b * U * NT + tid;
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (first + i * NT >= v1) break;
                const Pack<T> x = from[first + i * NT];
                const int id = lead + (first + i * NT) * VEC;
#pragma unroll
                for (int j = 0; j < VEC; ++j) f(key_of(x.at(j), id + j));
            }
        };
        auto every = [&](auto f) {
            if (ahead >= 0) f(key_of(to_f32<T>(row[ahead]), ahead));
            for (int b = 0; b < n_batches; ++b) vectors(b, f);
            if (behind >= 0) f(key_of(to_f32<T>(row[behind]), behind));
        };
        u64 best = 0;
        auto raise = [&](u64 key) { best = key > best ? key : best; };
        if (ahead >= 0) raise(key_of(to_f32<T>(row[ahead]), ahead));
        if (behind >= 0) raise(key_of(to_f32<T>(row[behind]), behind));
        if (best_batch >= 0) vectors(best_batch, raise);
        else if (n_batches > 0) vectors(0, raise);               // nothing but minus infinity: the first ids
        select_top<NT>(top, best, p.k, [&](u64 cut, auto f) {
            const bool one = best_batch >= 0 && key_of(second, 0) < cut;       // no other batch reaches the bound
            if (!one) { every(f); return; }
            if (ahead >= 0) f(key_of(to_f32<T>(row[ahead]), ahead));
            vectors(best_batch, f);
            if (behind >= 0) f(key_of(to_f32<T>(row[behind]), behind));
        });
    }
    Part all = block_join<NT>(mine, s_parts);
    if (CLUSTER) {
        if (tid == 0) s_mine = all;
        cluster_sync_all();
        if (part == 0) {
            if (tid < 32) {
                Part q = {-INFINITY, 0.0f, 0.0f};
                if (tid < parts) {
                    const uint32_t a = map_to_cta((uint32_t)__cvta_generic_to_shared(&s_mine), (uint32_t)tid);
                    q = {ld_cluster_f32(a), ld_cluster_f32(a + 4), ld_cluster_f32(a + 8)};
                }
                all = warp_join(q);
            }
            if (p.k > 0) {
                const uint32_t tops = (uint32_t)__cvta_generic_to_shared(top.top);
                auto key_at = [&](int i) {
                    u64 key;
                    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(key) : "r"(map_to_cta(tops, (uint32_t)(i / p.k)) + 8u * (uint32_t)(i % p.k)) : "memory");
                    return key;
                };
                // (at most 8 blocks of 128 keys; this block's own list is overwritten, so all are read first)
                constexpr int MOST = (8 * TOP_MAX + NT - 1) / NT;
                u64 mine_k[MOST], best = 0;
#pragma unroll
                for (int i = 0; i < MOST; ++i) {
                    const int j = tid + i * NT;
                    mine_k[i] = j < parts * p.k ? key_at(j) : 0;
                    best = mine_k[i] > best ? mine_k[i] : best;
                }
                select_top<NT>(top, best, p.k, [&](u64, auto f) {
#pragma unroll
                    for (int i = 0; i < MOST; ++i) if (mine_k[i]) f(mine_k[i]);
                });
            }
        }
        cluster_sync_all();                                      // nobody leaves while its memory is read
        if (part != 0) return;
    }
    if (tid == 0) {
        const float ln_s = logf(all.s);
        s_mine = {all.m, ln_s, 0.0f};
        p.logprob[r] = log_prob(all, ln_s, given);
        if (p.lse) p.lse[r] = fabsf(all.m) < INFINITY ? all.m + ln_s : all.m;
        if (p.entropy) p.entropy[r] = all.m == -INFINITY ? 0.0f : all.m == INFINITY ? __int_as_float(0x7fffffff) : ln_s - all.u / all.s;
    }
    if (p.k > 0) {
        __syncthreads();
        const Part q = {s_mine.m, 0.0f, 0.0f};
        for (int i = tid; i < p.k; i += NT) {
            const u64 key = top.top[i];
            p.top_ids[(size_t)r * p.k + i] = key ? key_id(key) : -1;
            p.top_logprobs[(size_t)r * p.k + i] = key ? log_prob(q, s_mine.s, key_logit(key)) : -INFINITY;
        }
    }
}

template <typename T, int NT>
static int launch_tokens(const TokenParams& p, int n, int parts, cudaStream_t stream) {
    if constexpr (NT == 512) {
        if (parts > 1) {
            airun_launch_clusters(token_logprobs_kernel<T, NT, true>, dim3(n * parts), dim3(NT), 0, stream, dim3(parts), p, parts);
            return airun_launch_status();
        }
    }
    airun_launch(token_logprobs_kernel<T, NT, false>, dim3(n), dim3(NT), 0, stream, p, 1);
    return airun_launch_status();
}

// logits: [held][V] rows ld elements apart; rows: [n] or null (then held >= n); tokens, logprob, entropy, lse: [n]; top_*: [n][k].
AIRUN_EXPORT int airun_token_logprobs(const void* logits, int dtype, long long ld, int held, int V, const int32_t* rows, const int32_t* tokens, int n,
                                      float* logprob, float* entropy, float* lse, int k, int32_t* top_ids, float* top_logprobs, int* err,
                                      cudaStream_t stream) {
    if (n < 0 || held < 0 || V <= 0 || ld < V || k < 0 || k > TOP_MAX || k > V || n > (1 << 27)) return AIRUN_ERR_ARG;
    if (n == 0) return AIRUN_OK;
    if (!logits || !tokens || !logprob || (k > 0 && (!top_ids || !top_logprobs)) || (!rows && n > held)) return AIRUN_ERR_ARG;
    const TokenParams p = {logits, ld, held, V, rows, tokens, logprob, entropy, lse, k, top_ids, top_logprobs, err};
    const int sms = airun_sm_count();
    // a block a row once there are rows for the SMs; below, rows in up to 8 parts of 4,096 logits and more
    int parts = 1;
    while (parts < 8 && 2 * parts * n <= 2 * sms && V / (2 * parts) >= 4096) parts *= 2;
    if (dtype == AIRUN_DT_F32) return V <= 2048 ? launch_tokens<float, 128>(p, n, 1, stream) : launch_tokens<float, 512>(p, n, parts, stream);
    if (dtype == AIRUN_DT_BF16) return V <= 2048 ? launch_tokens<__nv_bfloat16, 128>(p, n, 1, stream) : launch_tokens<__nv_bfloat16, 512>(p, n, parts, stream);
    return AIRUN_ERR_UNSUPPORTED;
}
