// Log probabilities of given tokens, with the entropy of their rows and the likeliest alternatives.
//
// A row of logits x (not a number counts as minus infinity):
//   m = max x,  s = sum exp(x - m),  u = sum exp(x - m) (x - m);
//   logprob = (x[token] - m) - ln s,  lse = m + ln s,  entropy = -sum p ln p = ln s - u / s,
// and the k largest logits, the first id first among equals, as (x - m) - ln s.  All three sums are kept over any part of a
// row in one pass, the maximum as it is so far; two parts join as
//   m = max(m1, m2),  d_i = m_i - m,  f_i = exp(d_i),  s = sum f_i s_i,  u = sum f_i (u_i + d_i s_i).
// A row with nothing above minus infinity has no distribution: its log probabilities are minus infinity, its entropy is 0.
// A row with plus infinity has entropy NaN and log probabilities x - inf.  A token outside the vocabulary has minus infinity.
//
// The reference takes the same numbers from whole rows on the host (crates/airun-core/src/sample.rs:128-140, :489-503).
#include "tcgen05.cuh"

typedef unsigned long long u64;

#define TOP_MAX 128

// ------------------------------------------------------------------ parts of a row
#define LOWEST (-200.0f)               // exp is 0 from here on, and so is a term's part in u

// A part's s without the 1 that its maximum stands for: where one token leads, s is 1 and a little, and each addition would round the little, and with it the
// entropy, to 2^-24 of the 1.  Entropies of single rows of 151,936 were off by 1.5e-7 in the mean square with s itself, 0.8e-7 now.
struct Part { float m, rest, u; };

__device__ __forceinline__ float exp_of(float d) {
    float e;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(d * 1.4426950408889634f));
    return e;
}
// x - m, bounded below: minus infinity, what is not a number and the difference of two equal infinities become terms of 0.
__device__ __forceinline__ float below(float x, float m) { return fmaxf(x - m, LOWEST); }

__device__ __forceinline__ Part join(const Part& a, const Part& b) {
    const float m = fmaxf(a.m, b.m), da = below(a.m, m), db = below(b.m, m), fa = exp_of(da), fb = exp_of(db);
    const float ra = fmaf(fa, a.rest, fa), rb = fmaf(fb, b.rest, fb);
    return {m, a.m >= b.m ? a.rest + rb : ra + b.rest, fa * a.u + da * ra + (fb * b.u + db * rb)};
}

// A part that grows, chunk by chunk.  A chunk's sums start at zero and join the others with what the additions before have rounded
// away (compensated summation, W. Kahan, Communications of the ACM 8, 1965): beside one leading token, 8,000 terms of 1e-6 added one by one
// are off by 3e-6, as much as the logits of a head of 4,096 values.  The maximum's 1 is in no running sum either, whether it comes early or late (an entropy from a
// second token of probability 3e-8 was off by 5 % where the leading one came later).
struct Run {
    float m = -INFINITY, rest = 0.0f, u = 0.0f, rest_lost = 0.0f, u_lost = 0.0f;
    __device__ __forceinline__ Part part() const { return {m, rest - rest_lost, u}; }
};

__device__ __forceinline__ void add_to(float& sum, float& lost, float x) {
    const float y = __fsub_rn(x, lost), t = __fadd_rn(sum, y);
    lost = __fsub_rn(__fsub_rn(t, sum), y);
    sum = t;
}

__device__ __forceinline__ u64 pair_of(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void of_pair(u64 r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ u64 add_pair(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ u64 fma_pair(u64 a, u64 b, u64 c) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ u64 mul_pair(u64 a, u64 b) {
    u64 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// What the chunk with the maximum adds up to is rounded to 2^-24 of its 1.  Where less than this is left of a whole row without the 1, the chunk is looked at
// again (others_again).  Log probabilities of 120 single rows of 151,936: off by 0.6e-7 in the mean square, with a look below 1/16 by 2.0e-7; a look takes 0.2 us.  Not so
// where logits are formed and used at once: to keep 32 of them until the row's end costs prompts 1 to 2 % and 700 capped rows 4 %.  There the 31 ids beside a leading one
// are added to its 1 in two chains of 16, so a log probability near 0 is off by 16 times 2^-24 at most, by 3e-7 where all 31 are 1e-7.
#define FEW_OTHERS 0.25f

// N logits, of which none is larger than `most`; true where they have brought the maximum.  Two at a time: additions and products take half the issue slots that way.
template <int N> __device__ __forceinline__ bool add_chunk(Run& r, const float (&x)[N], float most) {
    const bool moved = most > r.m;
    if (moved) {
        const float d = below(r.m, most), f = exp_of(d);
        r.u = f * fmaf(d, 1.0f + r.rest, r.u);
        r.u_lost = f * fmaf(d, r.rest_lost, r.u_lost);
        r.rest = fmaf(f, r.rest, f);
        r.rest_lost *= f;
        r.m = most;
    }
    const u64 minus_m = pair_of(-r.m, -r.m), log2_e = pair_of(1.4426950408889634f, 1.4426950408889634f);
    u64 s = 0, u = 0;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        float a, b, ea, eb;
        of_pair(add_pair(pair_of(x[i], x[i + 1]), minus_m), a, b);
        const u64 d = pair_of(fmaxf(a, LOWEST), fmaxf(b, LOWEST));
        of_pair(mul_pair(d, log2_e), a, b);
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(ea) : "f"(a));
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(eb) : "f"(b));
        const u64 e = pair_of(ea, eb);
        s = add_pair(s, e);
        u = fma_pair(e, d, u);
    }
    float a, b;
    of_pair(s, a, b);
    float sum = a + b;
    if (moved) sum -= 1.0f;
    add_to(r.rest, r.rest_lost, sum);
    of_pair(u, a, b);
    add_to(r.u, r.u_lost, a + b);
    return moved;
}

template <int N> __device__ __forceinline__ float most_of(const float (&x)[N]) {
    float most = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) most = fmaxf(most, x[i]);
    return most == most ? most : -INFINITY;                        // (all of them not numbers)
}

// `leader`: the first lane that has the maximum.
__device__ __forceinline__ Part warp_join(const Part& p, int& leader) {
    const float m = warp_max(p.m), d = below(p.m, m), f = exp_of(d), r = fmaf(f, p.rest, f);
    leader = __ffs(__ballot_sync(0xffffffffu, p.m == m)) - 1;
    return {m, warp_sum((int)(threadIdx.x & 31) == leader ? p.rest : r), warp_sum(fmaf(f, p.u, d * r))};
}
__device__ __forceinline__ Part warp_join(const Part& p) {
    int leader;
    return warp_join(p, leader);
}

// A whole row's part, by a converged warp: whether the chunk with its maximum is worth a second look, and that look, lane i with the chunk's i-th logit (minus infinity
// where there is none): what add_chunk has added up, in its order, goes, and the sum without the maximum comes.  (Two equal maxima are 1 and more, so there is one.)
__device__ __forceinline__ bool few_others(const Part& p) { return p.rest < FEW_OTHERS && fabsf(p.m) < INFINITY; }
template <int N> __device__ __forceinline__ Part others_again(const Part& p, float x) {
    const float e = exp_of(below(x, p.m));
    float a = 0.0f, b = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        a += __shfl_sync(0xffffffffu, e, i);
        b += __shfl_sync(0xffffffffu, e, i + 1);
    }
    return {p.m, (p.rest - ((a + b) - 1.0f)) + warp_sum(x < p.m ? e : 0.0f), p.u};
}

// The joined part of the block's threads, in its first warp.  `sh` holds one Part a warp.
template <int NT> __device__ __forceinline__ Part block_join(Part p, Part* sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    p = warp_join(p);
    __syncthreads();
    if (lane == 0) sh[warp] = p;
    __syncthreads();
    if (warp == 0) p = warp_join(lane < NT / 32 ? sh[lane] : Part{-INFINITY, 0.0f, 0.0f});
    return p;
}

// The same of the parts of a row's batches (the kernel on logits), with the thread that has the maximum, and the batch that has brought it.
struct Place { int thread, batch; };
struct ThreadPart { Part p; Place at; };
template <int NT> __device__ __forceinline__ Part block_join(const Run& r, int batch, ThreadPart* sh, Place& at) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int leader;
    Part p = warp_join(r.part(), leader);
    __syncthreads();
    if (lane == leader) sh[warp] = {p, {(int)threadIdx.x, batch}};
    __syncthreads();
    if (warp == 0) {
        ThreadPart mine = {{-INFINITY, 0.0f, 0.0f}, {0, 0}};
        if (lane < NT / 32) mine = sh[lane];
        p = warp_join(mine.p, leader);
        at = {__shfl_sync(0xffffffffu, mine.at.thread, leader), __shfl_sync(0xffffffffu, mine.at.batch, leader)};
    }
    return p;
}

// What is left of a whole row's part: the maximum, ln sum exp(x - m), the entropy.
struct Row { float m, ln_s, entropy; };
__device__ __forceinline__ Row row_of(const Part& p) {
    if (p.m == -INFINITY) return {p.m, -INFINITY, 0.0f};
    if (p.m == INFINITY) return {p.m, 0.0f, __int_as_float(0x7fffffff)};
    const float ln_s = log1pf(p.rest);
    return {p.m, ln_s, ln_s - p.u / (1.0f + p.rest)};
}
__device__ __forceinline__ float log_prob(const Row& r, float x) {
    return x > -INFINITY && r.m > -INFINITY ? (x - r.m) - r.ln_s : -INFINITY;
}
__device__ __forceinline__ float row_lse(const Row& r) { return fabsf(r.m) < INFINITY ? r.m + r.ln_s : r.m; }

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
    u64 joined[NT >= 256 ? 8 * TOP_MAX : 1];                  // a cluster's lists
    u64 cut;
    int count;
};

// The k largest of the list's n keys, in order, in sh.top (0 beyond the last): each counts the larger ones.
template <int NT> __device__ __forceinline__ void rank_top(TopShared<NT>& sh, int n, int k) {
    const int tid = threadIdx.x;
    for (int i = tid; i < k; i += NT) if (i >= n) sh.top[i] = 0;
    for (int i = tid; i < n; i += NT) {
        const u64 mine = sh.list[i];
        int larger = 0;
#pragma unroll 4
        for (int j = 0; j < n; ++j) larger += sh.list[j] > mine || (sh.list[j] == mine && j < i);
        if (larger < k) sh.top[larger] = mine;
    }
    __syncthreads();
}

// The k largest of all threads' keys, in order, in sh.top; false where more keys than the list holds reach the bound that is found for them.  The
// threads' keys are all different.  `low` and `high` are bounds of a thread's largest key (0: it has none), the same where it is known, and
// each(f) calls f on every key of the thread that can be as large as `cut`.
// The k-th largest of the maxima of groups of threads is a lower bound of the k-th largest of all, and close to it when
// there are twice as many groups as wanted keys: about k to 2 k keys reach it.  Those are listed and each counts the larger ones.
// A group is as many lanes as leave 2 k groups, and fewer where logits may come `VEC` neighbours to a thread: equal logits in every place, whose keys
// fall with the id, list the first vectors of k groups, 1,024 keys or those of k threads.  A list longer than `few` is cut again in the same way.
template <int NT, int VEC, typename Each>
__device__ __forceinline__ bool select_top(TopShared<NT>& sh, u64 low, u64 high, int k, Each each) {
    constexpr int CAP = TopShared<NT>::CAP, MINE = CAP / NT;
    const int tid = threadIdx.x;
    int g = 32;
    while (g > 1 && (NT / g < 2 * k || k * g * VEC > 1024)) g >>= 1;
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
    u64 cut = find_cut(low);
    if (high >= cut) each(cut, [&](u64 key) { if (key >= cut) push(key); });
    __syncthreads();
    int n = sh.count;
    if (n > CAP) return false;
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
    rank_top(sh, n, k);
    return true;
}

// The same one after the other, for what select_top refuses: large logits that repeat at the threads' stride.
template <int NT, typename Each>
__device__ __forceinline__ void one_by_one(TopShared<NT>& sh, int k, Each each) {
    const int tid = threadIdx.x;
    u64 below = ~0ull;
    __syncthreads();
    for (int i = tid; i < k; i += NT) sh.top[i] = 0;
    for (int i = 0; i < k; ++i) {
        u64 b = 0;
        each(1ull, [&](u64 key) { if (key < below && key > b) b = key; });
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
        if (b == 0) break;                                       // (the same for all threads)
    }
    __syncthreads();
}
// The least logit that reaches a bound.
__device__ __forceinline__ float cut_logit(u64 cut) { return cut <= 1ull ? -INFINITY : key_logit(cut); }

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
    __device__ __forceinline__ void nothing() { v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }
    __device__ __forceinline__ float at(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
};
template <> struct Pack<__nv_bfloat16> {
    static constexpr int N = 8;
    uint4 v;
    __device__ __forceinline__ void nothing() { v = make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u); }      // minus infinities
    __device__ __forceinline__ float at(int i) const {
        const unsigned w = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
        return __uint_as_float((i & 1) ? (w & 0xFFFF0000u) : (w << 16));
    }
};

// Where the vectors of a row lie: the elements ahead of the first, and their number.
template <typename T> struct Vectors {
    int lead, n;
    __device__ __forceinline__ Vectors(const T* row, int V)
        : lead(min(V, (int)((16 - ((uintptr_t)row & 15)) % 16 / sizeof(T)))), n((V - lead) / Pack<T>::N) {}
};
// The i-th logit of a batch (-1: of the elements ahead of the vectors and behind them); minus infinity where there is none.  All of it is worked
// out again: kept in registers until here it costs the loop over the row some of its own.
template <typename T, int NT, int U> __device__ __forceinline__ float logit_at(const TokenParams& p, int r, int part, int parts, Place at, int i) {
    constexpr int VEC = Pack<T>::N;
    const T* row = (const T*)p.logits + (size_t)(p.rows ? p.rows[r] : r) * p.ld;
    const Vectors<T> vecs(row, p.V);
    int id = -1;
    if (at.batch < 0) {
        const int behind = vecs.lead + vecs.n * VEC + at.thread;
        if (i == 0 && part == 0 && at.thread < vecs.lead) id = at.thread;
        if (i == 1 && part == parts - 1 && behind < p.V) id = behind;
    } else if (i < U * VEC) {
        const int v = at.batch + i / VEC * NT;
        if (v < (int)((long long)vecs.n * (part + 1) / parts)) id = vecs.lead + v * VEC + i % VEC;
    }
    return id >= 0 ? to_f32<T>(row[id]) : -INFINITY;
}

// A cluster of C blocks a row (C = 1: a block).  The row's 16-byte vectors are dealt to the blocks in turn ranges and, inside, to
// the threads in batches of U: a thread's elements come by ascending id.  The few elements ahead of the first
// 16-byte boundary and behind the last belong to the first block's first threads and the last block's first threads.
// What reaches the bound of the k largest is read again: by few threads, and with C = 1 while the SM's other blocks stream.  TOP: alternatives are wanted.
// Blocks an SM: three of 512 threads where rows are many, so that some stream while others select (2,048 rows with 20 alternatives 257 us with two, 227); 16
// logits a batch (bfloat16 in batches of 32 leaves room for two: 333 rows of 50,001 22.8 us, 19.5).
template <typename T, int NT, bool CLUSTER, bool TOP>
__global__ __launch_bounds__(NT, NT == 128 ? 8 : CLUSTER ? 2 : 3) void token_logprobs_kernel(const TokenParams p, int n_parts) {
    pdl_trigger();
    constexpr int VEC = Pack<T>::N, U = 16 / VEC;
    __shared__ TopShared<NT> top;
    __shared__ ThreadPart s_parts[NT / 32];
    __shared__ ThreadPart s_part_of[8];                          // of the cluster's blocks, in the first one's memory
    __shared__ Row s_row;
    const int tid = threadIdx.x;
    const int part = CLUSTER ? (int)cluster_rank() : 0, parts = CLUSTER ? n_parts : 1;
    const int r = CLUSTER ? blockIdx.x / parts : blockIdx.x;
    if (CLUSTER) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    pdl_wait();
    const int at = p.rows ? p.rows[r] : r;
    const int token = p.tokens[r];
    const bool there = at >= 0 && at < p.held;
    if (!there && tid == 0 && part == 0 && p.err) atomicOr(p.err, AIRUN_DEV_BAD_ROW);
    const int V = there ? p.V : 0;
    const T* row = (const T*)p.logits + (size_t)(there ? at : 0) * p.ld;
    const float given = part == 0 && token >= 0 && token < V ? to_f32<T>(row[token]) : -INFINITY;

    const Vectors<T> place_of(row, V);
    const int lead = place_of.lead, vecs = place_of.n, tail = lead + vecs * VEC;
    const int v0 = (int)((long long)vecs * part / parts) + tid, v1 = (int)((long long)vecs * (part + 1) / parts);      // this thread's first; the block's end
    const Pack<T>* from = reinterpret_cast<const Pack<T>*>(row + lead);
    // the element ahead of the vectors that is this thread's, and the one behind them
    const int ahead = part == 0 && tid < lead ? tid : -1, behind = part == parts - 1 && tid < V - tail ? tail + tid : -1;

    Run mine;
    float x[U * VEC];                                            // a batch, named by its first vector
    auto load = [&](int v) {
        Pack<T> in[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (v + i * NT < v1) in[i] = from[v + i * NT];
            else in[i].nothing();
        }
#pragma unroll
        for (int i = 0; i < U * VEC; ++i) x[i] = in[i / VEC].at(i % VEC);
    };
    auto id_of = [&](int v, int i) { return lead + (v + i / VEC * NT) * VEC + i % VEC; };
    float second = -INFINITY;                                    // largest of the batches but the one with the maximum
    int best = -1;                                               // that one
    const float one_ahead = ahead >= 0 ? to_f32<T>(row[ahead]) : -INFINITY, one_behind = behind >= 0 ? to_f32<T>(row[behind]) : -INFINITY;
    for (int v = v0; v < v1; v += U * NT) {
        load(v);
        const float most = most_of(x);
        if (most > mine.m) {
            if (best >= 0) second = mine.m;
            best = v;
        } else {
            second = fmaxf(second, most);
        }
        add_chunk(mine, x, most);
    }
    const float most = mine.m;                                   // of the vectors
    int brought = best;                                          // the batch that has brought the maximum; -1: the elements ahead of the vectors and behind them
    if (ahead >= 0 || behind >= 0) {
        const float ends[2] = {one_ahead, one_behind};
        if (add_chunk(mine, ends, most_of(ends))) brought = -1;
    }

    if constexpr (TOP) {
        u64 end_best = 0;
        if (ahead >= 0) end_best = key_of(one_ahead, ahead);
        if (behind >= 0) end_best = max(end_best, key_of(one_behind, behind));
        auto ends = [&](auto f) {
            if (ahead >= 0) f(key_of(one_ahead, ahead));
            if (behind >= 0) f(key_of(one_behind, behind));
        };
        // the keys of the batch in x that can reach the bound
        auto batch = [&](int v, u64 cut, auto f) {
            const float least = cut_logit(cut);
#pragma unroll
            for (int i = 0; i < U * VEC; ++i)
                if (!(x[i] < least) && v + i / VEC * NT < v1) f(key_of(x[i], id_of(v, i)));
        };
        auto each = [&](u64 cut, auto f) {
            ends(f);
            if (best >= 0 && key_of(second, 0) < cut) {          // no other batch reaches the bound
                load(best);
                batch(best, cut, f);
                return;
            }
            for (int v = v0; v < v1; v += U * NT) {
                if (best < 0 && key_of(-INFINITY, id_of(v, 0)) < cut) break;              // (equal ones go on falling with their ids)
                load(v);
                batch(v, cut, f);
            }
        };
        // The largest of the vectors lies somewhere in its batch: from the first to the last id of it, unless there is nothing but minus infinity.
        u64 low = end_best, high = end_best;
        const int likely = best < 0 ? v0 : best;
        if (v0 < v1) {
            high = max(high, key_of(most, id_of(likely, 0)));
            low = max(low, key_of(most, best < 0 ? id_of(v0, 0) : id_of(best, U * VEC - 1)));
        }
        if (!select_top<NT, VEC>(top, low, high, p.k, each)) {
            // many equal ones: with the places of the maxima, the first ids are told from the others
            u64 key_best = end_best;
            if (v0 < v1) {
                load(likely);
                batch(likely, key_of(most, 0x7fffffff), [&](u64 key) { key_best = max(key_best, key); });
            }
            if (!select_top<NT, VEC>(top, key_best, key_best, p.k, each)) one_by_one<NT>(top, p.k, each);
        }
    }
    Place place;
    Part all = block_join<NT>(mine, brought, s_parts, place);
    int owner = part;                                            // the block with the maximum
    if (CLUSTER) {
        // every block stores its part and its list into the first one's memory, and all but that one may leave
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");         // every block runs: its memory may be written
        if (tid == 0) {
            const uint32_t to = map_to_cta((uint32_t)__cvta_generic_to_shared(&s_part_of[part]), 0);
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(all.m) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4), "f"(all.rest) : "memory");
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 8), "f"(all.u) : "memory");
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 12), "r"(place.thread) : "memory");
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(to + 16), "r"(place.batch) : "memory");
        }
        if constexpr (TOP) {
            const uint32_t to = map_to_cta((uint32_t)__cvta_generic_to_shared(top.joined) + 8u * (uint32_t)(part * p.k), 0);
            for (int i = tid; i < p.k; i += NT) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to + 8u * (uint32_t)i), "l"(top.top[i]) : "memory");
        }
        cluster_sync_all();
        if (part != 0) return;
        if (tid < 32) {
            all = warp_join(tid < parts ? s_part_of[tid].p : Part{-INFINITY, 0.0f, 0.0f}, owner);
            place = s_part_of[owner].at;
        }
    }
    if (tid < 32 && few_others(all)) all = others_again<U * VEC>(all, logit_at<T, NT, U>(p, r, owner, parts, place, tid));
    if (tid == 0) {
        const Row w = row_of(all);
        s_row = w;
        p.logprob[r] = log_prob(w, given);
        if (p.lse) p.lse[r] = row_lse(w);
        if (p.entropy) p.entropy[r] = w.entropy;
    }
    if constexpr (TOP) {
        __syncthreads();
        const Row w = s_row;
        if (CLUSTER) {
            // 8 lists of 128 at the most: each key counts the larger ones
            const int n_keys = parts * p.k;
            for (int i = tid; i < n_keys; i += NT) {
                const u64 mine_k = top.joined[i];
                int larger = 0;
#pragma unroll 8
                for (int j = 0; j < n_keys; ++j) larger += top.joined[j] > mine_k || (top.joined[j] == mine_k && j < i);
                if (larger < p.k) top.top[larger] = mine_k;
            }
            __syncthreads();
        }
        for (int i = tid; i < p.k; i += NT) {
            const u64 key = top.top[i];
            p.top_ids[(size_t)r * p.k + i] = key ? key_id(key) : -1;
            p.top_logprobs[(size_t)r * p.k + i] = key ? log_prob(w, key_logit(key)) : -INFINITY;
        }
    }
}

template <typename T, int NT, bool TOP>
static int launch_tokens(const TokenParams& p, int n, int parts, cudaStream_t stream) {
    if constexpr (NT == 512) {
        if (parts > 1) {
            airun_launch_clusters(token_logprobs_kernel<T, NT, true, TOP>, dim3(n * parts), dim3(NT), 0, stream, dim3(parts), p, parts);
            return airun_launch_status();
        }
    }
    airun_launch(token_logprobs_kernel<T, NT, false, TOP>, dim3(n), dim3(NT), 0, stream, p, 1);
    return airun_launch_status();
}

template <typename T>
static int launch_tokens(const TokenParams& p, int n, cudaStream_t stream) {
    if (p.V <= 2048) return p.k > 0 ? launch_tokens<T, 128, true>(p, n, 1, stream) : launch_tokens<T, 128, false>(p, n, 1, stream);
    // A block a row once there are rows for the SMs; below, rows in up to 8 parts of 4,096 logits and more, as long as all blocks run at once.  Five
    // alternatives of 151,936 logits, us, one, two, four and eight parts: 20 rows 18.0, 10.3, 11.6, 9.9; 60 rows 33, 22, 15, 20; 148 rows 36, 26, 33, 44;
    // 295 rows 49, 44, 56, 83; of 32,000 logits, 20 rows 7.1, 6.5, 6.8, 7.1; 200 rows 11, 14, 20, 39.
    const int sms = airun_sm_count();
    int parts = 1;
    while (parts < 8 && 2 * parts * n <= 2 * sms && p.V / (2 * parts) >= 4096) parts *= 2;
    return p.k > 0 ? launch_tokens<T, 512, true>(p, n, parts, stream) : launch_tokens<T, 512, false>(p, n, parts, stream);
}

// logits: [held][V] rows ld elements apart; rows: [n] or null (then held >= n); tokens, logprob, entropy, lse: [n]; top_*: [n][k].
AIRUN_EXPORT int airun_token_logprobs(const void* logits, int dtype, long long ld, int held, int V, const int32_t* rows, const int32_t* tokens, int n,
                                      float* logprob, float* entropy, float* lse, int k, int32_t* top_ids, float* top_logprobs, int* err,
                                      cudaStream_t stream) {
    if (n < 0 || held < 0 || V <= 0 || ld < V || k < 0 || k > TOP_MAX || k > V || n > (1 << 27) || V > 0x7fff0000) return AIRUN_ERR_ARG;
    if (n == 0) return AIRUN_OK;
    if (!logits || !tokens || !logprob || (k > 0 && (!top_ids || !top_logprobs)) || (!rows && n > held)) return AIRUN_ERR_ARG;
    const TokenParams p = {logits, ld, held, V, rows, tokens, logprob, entropy, lse, k, top_ids, top_logprobs, err};
    if (dtype == AIRUN_DT_F32) return launch_tokens<float>(p, n, stream);
    if (dtype == AIRUN_DT_BF16) return launch_tokens<__nv_bfloat16>(p, n, stream);
    return AIRUN_ERR_UNSUPPORTED;
}

// ------------------------------------------------------------------ from hidden states
// The logits of a row are its product with the head's weight [V][K].  They are formed in tensor memory, a tile of rows x `bn` ids at a
// time, and every thread of the epilogue keeps the three sums, the given token's logit and a list of the k largest for one row:
// its lane of tensor memory is that row, its ids those of half of the tiles' columns.  The vocabulary is cut into `splits` ranges of
// `tiles` tiles; a block (a pair) walks the tiles of one range for one block of rows, then the parts of each row are joined by
// head_join_kernel.  Neither logits nor anything of their size is written.
//   PAIR   : two SMs to 256 rows, tcgen05.mma.cta_group::2 with M = 256; each brings 128 rows and half of the ids, 32 KB a K-step of 64
//            values, which is what 512 clocks of products leave time for.  What prompts run on.
//   !PAIR  : an SM to 128 rows, of which only `x_rows` are brought (what the products read behind them ends in lanes nobody looks at): up
//            to 128 rows are bound by the weights' bytes.  (Up to 32 rows head_few_kernel takes.)
//   warp 0    : TMA loads into a ring of stages; asks for weights, which no kernel writes, ahead of the wait for the kernel in front;
//   warp 1    : allocates tensor memory, issues the products (in a pair, the leader's);
//   warps 4-11: epilogue, two warps a quadrant of lanes, every other 32 ids of a tile; they take the registers of the first four.
// The tensor cores cut a running sum off where float32 rounds, so its error grows with the products in it.  A buffer of tensor memory holds
// `part` K-steps; the epilogue adds the parts up in registers, rounded, 128 sums a thread, while the other buffer fills.
#define HEAD_THREADS 384
#define HEAD_TOP 16                                                // longest list
#define HEAD_SMEM 230400                                           // stages and 1 KB to align them
#define HEAD_STAGES 12                                             // at most
#define HEAD_REGS 168                                              // a thread at launch: 384 x 168 = 128 x 40 + 256 x 232
#define BK 64

struct HeadParams {
    int n, V, K;
    int row_blocks, splits, tiles, bn, part;
    int x_rows, stages;                                            // rows a stage brings; stages
    const int32_t* tokens;
    float scale, cap;
    int k;
    float* stats;                                                  // [3][2 splits][n]: a part's m, s - 1, u
    float* given;                                                  // [n] logits of the given tokens
    u64* keys;                                                     // [n][2 splits][k]
    int* err;
};

// A thread's k <= N largest logits with their ids: the largest first, equal ones in the order they come, which is that of their ids.  In registers: while
// products read their operands from shared memory, a load from there takes hundreds of clocks (a logit put into a list there took 1,900).
template <int N> struct TopList {
    float x[N];
    int id[N];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < N; ++i) { x[i] = -INFINITY; id[i] = -1; }
    }
    __device__ __forceinline__ void put(float v, int at) {
#pragma unroll
        for (int i = N - 1; i >= 0; --i) {
            const bool here = v > x[i], before = i > 0 && v > x[i > 0 ? i - 1 : 0];
            x[i] = before ? x[i > 0 ? i - 1 : 0] : here ? v : x[i];
            id[i] = before ? id[i > 0 ? i - 1 : 0] : here ? at : id[i];
        }
    }
    __device__ __forceinline__ float least(int k) const {
        float v = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) v = k > i ? x[i] : v;
        return v;
    }
};
template <> struct TopList<0> {};

// cap * tanh(x / cap).  tanh z = 1 - 2 / (e^2z + 1), where the exponential is off by 2^-22 of itself and the reciprocal by 2^-23: 2^-21 of the cap at most, 4.3 times
// 2^-24 in 2.6 million logits; below 1/4, where that would be many units, the odd series to z^9 (the next term is below 3e-9).  A logit near 7 under a cap of 30 is off by
// 6e-7 so, by what its product is off by too.  700 rows x [20000, 1024] take 37 us with it, 39 with tanhf; 2,048 x [20000, 512] 59 and 65.
__device__ __forceinline__ float capped(float x, float cap, float over_cap) {
    const float z = x * over_cap, q = z * z;
    const float near = fmaf(z * q, fmaf(q, fmaf(q, fmaf(q, 62.0f / 2835.0f, -17.0f / 315.0f), 2.0f / 15.0f), -1.0f / 3.0f), z);
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * (2.0f * 1.4426950408889634f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
    return cap * (fabsf(z) < 0.25f ? near : fmaf(-2.0f, r, 1.0f));
}

// ROLLED: the epilogue's code, which runs once a tile and comes cold, is a quarter as long.  Unrolled it saves the moves, which only pays where tiles follow each
// other fast: us, rolled and not, 2,048 rows x [151936, 2048] 950, 924, with five alternatives 996, 979; 64 rows x [151936, 4096] with five 215, 224; 100 rows x
// [151936, 2048] with five 117, 125; capped, 700 rows x [20000, 1024] 37, 40, with five 57, 67.
template <bool PAIR, int TOP, bool ROLLED>
__global__ __launch_bounds__(HEAD_THREADS, 1) void head_logprobs_kernel(
    const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const HeadParams p) {
    constexpr int CTAS = PAIR ? 2 : 1;
    __shared__ __align__(8) uint64_t bars[2 * HEAD_STAGES + 4];    // full (a pair: the leader's), empty of the stages; full, empty (the leader's) of the sums
    __shared__ uint32_t tmem_slot;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int rank = PAIR ? (int)cluster_rank() : 0, group = PAIR ? blockIdx.x >> 1 : blockIdx.x, groups = PAIR ? gridDim.x >> 1 : gridDim.x;
    const int kb_total = (p.K + BK - 1) / BK, units = p.row_blocks * p.splits, range = p.tiles * p.bn;
    const int w_rows = p.bn / CTAS, w_bytes = w_rows * (BK * 2), x_bytes = p.x_rows * (BK * 2), stages = p.stages;
    // the stages' weights, then their rows
    const uint32_t w_at = smem_u32(smem), x_at = w_at + stages * w_bytes;
    const uint32_t full = smem_u32(bars), empty = full + 8 * HEAD_STAGES, accf = empty + 8 * HEAD_STAGES, acce = accf + 16;
    if (threadIdx.x == 0) {
        for (int s = 0; s < HEAD_STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(accf + 8 * b, 1); mbar_init(acce + 8 * b, 8 * CTAS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            tmem_alloc(smem_u32(&tmem_slot), 512);
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();                        // the leader's barriers are there before anything arrives at them
    pdl_trigger();                                                 // (not sooner: a kernel behind could take the tensor memory and wait for this one)
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const uint32_t full_lead = PAIR ? map_to_cta(full, 0) : full, acce_lead = PAIR ? map_to_cta(acce, 0) : acce;

    struct Unit { int x0, w0, w_end; };                            // first row of this CTA; ids
    auto unit_of = [&](int u) {
        const int w0 = u / p.row_blocks * range;
        return Unit{u % p.row_blocks * (128 * CTAS) + rank * 128, w0, min(p.V, w0 + range)};
    };
    const uint32_t bytes = CTAS * (x_bytes + w_bytes);
    auto load = [&](const CUtensorMap* map, uint32_t dst, uint32_t bar, int x, int y) {
        if constexpr (PAIR) tma_load_2d_pair(dst, map, bar, x, y);
        else tma_load_2d(dst, map, bar, x, y);
    };
    const int first_n = group < units ? min(kb_total, stages) : 0;
    if (warp == 0 && elect_one()) {
        for (int i = 0; i < first_n; ++i) {
            if (rank == 0) mbar_expect_tx(full + 8 * i, bytes);
            load(&map_w, w_at + i * w_bytes, full_lead + 8 * i, i * BK, unit_of(group).w0 + rank * w_rows);
        }
    }
    pdl_wait();

    bool ok = true;
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        int it = 0, s = 0;                                         // K-steps so far, and their place in the ring
        uint32_t phase = 0;                                        // of the ring's barriers, one round after the other
        if (warp == 0) {
            for (int u = group; u < units && ok; u += groups) {
                const Unit t = unit_of(u);
                for (int w0 = t.w0; w0 < t.w_end && ok; w0 += p.bn) {
                    for (int kb = 0; kb < kb_total; ++kb, ++it) {
                        if (it >= first_n && !mbar_wait_warp(empty + 8 * s, phase ^ 1)) { ok = false; break; }
                        const uint32_t bar = full_lead + 8 * s;
                        if (elect_one()) {
                            if (it >= first_n) {
                                if (rank == 0) mbar_expect_tx(full + 8 * s, bytes);
                                load(&map_w, w_at + s * w_bytes, bar, kb * BK, w0 + rank * w_rows);
                            }
                            load(&map_x, x_at + s * x_bytes, bar, kb * BK, t.x0);
                        }
                        __syncwarp();
                        if (++s == stages) { s = 0; phase ^= 1; }
                    }
                }
            }
            // the last commits arrive at this CTA's barriers before it may leave
            for (int i = max(0, it - stages); i < it && ok; ++i)
                ok = mbar_wait_warp(empty + 8 * (i % stages), (i / stages) & 1);
            if (!ok) {
                atomicOr(p.err, AIRUN_DEV_TIMEOUT);
                // what is on its way lands before the memory is given up (a pair's loads all tell the leader, and both leave together)
                for (int i = max(0, it - stages); i < it && rank == 0; ++i)
                    if (!mbar_wait_warp(full + 8 * (i % stages), (i / stages) & 1)) break;
            }
        } else if (warp == 1 && rank == 0) {
            const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(p.bn >> 3) << 17) | ((uint32_t)(128 * CTAS >> 4) << 24);
            int n = 0;                                             // sums so far
            auto sum_up = [&](int first, int end) {
                const int buf = n & 1;
                if (!mbar_wait_warp(acce + 8 * buf, ((n >> 1) & 1) ^ 1)) { ok = false; return; }
                tc_fence_after();
                for (int kb = first; kb < end; ++kb) {
                    if (!mbar_wait_warp(full + 8 * s, phase)) { ok = false; return; }
                    tc_fence_after();
                    const uint64_t da = smem_desc_sw128(x_at + s * x_bytes), db = smem_desc_sw128(w_at + s * w_bytes);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < BK / 16; ++k) {
                            const uint32_t more = (kb > first || k > 0) ? 1u : 0u;
                            if constexpr (PAIR) umma_bf16_pair(tmem + buf * 256, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, more);
                            else umma_bf16(tmem + buf * 256, da + (uint64_t)(k * 2), db + (uint64_t)(k * 2), idesc, more);
                        }
                        if constexpr (PAIR) {
                            umma_commit_pair(empty + 8 * s);
                            if (kb + 1 == end) umma_commit_pair(accf + 8 * buf);
                        } else {
                            umma_commit(empty + 8 * s);
                            if (kb + 1 == end) umma_commit(accf + 8 * buf);
                        }
                    }
                    __syncwarp();
                    if (++s == stages) { s = 0; phase ^= 1; }
                }
                ++n;
            };
            for (int u = group; u < units && ok; u += groups) {
                const Unit t = unit_of(u);
                for (int w0 = t.w0; w0 < t.w_end && ok; w0 += p.bn)
                    for (int first = 0; first < kb_total && ok; first += p.part) sum_up(first, min(first + p.part, kb_total));
            }
            if (!ok) atomicOr(p.err, AIRUN_DEV_TIMEOUT);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int quad = warp & 3, half = (warp - 4) >> 2;
        const float over_cap = 1.0f / p.cap;
        int n = 0;                                                 // sums so far
        for (int u = group; u < units && ok; u += groups) {
            const Unit t = unit_of(u);
            const int row = t.x0 + quad * 32 + lane;
            const bool row_on = row < p.n, warp_on = t.x0 + quad * 32 < p.n;
            const int token = row_on ? p.tokens[row] : -1;
            Run mine;
            [[maybe_unused]] TopList<TOP> list;
            [[maybe_unused]] float least = row_on ? -INFINITY : INFINITY;        // of the list
            if constexpr (TOP > 0) list.clear();
            for (int w0 = t.w0; w0 < t.w_end && ok; w0 += p.bn) {
                float acc[4][32];                                  // ids 32 half + 64 j and 31 more
                for (int kb = 0; kb < kb_total; kb += p.part, ++n) {
                    const int buf = n & 1;
                    ok = mbar_wait_warp(accf + 8 * buf, (n >> 1) & 1);
                    if (!ok) { atomicOr(p.err, AIRUN_DEV_TIMEOUT); break; }
                    tc_fence_after();
                    __syncwarp();
                    if (warp_on) {
                        // (a load takes 1,100 clocks while products run, four at once 1,900, so as many as registers are free for are on their
                        // way together.  What lies beyond the tile's ids, but inside the buffer, is read and not looked at.)
                        const uint32_t lanes = tmem + buf * 256 + ((uint32_t)(quad * 32) << 16) + 32 * half;
                        if (kb == 0) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) tmem_ld32_async(lanes + 64 * j, reinterpret_cast<uint32_t*>(acc[j]));
#pragma unroll
                            for (int j = 0; j < 4; ++j) tmem_wait32(reinterpret_cast<uint32_t*>(acc[j]));
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; j += 2) {
                                uint32_t a[32], b[32];
                                tmem_ld32_async(lanes + 64 * j, a);
                                tmem_ld32_async(lanes + 64 * j + 64, b);
                                tmem_wait32(a);
                                tmem_wait32(b);
#pragma unroll
                                for (int i = 0; i < 32; ++i) {
                                    acc[j][i] += __uint_as_float(a[i]);
                                    acc[j + 1][i] += __uint_as_float(b[i]);
                                }
                            }
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if constexpr (PAIR) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(acce_lead + 8 * buf) : "memory");
                        else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(acce + 8 * buf) : "memory");
                    }
                }
                if (!ok) break;
                if (!warp_on) continue;
                const int ids = min(p.bn, t.w_end - w0);           // of this tile
                // ROLLED: one body, and the next ids are moved up in the registers
#pragma unroll ROLLED ? 1 : 4
                for (int j = 0; j < 4; ++j) {
                    const int c = 32 * half + 64 * j, first = w0 + c;
                    if (c >= ids) break;
                    float (&v)[32] = acc[ROLLED ? 0 : j];
                    if (c + 32 > ids) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = c + i < ids ? v[i] : __int_as_float(0x7fffffff);       // no number: nowhere counted
                    }
                    if (p.scale != 1.0f) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] *= p.scale;
                    }
                    if (p.cap > 0.0f) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = capped(v[i], p.cap, over_cap);
                    }
                    if (token >= first && token < min(first + 32, w0 + ids)) {      // (a tile may end inside the 32, and the next one begins there)
                        float x = v[0];
#pragma unroll
                        for (int i = 1; i < 32; ++i) x = token == first + i ? v[i] : x;
                        p.given[row] = x;
                    }
                    const float most = most_of(v);
                    add_chunk(mine, v, most);
                    if constexpr (TOP > 0) {
                        if (__any_sync(0xffffffffu, most > least)) {
                            // every lane puts its next one into its list, until none has any
                            uint32_t larger = 0;
#pragma unroll
                            for (int i = 0; i < 32; ++i) larger |= v[i] > least ? 1u << i : 0u;
                            while (__any_sync(0xffffffffu, larger != 0)) {
                                const int i = larger ? __ffs(larger) - 1 : 0;
                                float x[16];
#pragma unroll
                                for (int a = 0; a < 16; ++a) x[a] = i & 1 ? v[2 * a + 1] : v[2 * a];
#pragma unroll
                                for (int b = 1; b < 5; ++b)
#pragma unroll
                                    for (int a = 0; a < (16 >> b); ++a) x[a] = (i >> b) & 1 ? x[2 * a + 1] : x[2 * a];
                                list.put(larger ? x[0] : -INFINITY, first + i);
                                larger &= larger - 1;
                            }
                            least = row_on ? list.least(p.k) : INFINITY;
                        }
                    }
                    if constexpr (ROLLED) {
#pragma unroll
                        for (int a = 0; a < 3; ++a)
#pragma unroll
                            for (int i = 0; i < 32; ++i) acc[a][i] = acc[a + 1][i];
                    }
                }
            }
            if (row_on) {
                const int parts = 2 * p.splits, part = 2 * (u / p.row_blocks) + half;
                float* to = p.stats + (size_t)part * p.n + row;
                const Part all = mine.part();
                to[0] = all.m;
                to[(size_t)parts * p.n] = all.rest;
                to[(size_t)2 * parts * p.n] = all.u;
                if constexpr (TOP > 0) {
                    u64* keys = p.keys + ((size_t)row * parts + part) * p.k;
#pragma unroll
                    for (int i = 0; i < TOP; ++i) if (i < p.k) keys[i] = list.id[i] < 0 ? 0 : key_of(list.x[i], list.id[i]);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();                        // neither CTA leaves, or frees, while the other works on both
    if (warp == 1) {
        tc_fence_after();
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
        else tmem_dealloc(tmem, 512);
    }
}

// The parts of a row become its results.  Without alternatives by warps.
__device__ __forceinline__ Part part_at(const float* stats, int i, int parts, int n, int r) {
    const float* at = stats + (size_t)i * n + r;
    return {at[0], at[(size_t)parts * n], at[(size_t)2 * parts * n]};
}
__device__ __forceinline__ Row write_row(const Part& all, const float* given, int token, int V, int r, float* logprob, float* entropy, float* lse) {
    const Row w = row_of(all);
    logprob[r] = token >= 0 && token < V ? log_prob(w, given[r]) : -INFINITY;
    if (lse) lse[r] = row_lse(w);
    if (entropy) entropy[r] = w.entropy;
    return w;
}

template <int ROWS>                                                // of a block of 128 threads: 4, or 1 where rows are few and have many parts
__global__ __launch_bounds__(128) void head_rows_kernel(
    const float* stats, const float* given, const int32_t* tokens, int n, int V, int parts, float* logprob, float* entropy, float* lse) {
    pdl_trigger();
    __shared__ Part s_parts[4];
    constexpr int THREADS = 128 / ROWS;
    const int r = blockIdx.x * ROWS + threadIdx.x / THREADS, at = threadIdx.x % THREADS;
    pdl_wait();
    Part mine = {-INFINITY, 0.0f, 0.0f};
    if (r < n) {
#pragma unroll 4
        for (int i = at; i < parts; i += THREADS) mine = join(mine, part_at(stats, i, parts, n, r));
    }
    mine = ROWS == 1 ? block_join<128>(mine, s_parts) : warp_join(mine);
    if (r < n && at == 0) write_row(mine, given, tokens[r], V, r, logprob, entropy, lse);
}

// With alternatives a block a row.  What is in no list is minus infinity (or not a number, which counts as that): where the lists
// hold fewer than k, the lowest ids that are in none follow.
template <int NT>
__global__ __launch_bounds__(NT) void head_join_kernel(
    const float* stats, const float* given, const u64* keys, const int32_t* tokens, int n, int V, int parts, int k,
    float* logprob, float* entropy, float* lse, int32_t* top_ids, float* top_logprobs) {
    pdl_trigger();
    __shared__ TopShared<NT> top;
    __shared__ Part s_parts[NT / 32];
    __shared__ Row s_row;
    const int r = blockIdx.x, tid = threadIdx.x;
    pdl_wait();
    Part mine = {-INFINITY, 0.0f, 0.0f};
    for (int i = tid; i < parts; i += NT) mine = join(mine, part_at(stats, i, parts, n, r));
    const u64* mine_k = keys + (size_t)r * parts * k;
    u64 best = 0;
    for (int i = tid; i < parts * k; i += NT) best = mine_k[i] > best ? mine_k[i] : best;
    auto each = [&](u64, auto f) {
        for (int i = tid; i < parts * k; i += NT) if (mine_k[i]) f(mine_k[i]);
    };
    if (!select_top<NT, 1>(top, best, best, k, each)) one_by_one<NT>(top, k, each);
    if (tid == 0) {
        int at = 0, id = 0;
        while (at < k && top.top[at]) ++at;
        for (const int found = at; at < k; ++at, ++id) {
            for (int j = 0; j < found; ++j) if (key_id(top.top[j]) == id) { ++id; j = -1; }
            top.top[at] = key_of(-INFINITY, id);
        }
    }
    const Part all = block_join<NT>(mine, s_parts);
    if (tid == 0) s_row = write_row(all, given, tokens[r], V, r, logprob, entropy, lse);
    __syncthreads();
    const Row w = s_row;
    for (int i = tid; i < k; i += NT) {
        const u64 key = top.top[i];
        top_ids[(size_t)r * k + i] = key_id(key);
        top_logprobs[(size_t)r * k + i] = log_prob(w, key_logit(key));
    }
}

// A tensor map of a row-major [rows][K] bfloat16 matrix with boxes of box_rows x 64.
static int head_map(CUtensorMap* out, const void* ptr, long long rows, long long K, long long ld, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return AIRUN_ERR_UNSUPPORTED;
    cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {BK, (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? AIRUN_OK : AIRUN_ERR_ARG;
}

template <bool PAIR, int TOP, bool ROLLED>
static int launch_head(const CUtensorMap& mx, const CUtensorMap& mw, HeadParams p, cudaStream_t stream) {
    static unsigned long long configured = 0;
    auto kern = head_logprobs_kernel<PAIR, TOP, ROLLED>;
    const int w_bytes = p.bn / (PAIR ? 2 : 1) * (BK * 2), x_bytes = p.x_rows * (BK * 2);
    // the products read 128 rows from a stage's first on, in the last one beyond what it brings
    const int beyond = 128 * BK * 2 - x_bytes;
    p.stages = (HEAD_SMEM - 1024 - beyond) / (w_bytes + x_bytes);
    if (p.stages > HEAD_STAGES) p.stages = HEAD_STAGES;
    const int smem = 1024 + p.stages * (w_bytes + x_bytes) + beyond;
    if (first_on_device(configured)) {
        cudaFuncAttributes at;
        cudaError_t e = cudaFuncGetAttributes(&at, kern);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, HEAD_SMEM);
        // the epilogue's warps would wait for good for registers that the block was not launched with
        if (e == cudaSuccess && at.numRegs < HEAD_REGS) e = cudaErrorInvalidKernelImage;
        if (e != cudaSuccess) { configured = 0; return (int)e; }
    }
    const long long units = (long long)p.row_blocks * p.splits;
    const int most = airun_sm_count() / (PAIR ? 2 : 1);
    const int groups = units < most ? (int)units : most;
    if constexpr (PAIR) airun_launch_clusters(kern, dim3(2 * groups), dim3(HEAD_THREADS), smem, stream, dim3(2), mx, mw, p);
    else airun_launch(kern, dim3(groups), dim3(HEAD_THREADS), smem, stream, mx, mw, p);
    return AIRUN_OK;
}

// x: [n][K], W: [V][K] bfloat16, rows ldx, ldw elements apart (16-byte aligned); the vocabulary in `splits` ranges of `tiles` tiles of `bn` ids, of which
// none is empty.  scratch: 4 (6 splits + 1) n bytes, rounded up to 16, and 16 splits n k more.
AIRUN_EXPORT int airun_head_logprobs(const void* x, const void* W, int n, int V, int K, long long ldx, long long ldw, const int32_t* tokens,
                                     float scale, float cap, int pair, int splits, int tiles, int bn, int part, void* scratch, float* logprob, float* entropy,
                                     float* lse, int k, int32_t* top_ids, float* top_logprobs, int* err, cudaStream_t stream) {
    if (n <= 0 || V <= 0 || K <= 0 || K % 8 || ldx < K || ldw < K || ldx % 8 || ldw % 8 || ((uintptr_t)x | (uintptr_t)W | (uintptr_t)scratch) & 15) return AIRUN_ERR_ARG;
    if (!x || !W || !tokens || !scratch || !logprob || !err || k < 0 || k > HEAD_TOP || k > V || (k > 0 && (!top_ids || !top_logprobs))) return AIRUN_ERR_ARG;
    if (bn < 16 || bn > 256 || bn % (pair ? 32 : 16) || part < 1 || tiles < 1 || splits < 1 || (long long)splits * tiles * bn < V || (long long)(splits - 1) * tiles * bn >= V) return AIRUN_ERR_ARG;
    const int row_blocks = (n + (pair ? 255 : 127)) / (pair ? 256 : 128);
    if ((long long)splits * tiles * bn > 0x7fff0000 || (long long)row_blocks * splits > 0x3fffffff || n > (1 << 27)) return AIRUN_ERR_ARG;
    CUtensorMap mx, mw;
    int r;
    const int x_rows = pair || n > 128 ? 128 : (n + 7) / 8 * 8;
    if ((r = head_map(&mx, x, n, K, ldx, x_rows)) != AIRUN_OK) return r;
    if ((r = head_map(&mw, W, V, K, ldw, pair ? bn / 2 : bn)) != AIRUN_OK) return r;
    HeadParams p = {n, V, K, row_blocks, splits, tiles, bn, part, x_rows, 0, tokens, scale, cap, k, (float*)scratch, nullptr, nullptr, err};
    p.given = p.stats + (size_t)6 * splits * n;
    p.keys = (u64*)((uint8_t*)scratch + ((size_t)4 * (6 * (size_t)splits + 1) * n + 15) / 16 * 16);
#define LAUNCH_HEAD(PAIR, ROLLED) (k == 0 ? launch_head<PAIR, 0, ROLLED>(mx, mw, p, stream) : k <= 8 ? launch_head<PAIR, 8, ROLLED>(mx, mw, p, stream) \
                                                                                            : launch_head<PAIR, 16, ROLLED>(mx, mw, p, stream))
    r = !pair ? LAUNCH_HEAD(false, true) : cap > 0.0f ? LAUNCH_HEAD(true, true) : LAUNCH_HEAD(true, false);
#undef LAUNCH_HEAD
    if (r != AIRUN_OK) return r;
    const float *stats = p.stats, *given = p.given;
    const u64* keys = p.keys;
    // few rows have a part an SM and more; a thread then looks at a few of them
    if (k == 0 && 2 * splits > 64)
        airun_launch(head_rows_kernel<1>, dim3(n), dim3(128), 0, stream, stats, given, tokens, n, V, 2 * splits, logprob, entropy, lse);
    else if (k == 0)
        airun_launch(head_rows_kernel<4>, dim3((n + 3) / 4), dim3(128), 0, stream, stats, given, tokens, n, V, 2 * splits, logprob, entropy, lse);
    else if (2 * splits * k > 256)
        airun_launch(head_join_kernel<512>, dim3(n), dim3(512), 0, stream, stats, given, keys, tokens, n, V, 2 * splits, k, logprob, entropy, lse, top_ids, top_logprobs);
    else
        airun_launch(head_join_kernel<128>, dim3(n), dim3(128), 0, stream, stats, given, keys, tokens, n, V, 2 * splits, k, logprob, entropy, lse, top_ids, top_logprobs);
    return airun_launch_status();
}

// ------------------------------------------------------------------ from hidden states, few rows
// Up to 32 rows the ids are the M side of the product and the rows its N side: an SM multiplies 16 or 32 columns where head_logprobs_kernel multiplies 128 rows
// whatever is in them, and its power goes into bytes.  The logits of a few rows are little beside the weights (4 n V bytes for 2 K V): they are written, and
// token_logprobs_kernel takes them from the L2.  A block walks a range of the vocabulary in tiles of `bn` <= 128 ids, of any number, so that the ranges come
// out even.  us, this and head_logprobs_kernel, weights of [151936, 4096] on a cool chip: 5 rows 191 and 190, with five alternatives 198 and 203; 24 rows 201 and 194, with eight
// 207 and 213; 32 rows 206 and 204, with eight 213 and 211; on a hot one 5 rows 202 and 196, with five 211 and 232, 32 rows 223 and 218, with eight 223 and 233.  5 rows x
// [20000, 1024] 13.0 and 14.6, 32 rows with five 18.9 and 28.4; 32 rows x [384, 64] 6.4 and 5.2, with three 8.8 and 10.2.  Without alternatives up to
// 3.5 % slower where weights are many, with them up to a third faster, and its sums are the more exact.
//   warp 0: TMA loads; warp 1: tensor memory, products; warps 2-5: the sums of a quadrant of lanes each, one id a thread.
// A stage is FEW_K K-steps, and its sums are parts of 64 values (128 for more than 16 rows) in neighbouring columns that are loaded together: a load takes 1,100
// clocks whatever its width.  (Stages of one K-step 237 us for 5 rows, of two 197.)  The stages' sums are added with compensation: entropies of 5 rows x 4,096
// off by 3.1e-7 in the mean square, by 7.8e-7 in parts of 128 without it (float32 products of cuBLAS 6.6e-7), 188.5 us for 187.6; 5 rows
// x [20000, 1024] 12.9 us for 12.2.
#define FEW_THREADS 192
#define FEW_STAGES 16                                              // at most
#define FEW_BUFS 4
#define FEW_K 4

struct FewParams {
    int n, V, K, tiles, bn;
    int w_stride, x_bytes, stages;                                 // bytes of a K-step; stages
    float scale, cap;
    float* logits;
    long long ld;
    int* err;
};

template <int N>
__global__ __launch_bounds__(FEW_THREADS, 1) void head_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const FewParams p) {
    __shared__ __align__(8) uint64_t bars[2 * FEW_STAGES + 2 * FEW_BUFS];
    __shared__ uint32_t tmem_slot;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    constexpr int PART = N == 16 ? 1 : 2;                          // K-steps of a part
    constexpr int COLS = N * (FEW_K / PART);                        // of a buffer: the parts of a stage
    const int kb_total = (p.K + FEW_K * BK - 1) / (FEW_K * BK), stages = p.stages;
    const int first_id = blockIdx.x * p.tiles * p.bn, end_id = min(p.V, first_id + p.tiles * p.bn);
    const uint32_t w_at = smem_u32(smem), x_at = w_at + stages * FEW_K * p.w_stride;
    const uint32_t full = smem_u32(bars), empty = full + 8 * FEW_STAGES, accf = empty + 8 * FEW_STAGES, acce = accf + 8 * FEW_BUFS;
    if (threadIdx.x == 0) {
        for (int s = 0; s < FEW_STAGES; ++s) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, 1); }
        for (int b = 0; b < FEW_BUFS; ++b) { mbar_init(accf + 8 * b, 1); mbar_init(acce + 8 * b, 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), FEW_BUFS * COLS);
    tc_fence_before();
    __syncthreads();
    pdl_trigger();                                                 // (as above)
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int n_steps = (end_id - first_id + p.bn - 1) / p.bn * kb_total, first_n = min(n_steps, stages);
    const uint32_t bytes = FEW_K * (p.bn * (BK * 2) + p.x_bytes);
    auto load_w = [&](int s, int kb, int w0) {
        mbar_expect_tx(full + 8 * s, bytes);
#pragma unroll
        for (int a = 0; a < FEW_K; ++a) tma_load_2d(w_at + (FEW_K * s + a) * p.w_stride, &map_w, full + 8 * s, (FEW_K * kb + a) * BK, w0);
    };
    if (warp == 0 && elect_one()) {                                // weights: no kernel writes them
        for (int it = 0, kb = 0, w0 = first_id; it < first_n; ++it) {
            load_w(it, kb, w0);
            if (++kb == kb_total) { kb = 0; w0 += p.bn; }
        }
    }
    __syncwarp();
    pdl_wait();                                                    // all warps: the waits below are bounded, the kernel in front is not
    bool ok = true;
    if (warp == 0) {
        int it = 0, s = 0, kb = 0, w0 = first_id;
        uint32_t phase = 0;
        for (; it < n_steps; ++it) {
            if (it >= first_n && !mbar_wait_warp(empty + 8 * s, phase ^ 1)) { ok = false; break; }
            if (elect_one()) {
                if (it >= first_n) load_w(s, kb, w0);
#pragma unroll
                for (int a = 0; a < FEW_K; ++a) tma_load_2d(x_at + (FEW_K * s + a) * p.x_bytes, &map_x, full + 8 * s, (FEW_K * kb + a) * BK, 0);
            }
            __syncwarp();
            if (++s == stages) { s = 0; phase ^= 1; }
            if (++kb == kb_total) { kb = 0; w0 += p.bn; }
        }
        // the last commits arrive at the barriers, and where a wait has run out the loads on their way land, before the block may leave
        const uint32_t last = ok ? empty : full;
        if (!ok) atomicOr(p.err, AIRUN_DEV_TIMEOUT);
        for (int i = max(0, it - stages); i < it; ++i)
            if (!mbar_wait_warp(last + 8 * (i % stages), (i / stages) & 1)) { atomicOr(p.err, AIRUN_DEV_TIMEOUT); break; }
    } else if (warp == 1) {
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        int s = 0;
        uint32_t phase = 0;
        for (int n = 0; n < n_steps; ++n) {
            const int buf = n % FEW_BUFS;
            ok = mbar_wait_warp(acce + 8 * buf, ((n / FEW_BUFS) & 1) ^ 1) && mbar_wait_warp(full + 8 * s, phase);
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int a = 0; a < FEW_K; ++a) {
                    const uint64_t dw = smem_desc_sw128(w_at + (FEW_K * s + a) * p.w_stride), dx = smem_desc_sw128(x_at + (FEW_K * s + a) * p.x_bytes);
#pragma unroll
                    for (int k = 0; k < BK / 16; ++k) umma_bf16(tmem + buf * COLS + a / PART * N, dw + (uint64_t)(k * 2), dx + (uint64_t)(k * 2), idesc, a % PART > 0 || k > 0 ? 1u : 0u);
                }
                umma_commit(empty + 8 * s);
                umma_commit(accf + 8 * buf);
            }
            __syncwarp();
            if (++s == stages) { s = 0; phase ^= 1; }
        }
        if (!ok) atomicOr(p.err, AIRUN_DEV_TIMEOUT);
    } else {
        const int quad = warp & 3;
        int n = 0;
        const float over_cap = 1.0f / p.cap;
        for (int w0 = first_id; w0 < end_id && ok; w0 += p.bn) {
            float acc[N], lost[N];                                 // (compensated as a row's sums are)
#pragma unroll
            for (int i = 0; i < N; ++i) acc[i] = lost[i] = 0.0f;
            for (int kb = 0; kb < kb_total; ++kb, ++n) {
                const int buf = n % FEW_BUFS;
                ok = mbar_wait_warp(accf + 8 * buf, (n / FEW_BUFS) & 1);
                if (!ok) { atomicOr(p.err, AIRUN_DEV_TIMEOUT); break; }
                tc_fence_after();
                uint32_t a[COLS];
#pragma unroll
                for (int i = 0; i < COLS; i += 32) tmem_ld32_async(tmem + buf * COLS + i + ((uint32_t)(quad * 32) << 16), a + i);
#pragma unroll
                for (int i = 0; i < COLS; i += 32) tmem_wait32(a + i);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(acce + 8 * buf) : "memory");
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    float sum = __uint_as_float(a[i]);
#pragma unroll
                    for (int j = N; j < COLS; j += N) sum += __uint_as_float(a[i + j]);
                    add_to(acc[i], lost[i], sum);
                    if (!(fabsf(lost[i]) < INFINITY)) lost[i] = 0.0f;        // (a sum that is infinite stays so)
                }
            }
            const int i = quad * 32 + lane;
            if (ok && i < min(p.bn, end_id - w0)) {
                float* to = p.logits + w0 + i;
#pragma unroll
                for (int r = 0; r < N; ++r) {
                    if (r < p.n) {
                        float x = acc[r];
                        if (p.scale != 1.0f) x *= p.scale;
                        if (p.cap > 0.0f) x = capped(x, p.cap, over_cap);
                        to[r * p.ld] = x;
                    }
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, FEW_BUFS * COLS);
    }
}

template <int N>
static int launch_few(const CUtensorMap& mx, const CUtensorMap& mw, FewParams p, cudaStream_t stream) {
    static unsigned long long configured = 0;
    auto kern = head_few_kernel<N>;
    // the products read 128 ids and N rows from a stage's first on, in the last ones beyond what they bring
    const int beyond_x = N * BK * 2 - p.x_bytes, beyond_w = 128 * BK * 2 - p.w_stride;
    p.stages = (HEAD_SMEM - 1024 - beyond_x - beyond_w) / (FEW_K * (p.w_stride + p.x_bytes));
    if (p.stages > FEW_STAGES) p.stages = FEW_STAGES;
    // all of the SM's shared memory, whatever the stages need: a kernel in front that has not taken its own tensor memory yet must not meet this one on its SM, which would
    // take it and wait for that kernel to end (head_logprobs_kernel has all of the SM's registers)
    const int smem = HEAD_SMEM;
    if (first_on_device(configured)) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, HEAD_SMEM);
        if (e != cudaSuccess) { configured = 0; return (int)e; }
    }
    airun_launch(kern, dim3((p.V + p.tiles * p.bn - 1) / (p.tiles * p.bn)), dim3(FEW_THREADS), smem, stream, mx, mw, p);
    return airun_launch_status();
}

// x, W and the results as above, n <= 32, k <= TOP_MAX; the vocabulary in ranges of `tiles` tiles of `bn` ids; logits: [n][ld] float32.
AIRUN_EXPORT int airun_head_few(const void* x, const void* W, int n, int V, int K, long long ldx, long long ldw, const int32_t* tokens, float scale, float cap,
                                int tiles, int bn, float* logits, long long ld, float* logprob, float* entropy, float* lse, int k, int32_t* top_ids,
                                float* top_logprobs, int* err, cudaStream_t stream) {
    if (n <= 0 || n > 32 || V <= 0 || V > 0x7fff0000 || K <= 0 || K % 8 || ldx < K || ldw < K || ldx % 8 || ldw % 8 || ((uintptr_t)x | (uintptr_t)W) & 15) return AIRUN_ERR_ARG;
    if (!tokens || !logprob || k < 0 || k > TOP_MAX || k > V || (k > 0 && (!top_ids || !top_logprobs))) return AIRUN_ERR_ARG;
    if (!x || !W || !logits || !err || ld < V || bn < 1 || bn > 128 || tiles < 1 || (long long)tiles * bn > 0x3fffffff) return AIRUN_ERR_ARG;
    if ((long long)V + (long long)tiles * bn > 0x7fff0000 || (long long)tiles * ((K + BK - 1) / BK) > 0x3fffffff) return AIRUN_ERR_ARG;
    CUtensorMap mx, mw;
    const int x_rows = (n + 7) / 8 * 8;
    int r;
    if ((r = head_map(&mx, x, n, K, ldx, x_rows)) != AIRUN_OK) return r;
    if ((r = head_map(&mw, W, V, K, ldw, bn)) != AIRUN_OK) return r;
    const FewParams p = {n, V, K, tiles, bn, (bn + 7) / 8 * 8 * (BK * 2), x_rows * (BK * 2), 0, scale, cap, logits, ld, err};
    if ((r = n <= 16 ? launch_few<16>(mx, mw, p, stream) : launch_few<32>(mx, mw, p, stream)) != AIRUN_OK) return r;
    return airun_token_logprobs(logits, AIRUN_DT_F32, ld, n, V, nullptr, tokens, n, logprob, entropy, lse, k, top_ids, top_logprobs, nullptr, stream);
}
