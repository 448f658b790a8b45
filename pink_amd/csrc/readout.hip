// readout.hip -- the read-out of a trained map (pink_hip_readout_* of include/pink_hip.h): images routed to neurons by
// their distances, the neurons' two-layer models, and the optimiser that trains both.  readout_rows.hip and readout_gated.hip have the handle's
// other operators.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <new>
#include <type_traits>

#include "readout_handle.h"
#include "readout_product.inc"

namespace {

constexpr uint32_t kMaxNeurons = 32768, kMaxChosen = 64, kMaxGroups = 1024;
constexpr uint32_t kBlock8 = 256;                          // codes that share a scale

// ---------------------------------------------------------------------------------
// Routing
// ---------------------------------------------------------------------------------

struct RouteArgs {
    const float *distances;
    uint64_t stride;
    const float *sharpness, *radius, *bias;
    uint32_t images, neurons, chosen, groups, groups_kept, group_size;
    uint32_t sigmoid, renormalise;
    int32_t *neuron;
    float *gates;
};

// An entry's key in the choice: a number that grows with z + bias, 0 where the entry takes no part.
// (An infinite or NaN z does not become finite by a bias.)
__device__ __forceinline__ uint32_t order_key(float biased)
{
    if (!isfinite(biased)) return 0;
    const uint32_t bits = __float_as_uint(biased + 0.0f);  // (-0 and 0 tie)
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t key)
{
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// A group's key from the two largest of its neurons.
__device__ __forceinline__ uint32_t group_score(uint32_t first, uint32_t second)
{
    if (!second) return first;
    const float both = key_value(first) + key_value(second);
    return order_key(fminf(fmaxf(both, -3.402823466e38f), 3.402823466e38f));
}

__device__ __forceinline__ float logit(const RouteArgs &g, const float *row, uint32_t n)
{
    return g.sharpness[n] * (g.radius[n] - row[n]);
}

// Gates of an image's chosen neurons, a lane each (at most 64); `z` of a lane without a neuron does not count.
__device__ __forceinline__ float gate_of(const RouteArgs &g, float z, bool valid, float top, float total)
{
    if (g.renormalise) {
        const float level = g.sigmoid ? fminf(z, 0.0f) - log1pf(expf(-fabsf(z))) : z;
        const float highest = wave_max(valid ? level : -INFINITY);
        const float e = valid ? expf(level - highest) : 0.0f;
        const float sum = wave_sum(e);
        return valid ? e / sum : 0.0f;
    }
    if (!valid) return 0.0f;
    return g.sigmoid ? 1.0f / (1.0f + expf(-z)) : expf(z - top) / total;
}

// The general form, a block per image: keys in LDS, the groups kept by counting how many go before each, then the largest key
// `chosen` times, each a pass over LDS.  For what k_route_wave does not take: more than 2048 neurons, or more than 64 groups.
// 16000 images, 8 chosen: 146 us of 2500 neurons, 240 of 5000 (34 and 67 for reading them); 424 with 10 of 50 groups of 2500.
__global__ __launch_bounds__(256) void k_route_block(const RouteArgs g)
{
    extern __shared__ __align__(16) uint32_t lds[];
    uint32_t *const keys = lds, *const group_keys = lds + g.neurons;     // neurons, groups
    __shared__ uint32_t best_key[4], best_at[4];
    __shared__ float wave_top[4], wave_total[4];
    __shared__ int32_t picked[kMaxChosen];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float *const row = g.distances + (uint64_t)blockIdx.x * g.stride;

    float top = -INFINITY;
    for (uint32_t n = tid; n < g.neurons; n += 256) {
        const float z = logit(g, row, n), biased = g.bias ? z + g.bias[n] : z;
        const uint32_t key = order_key(biased);
        keys[n] = key;
        if (key) top = fmaxf(top, z);
    }
    top = wave_max(top);
    if (lane == 0) wave_top[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
    float total = 0.0f;
    if (!g.renormalise && !g.sigmoid) {
        for (uint32_t n = tid; n < g.neurons; n += 256)
            if (keys[n]) total += expf(logit(g, row, n) - top);
        total = wave_sum(total);
        if (lane == 0) wave_total[wave] = total;
        __syncthreads();
        total = (wave_total[0] + wave_total[1]) + (wave_total[2] + wave_total[3]);
    }

    if (g.groups > 1) {
        for (uint32_t k = wave; k < g.groups; k += 4) {
            uint32_t first = 0, second = 0;
            const uint32_t end = min((k + 1) * g.group_size, g.neurons);
            for (uint32_t n = k * g.group_size + lane; n < end; n += 64) {
                const uint32_t key = keys[n];
                second = max(second, min(first, key));
                first = max(first, key);
            }
#pragma unroll
            for (int off = 32; off >= 1; off >>= 1) {
                const uint32_t a = __shfl_xor((int)first, off, 64), b = __shfl_xor((int)second, off, 64);
                second = max(max(second, b), min(first, a));
                first = max(first, a);
            }
            if (lane == 0) {
                group_keys[k] = group_score(first, second);
            }
        }
        __syncthreads();
        for (uint32_t n = tid; n < g.neurons; n += 256) {
            const uint32_t mine = n / g.group_size, key = group_keys[mine];
            uint32_t before = 0;
            for (uint32_t k = 0; k < g.groups; ++k) before += group_keys[k] > key || (group_keys[k] == key && k < mine);
            if (before >= g.groups_kept) keys[n] = 0;
        }
        __syncthreads();
    }

    for (uint32_t s = 0; s < g.chosen; ++s) {
        uint32_t key = 0, at = 0xffffffffu;
        for (uint32_t n = tid; n < g.neurons; n += 256)
            if (keys[n] > key) {
                key = keys[n];
                at = n;
            }
        const uint32_t highest = wave_max_u32(key);
        const uint32_t lowest = ~wave_max_u32(key == highest && key ? ~at : 0u);
        if (lane == 0) {
            best_key[wave] = highest;
            best_at[wave] = lowest;
        }
        __syncthreads();
        if (tid == 0) {
            uint32_t k = 0, a = 0xffffffffu;
            for (int w = 0; w < 4; ++w)
                if (best_key[w] > k || (best_key[w] == k && best_at[w] < a)) {
                    k = best_key[w];
                    a = best_at[w];
                }
            picked[s] = k ? (int32_t)a : -1;
            if (k) keys[a] = 0;
        }
        __syncthreads();
    }
    if (wave == 0) {
        const int32_t n = lane < g.chosen ? picked[lane] : -1;
        const float gate = gate_of(g, n >= 0 ? logit(g, row, n) : 0.0f, n >= 0, top, total);
        if (lane < g.chosen) {
            g.neuron[(uint64_t)blockIdx.x * g.chosen + lane] = n;
            g.gates[(uint64_t)blockIdx.x * g.chosen + lane] = gate;
        }
    }
}

// Neurons' keys in registers: what a wave holds of an image, candidate 64 j + lane in key[j].
template <int J> struct Candidates {
    static constexpr int kSet = J <= 8 ? J : J % 8 ? 4 : 8, kSets = J / kSet;
    static_assert(J % kSet == 0, "whole sets");
    uint32_t key[J], best[kSets], where[kSets];            // of each set of registers: the largest key and its register

    template <int B> __device__ __forceinline__ void find()
    {
        best[B] = key[B * kSet];
        where[B] = B * kSet;
#pragma unroll
        for (int i = 1; i < kSet; ++i)
            if (key[B * kSet + i] > best[B]) {
                best[B] = key[B * kSet + i];
                where[B] = B * kSet + i;
            }
    }
    template <int B> __device__ __forceinline__ void find_all()
    {
        find<B>();
        if constexpr (B + 1 < kSets) find_all<B + 1>();
    }
    // Takes one candidate, of register j in lane l, out; only its set of registers is gone through again.
    template <int B> __device__ __forceinline__ void remove(uint32_t j, uint32_t l, uint32_t lane)
    {
        if (j / kSet == B) {
#pragma unroll
            for (int i = 0; i < kSet; ++i)
                if (j == B * kSet + i && lane == l) key[B * kSet + i] = 0;
            find<B>();
        }
        if constexpr (B + 1 < kSets) remove<B + 1>(j, l, lane);
    }
    // The next candidate in order (the largest key, the lowest number on ties), or none: -1.
    __device__ __forceinline__ int take(uint32_t lane)
    {
        uint32_t k = best[0], w = where[0];
#pragma unroll
        for (int b = 1; b < kSets; ++b)
            if (best[b] > k) {
                k = best[b];
                w = where[b];
            }
        const uint32_t most = wave_max_u32(k);
        if (most == 0) return -1;
        const unsigned long long holders = __ballot(k == most);
        uint32_t c = w * 64 + lane;
        if (__popcll(holders) == 1) c = (uint32_t)__builtin_amdgcn_readlane((int)c, __ffsll(holders) - 1);
        else c = ~wave_max_u32(k == most ? ~c : 0);
        remove<0>(c / 64, c % 64, lane);
        return (int)c;
    }
};

// A wave per image, for up to 2048 neurons in at most 64 groups: keys in registers, the k largest taken one by one (a maximum over
// the wave each).  With groups, keys go through LDS: lane g finds group g's two largest, the largest groups are taken one by one, and
// only their neurons are candidates, in the order of their numbers.  Each distance is read once.  16000 images x 1600 neurons, 8 of
// 40 groups, 8 chosen: 48 us (2.1 TB/s; k_route_block 308 us), bound by the vector ALU (1500 instructions an image, 40 us of the
// chip's) and the latencies between them; a reading pass alone would take 22 us.  1001 x 331, full softmax: 4.4 us.
// J: registers for all neurons, C: for the candidates; FULL: gates over the sum of all neurons that take part.
template <int J, int C, bool FULL> __global__ __launch_bounds__(256) void k_route_wave(const RouteArgs g, uint32_t over_size)
{
    extern __shared__ __align__(16) uint32_t lds[];        // with groups: waves x (groups x line + 64)
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t t = blockIdx.x * 4 + wave;
    if (t >= g.images) return;                             // (no barriers below)
    const float *const row = g.distances + (uint64_t)t * g.stride;
    uint32_t keys_of[J];
    Candidates<C> c;
    float top = -INFINITY, total = 0.0f;
    {
        float z[FULL ? J : 1];
        constexpr int kAtOnce = J < 8 ? J : J % 8 ? 4 : 8;               // loads of so many registers are under way together
#pragma unroll
        for (int j0 = 0; j0 < J; j0 += kAtOnce) {
            float d[kAtOnce], of[kAtOnce], to[kAtOnce], bias[kAtOnce];
            uint32_t n[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                n[j] = min((uint32_t)(j0 + j) * 64 + lane, g.neurons - 1);
                d[j] = row[n[j]];
                of[j] = g.sharpness[n[j]];
                to[j] = g.radius[n[j]];
                bias[j] = 0.0f;
            }
            if (g.bias) {
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) bias[j] = g.bias[n[j]];
            }
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
                const float at = of[j] * (to[j] - d[j]);
                const uint32_t key = order_key(at + bias[j]);
                if (FULL) z[j0 + j] = at;
                keys_of[j0 + j] = (uint32_t)(j0 + j) * 64 + lane < g.neurons ? key : 0;
                asm volatile("" : "+v"(keys_of[j0 + j]));  // formed here: what it is formed from would take four registers, and waves with them
            }
        }
        if constexpr (FULL) {
#pragma unroll
            for (int j = 0; j < J; ++j) top = fmaxf(top, keys_of[j] ? z[j] : -INFINITY);
            top = wave_max(top);
#pragma unroll
            for (int j = 0; j < J; ++j) total += keys_of[j] ? expf(z[j] - top) : 0.0f;
            total = wave_sum(total);
        }
    }
    const uint32_t line = g.group_size | 1;                // a group's keys in LDS: an odd step, so that lanes reading one each meet no banks
    uint32_t *const keys = lds + wave * (g.groups * line + 64), *const kept_groups = keys + g.groups * line;
    if (g.groups > 1) {
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (j * 64 + lane < g.neurons) {
                const uint32_t n = j * 64 + lane, group = g.group_size == 1 ? n : __umulhi(n, over_size);
                keys[n + group * (line - g.group_size)] = keys_of[j];
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint32_t score = 0;
        if (lane < g.groups) {
            const uint32_t size = min(g.group_size, g.neurons - lane * g.group_size);
            const uint32_t *const mine = keys + lane * line;
            uint32_t first = 0, second = 0;
#pragma unroll 8
            for (uint32_t i = 0; i < size; ++i) {
                const uint32_t key = mine[i];
                second = max(second, min(first, key));
                first = max(first, key);
            }
            score = group_score(first, second);
        }
        unsigned long long all = 0;                        // the kept groups, taken one by one
        for (uint32_t k = 0; k < g.groups_kept; ++k) {
            const uint32_t most = wave_max_u32(score);
            if (most == 0) break;
            const unsigned long long one = __ballot(score == most) & -__ballot(score == most);
            all |= one;
            if (one >> lane & 1) score = 0;
        }
        const bool kept = all >> lane & 1;
        if (kept) kept_groups[__popcll(all & ((1ull << lane) - 1))] = lane;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint32_t count = __popcll(all) * g.group_size;
#pragma unroll
        for (int j = 0; j < C; ++j) {
            c.key[j] = 0;
            if (j * 64 < count) {
                const uint32_t i = j * 64 + lane, slot = g.group_size == 1 ? i : __umulhi(i, over_size);
                if (i < count) {
                    const uint32_t group = kept_groups[slot], in_group = i - slot * g.group_size;
                    if (group * g.group_size + in_group < g.neurons) c.key[j] = keys[group * line + in_group];
                }
            }
        }
    }
    if (g.groups == 1) {
#pragma unroll
        for (int j = 0; j < C; ++j) c.key[j] = j < J ? keys_of[j] : 0;
    }
    c.template find_all<0>();
    int mine = -1;
    for (uint32_t s = 0; s < g.chosen; ++s) {
        const int next = c.take(lane);
        if (next < 0) break;
        if (lane == s) mine = next;
    }
    if (mine >= 0 && g.groups > 1) {
        const uint32_t slot = g.group_size == 1 ? (uint32_t)mine : __umulhi((uint32_t)mine, over_size);
        mine = (int)(kept_groups[slot] * g.group_size + ((uint32_t)mine - slot * g.group_size));
    }
    const float gate = gate_of(g, mine >= 0 ? logit(g, row, mine) : 0.0f, mine >= 0, top, total);
    if (lane < g.chosen) {
        g.neuron[(uint64_t)t * g.chosen + lane] = mine;
        g.gates[(uint64_t)t * g.chosen + lane] = gate;
    }
}

struct RouteBackwardArgs {
    RouteArgs r;                   // neuron and gates are inputs here
    const void *gate_gradients;
    float *distance_gradients;
    float *sharpness_part, *radius_part;       // chunks x N each
    uint32_t chunk;                // images of a block
    uint32_t want_sums;
};

constexpr uint32_t kChunkMost = 64;

// Gradients of a chunk of images over a strip of 256 neurons.  Waves first form each image's own numbers: dz of its chosen
// neurons and, for the full softmax, its normaliser and what every neuron's share is multiplied with.  Then a thread goes
// down its neuron's column, in the images' order.
//   renormalised: dz_c = g_c (G_c - sum_s g_s G_s) [sigmoid: times 1 - sigmoid(z_c)];  sigmoid: dz_c = G_c s (1 - s);
//   softmax: dz_n = [n chosen] g_n G_n - share_n sum_s g_s G_s
// Sums over images are formed a chunk at a time and then over the chunks, always in the same order.  Bound by latency at the sizes
// of a batch: 1001 images x 331 neurons, full softmax, 9 us and 4 us for the sums over 251 chunks.  16000 x 1600: 80 us, with the full
// softmax 481 (every strip forms its images' maxima and sums anew), where reading and writing alone would take 43.
template <typename E> __global__ __launch_bounds__(256) void k_route_backward(const RouteBackwardArgs a)
{
    const RouteArgs &g = a.r;
    extern __shared__ __align__(16) char lds_raw[];
    float *const dz = (float *)lds_raw;                                  // chunk x chosen
    int32_t *const at = (int32_t *)(dz + a.chunk * g.chosen);            // chunk x chosen
    __shared__ float top_of[kChunkMost], over_of[kChunkMost], pull_of[kChunkMost];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t t0 = blockIdx.y * a.chunk, count = min(a.chunk, g.images - t0);
    const bool full = !g.sigmoid && !g.renormalise;

    for (uint32_t i = wave; i < count; i += 4) {
        const uint64_t slot = (uint64_t)(t0 + i) * g.chosen + lane;
        const float *const row = g.distances + (uint64_t)(t0 + i) * g.stride;
        const int32_t n = lane < g.chosen ? g.neuron[slot] : -1;
        const bool valid = n >= 0 && (uint32_t)n < g.neurons;
        const float gate = valid ? g.gates[slot] : 0.0f, grad = valid ? to_float(((const E *)a.gate_gradients)[slot]) : 0.0f;
        const float z = valid ? logit(g, row, n) : 0.0f;
        const float pull = wave_sum(gate * grad);
        float d;
        if (g.renormalise) {
            d = gate * (grad - pull);
            if (g.sigmoid) d /= 1.0f + expf(z);
        } else {
            d = gate * grad;
            if (g.sigmoid) d /= 1.0f + expf(z);
        }
        if (lane < g.chosen) {
            dz[i * g.chosen + lane] = valid ? d : 0.0f;
            at[i * g.chosen + lane] = valid ? n : -1;
        }
        if (full) {
            float top = -INFINITY, total = 0.0f;
            for (uint32_t m = lane; m < g.neurons; m += 64) {
                const float v = logit(g, row, m);
                if (order_key(g.bias ? v + g.bias[m] : v)) top = fmaxf(top, v);
            }
            top = wave_max(top);
            for (uint32_t m = lane; m < g.neurons; m += 64) {
                const float v = logit(g, row, m);
                if (order_key(g.bias ? v + g.bias[m] : v)) total += expf(v - top);
            }
            total = wave_sum(total);
            if (lane == 0) {
                top_of[i] = top;
                over_of[i] = total > 0.0f ? 1.0f / total : 0.0f;
                pull_of[i] = pull;
            }
        }
    }
    __syncthreads();

    const uint32_t n = blockIdx.x * 256 + tid;
    if (n >= g.neurons) return;
    const float sharpness = g.sharpness[n], radius = g.radius[n], bias = g.bias ? g.bias[n] : 0.0f;
    float of_sharpness = 0.0f, of_radius = 0.0f;
    for (uint32_t i = 0; i < count; ++i) {
        const uint64_t place = (uint64_t)(t0 + i) * g.stride + n;
        float d = 0.0f;
        if (full) {
            const float v = sharpness * (radius - g.distances[place]);
            if (order_key(v + bias)) d = -pull_of[i] * (expf(v - top_of[i]) * over_of[i]);
        }
        for (uint32_t s = 0; s < g.chosen; ++s)
            if (at[i * g.chosen + s] == (int32_t)n) d += dz[i * g.chosen + s];
        if (a.distance_gradients) a.distance_gradients[(uint64_t)(t0 + i) * g.neurons + n] = -sharpness * d;
        if (d != 0.0f) {
            of_sharpness += d * (radius - g.distances[place]);
            of_radius += sharpness * d;
        }
    }
    if (a.want_sums) {
        a.sharpness_part[(uint64_t)blockIdx.y * g.neurons + n] = of_sharpness;
        a.radius_part[(uint64_t)blockIdx.y * g.neurons + n] = of_radius;
    }
}

// Column sums of the chunks' parts: 64 columns by 16 waves, each a sixteenth of the chunks in order.
__global__ __launch_bounds__(1024) void k_route_sums(const float *sharpness_part, const float *radius_part, uint32_t chunks, uint32_t neurons,
                                                     float *sharpness_out, float *radius_out)
{
    __shared__ float held[2][16][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.x * 64 + lane;
    const uint32_t each = (chunks + 15) / 16, first = min(wave * each, chunks), end = min(first + each, chunks);
    float s = 0.0f, r = 0.0f;
    if (n < neurons) {
#pragma unroll 8
        for (uint32_t c = first; c < end; ++c) {
            s += sharpness_part[(uint64_t)c * neurons + n];
            r += radius_part[(uint64_t)c * neurons + n];
        }
    }
    held[0][wave][lane] = s;
    held[1][wave][lane] = r;
    __syncthreads();
    if (wave > 1 || n >= neurons) return;
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += held[wave][w][lane];
    float *const out = wave ? radius_out : sharpness_out;
    if (out) out[n] = sum;
}

// One block: how often each neuron was chosen, then a step of the bias against the mean.  4004 slots 5.6 us, 64000 slots 15 us.
__global__ __launch_bounds__(1024) void k_balance(const int32_t *neuron, uint64_t slots, uint32_t neurons, float rate, float *bias, int32_t *load)
{
    extern __shared__ __align__(16) uint32_t counts[];
    __shared__ uint32_t used;
    for (uint32_t n = threadIdx.x; n < neurons; n += 1024) counts[n] = 0;
    if (threadIdx.x == 0) used = 0;
    __syncthreads();
    uint32_t mine = 0;
    for (uint64_t i = threadIdx.x; i < slots; i += 1024) {
        const uint32_t n = (uint32_t)neuron[i];
        if (n < neurons) {
            atomicAdd(&counts[n], 1u);
            ++mine;
        }
    }
    if (mine) atomicAdd(&used, mine);
    __syncthreads();
    for (uint32_t n = threadIdx.x; n < neurons; n += 1024) {
        const uint64_t mean = used, now = (uint64_t)counts[n] * neurons;            // both times N: exact
        bias[n] += now < mean ? rate : now > mean ? -rate : 0.0f;
        if (load) load[n] = (int32_t)counts[n];
    }
}

// ---------------------------------------------------------------------------------
// Rows sorted by neuron
// ---------------------------------------------------------------------------------

// A stable counting sort of the slots by neuron.  A block takes waves * 64 * PER slots in order (four a lane where one block does
// all, one where blocks share the work); a wave goes through its own in order with a histogram of its own, so that ranks need no
// atomics and the order is that of the images always (sums over a neuron's rows are the same bits each time).  Lanes with the
// same neuron find each other by ballots over the bits of its number.
// 32000 slots, 100 neurons: 15 us in three launches; 602 slots, 331 neurons: 6 us in one.  Bound by latencies.

struct PlanArgs {
    const int32_t *neuron;
    uint32_t slots, neurons, tile_rows;
    uint32_t *counts;              // blocks x N
    uint32_t *order, *offsets, *tile_count;                // row -> slot; neuron -> first row
    int32_t *owner;                // slot -> neuron
    int32_t *place;                // slot -> row, -1 where it has none
    uint2 *tiles;
};

// Exclusive prefix sums over the block of one 64-bit value a thread.
__device__ __forceinline__ unsigned long long block_prefix(unsigned long long v, unsigned long long *shared, unsigned long long *total)
{
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    unsigned long long sum = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const unsigned long long o = __shfl_up(sum, off, 64);
        if ((int)lane >= off) sum += o;
    }
    if (lane == 63) shared[wave] = sum;
    __syncthreads();
    unsigned long long before = 0, all = 0;
    for (uint32_t w = 0; w < waves; ++w) {
        if (w < wave) before += shared[w];
        all += shared[w];
    }
    __syncthreads();
    *total = all;
    return before + sum - v;
}

// First rows and tiles of all neurons from their numbers of rows: rows in the low half, tiles in the high half of one sum.  A thread
// has a run of neurons; `count` gives a neuron's number of rows and `starts` is told its first row.
template <typename Count, typename Starts>
__device__ __forceinline__ void plan_offsets(const PlanArgs &g, const Count &count, const Starts &starts, unsigned long long *shared)
{
    const uint32_t each = (g.neurons + blockDim.x - 1) / blockDim.x;
    const uint32_t first = min(threadIdx.x * each, g.neurons), end = min(first + each, g.neurons);
    unsigned long long mine = 0, total;
    for (uint32_t n = first; n < end; ++n) {
        const uint32_t c = count(n);
        mine += c | (unsigned long long)((c + g.tile_rows - 1) / g.tile_rows) << 32;
    }
    unsigned long long at = block_prefix(mine, shared, &total);
    uint32_t last = (uint32_t)mine;                        // (of a run of one: its count)
    for (uint32_t n = first; n < end; ++n) {
        const uint32_t c = each == 1 ? last : count(n);
        g.offsets[n] = (uint32_t)at;
        starts(n, (uint32_t)at);
        uint32_t tile = (uint32_t)(at >> 32);
        for (uint32_t r = 0; r < c; r += g.tile_rows) g.tiles[tile++] = make_uint2(n, (uint32_t)at + r);
        at += c | (unsigned long long)((c + g.tile_rows - 1) / g.tile_rows) << 32;
    }
    if (threadIdx.x == 0) {
        g.offsets[g.neurons] = (uint32_t)total;
        *g.tile_count = (uint32_t)(total >> 32);
    }
}

// STAGE 0: count only; 1: place rows, from counts' prefixes; 2: all in one block, of which the first `waves` have slots.
template <int STAGE> constexpr uint32_t kPerWave = STAGE == 2 ? 4 : 1;

template <int STAGE> __global__ __launch_bounds__(1024) void k_plan(const PlanArgs g)
{
    constexpr uint32_t PER = kPerWave<STAGE>;
    extern __shared__ __align__(16) uint32_t hist[];       // waves x N
    __shared__ unsigned long long shared[16];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = STAGE == 2 ? (g.slots + 64 * PER - 1) / (64 * PER) : blockDim.x >> 6;
    const uint64_t first = ((uint64_t)blockIdx.x * waves + wave) * 64 * PER;
    uint32_t rank[PER], id[PER];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint64_t slot = first + i * 64 + lane;
        id[i] = slot < g.slots ? (uint32_t)g.neuron[slot] : 0xffffffffu;
    }
    for (uint32_t i = threadIdx.x; i < waves * g.neurons; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    volatile uint32_t *const mine = hist + min(wave, waves - 1) * g.neurons;         // (a wave without slots touches nothing)
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const bool valid = id[i] < g.neurons;
        unsigned long long same = __ballot(valid);
        for (uint32_t b = 0; (g.neurons - 1) >> b; ++b) {
            const unsigned long long set = __ballot(id[i] >> b & 1);
            same &= id[i] >> b & 1 ? set : ~set;
        }
        const uint32_t below = __popcll(same & ((1ull << lane) - 1));
        rank[i] = valid ? mine[id[i]] + below : 0;
        __builtin_amdgcn_wave_barrier();
        if (valid && below == 0) mine[id[i]] = rank[i] + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // Of a neuron's rows those of the waves before; returns all of the block's.
    const auto over_waves = [&](uint32_t n) {
        uint32_t before = 0;
        for (uint32_t w = 0; w < waves; ++w) {
            const uint32_t c = hist[w * g.neurons + n];
            hist[w * g.neurons + n] = before;
            before += c;
        }
        return before;
    };
    if constexpr (STAGE == 2) {
        bool again = false;                                // (of a run of several neurons, counts are looked at twice: kept in memory)
        plan_offsets(
            g,
            [&](uint32_t n) {
                if (g.neurons <= blockDim.x) return over_waves(n);
                const uint32_t each = (g.neurons + blockDim.x - 1) / blockDim.x;
                if (!again) g.counts[n] = over_waves(n);
                again = again || n + 1 == min((threadIdx.x + 1) * each, g.neurons);
                return g.counts[n];
            },
            [&](uint32_t n, uint32_t start) {
                for (uint32_t w = 0; w < waves; ++w) hist[w * g.neurons + n] += start;
            },
            shared);
    } else {
        for (uint32_t n = threadIdx.x; n < g.neurons; n += blockDim.x) {
            const uint32_t all = over_waves(n);
            if (STAGE == 0) g.counts[(uint64_t)blockIdx.x * g.neurons + n] = all;
        }
    }
    if (STAGE == 0) return;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint64_t slot = first + i * 64 + lane;
        if (slot >= g.slots) continue;
        int32_t row = -1;
        if (id[i] < g.neurons) {
            row = (int32_t)(mine[id[i]] + rank[i]);
            if (STAGE == 1) row += (int32_t)(g.offsets[id[i]] + g.counts[(uint64_t)blockIdx.x * g.neurons + id[i]]);
            g.order[row] = (uint32_t)slot;
        }
        g.place[slot] = row;
        g.owner[slot] = (int32_t)id[i];
    }
}

// One block: every block's counts become the rows of its neuron that lie in blocks before; first rows and tiles.
__global__ __launch_bounds__(1024) void k_plan_offsets(const PlanArgs g, uint32_t blocks, uint32_t *totals)
{
    __shared__ unsigned long long shared[16];
    for (uint32_t n = threadIdx.x; n < g.neurons; n += blockDim.x) {
        uint32_t before = 0;
        for (uint32_t b0 = 0; b0 < blocks; b0 += 16) {     // sixteen loads under way
            uint32_t c[16];
#pragma unroll
            for (uint32_t b = 0; b < 16; ++b) c[b] = b0 + b < blocks ? g.counts[(uint64_t)(b0 + b) * g.neurons + n] : 0;
#pragma unroll
            for (uint32_t b = 0; b < 16; ++b) {
                if (b0 + b < blocks) g.counts[(uint64_t)(b0 + b) * g.neurons + n] = before;
                before += c[b];
            }
        }
        totals[n] = before;
    }
    __syncthreads();
    plan_offsets(g, [&](uint32_t n) { return totals[n]; }, [](uint32_t, uint32_t) {}, shared);
}

// ---------------------------------------------------------------------------------
// Few images: a slot by itself
// ---------------------------------------------------------------------------------

struct FewArgs {
    const void *x;
    uint64_t x_stride;
    const int32_t *neuron;
    const float *gates;
    const void *first, *first_bias, *second, *second_bias, *residual;
    uint64_t residual_stride, y_stride;
    uint32_t neurons, chosen, features, hidden, outputs, activation;
    float *after;                  // slots x hidden
    void *y;
};

template <typename E> __device__ __forceinline__ void to_floats(const uint4 &chunk, float (&v)[16 / sizeof(E)])
{
    E e[16 / sizeof(E)];
    __builtin_memcpy(e, &chunk, sizeof e);
#pragma unroll
    for (uint32_t i = 0; i < 16 / sizeof(E); ++i) v[i] = to_float(e[i]);
}

// With a handful of slots nothing is shared and what there is to do is to read each slot's weights once: a wave takes four rows of
// a matrix, its lanes 16 bytes each along them, and sums up over the lanes.  No sorting, no tiles, two launches; sums and what
// lies between the layers stay in float32.  One image, 2 of 100 neurons, 1024 x 256 x 64: 5 us a launch, all latency (1.1 MB); 16
// slots of 331 neurons, 2025 x 200 x 45 float32: 14.5 us for both.
constexpr uint32_t kFewRows = 4;

template <typename E> __global__ __launch_bounds__(256) void k_few_hidden(const FewArgs g)
{
    constexpr uint32_t per = 16 / sizeof(E);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t slot = blockIdx.y, neuron = (uint32_t)g.neuron[slot], h0 = (blockIdx.x * 4 + wave) * kFewRows;
    if (neuron >= g.neurons || h0 >= g.hidden) return;
    const E *const x = (const E *)g.x + (uint64_t)(slot / g.chosen) * g.x_stride;
    const E *w[kFewRows];
#pragma unroll
    for (uint32_t i = 0; i < kFewRows; ++i) w[i] = (const E *)g.first + ((uint64_t)neuron * g.hidden + min(h0 + i, g.hidden - 1)) * g.features;
    float sum[kFewRows] = {};
    for (uint32_t k = lane * per; k < g.features; k += 64 * per) {
        const int valid = (int)(g.features - k);
        float a[per];
        uint4 b[kFewRows];
        to_floats<E>(load_chunk(x + k, valid), a);
#pragma unroll
        for (uint32_t i = 0; i < kFewRows; ++i) b[i] = load_chunk(w[i] + k, valid);
#pragma unroll
        for (uint32_t i = 0; i < kFewRows; ++i) {
            float v[per];
            to_floats<E>(b[i], v);
#pragma unroll
            for (uint32_t e = 0; e < per; ++e) sum[i] = fmaf(a[e], v[e], sum[i]);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kFewRows; ++i) {
        float v = wave_sum(sum[i]);
        if (lane == 0 && h0 + i < g.hidden) {
            if (g.first_bias) v += to_float(((const E *)g.first_bias)[(uint64_t)neuron * g.hidden + h0 + i]);
            g.after[(uint64_t)slot * g.hidden + h0 + i] = g.gates[slot] * activation<E, false>(g.activation, v).value;
        }
    }
}

template <typename E> __global__ __launch_bounds__(256) void k_few_answer(const FewArgs g)
{
    constexpr uint32_t per = 16 / sizeof(E);
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t t = blockIdx.y, o0 = (blockIdx.x * 4 + wave) * kFewRows;
    if (o0 >= g.outputs) return;
    float sum[kFewRows] = {}, bias[kFewRows] = {};
    for (uint32_t s = 0; s < g.chosen; ++s) {
        const uint32_t slot = t * g.chosen + s, neuron = (uint32_t)g.neuron[slot];
        if (neuron >= g.neurons) continue;
        const float *const after = g.after + (uint64_t)slot * g.hidden;
        const E *w[kFewRows];
#pragma unroll
        for (uint32_t i = 0; i < kFewRows; ++i) {
            const uint64_t row = (uint64_t)neuron * g.outputs + min(o0 + i, g.outputs - 1);
            w[i] = (const E *)g.second + row * g.hidden;
            if (g.second_bias) bias[i] += g.gates[slot] * to_float(((const E *)g.second_bias)[row]);
        }
        for (uint32_t k = lane * per; k < g.hidden; k += 64 * per) {
            const int valid = (int)(g.hidden - k);
            float a[per];
            uint4 b[kFewRows];
#pragma unroll
            for (uint32_t e = 0; e < per; ++e) a[e] = (int)e < valid ? after[k + e] : 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < kFewRows; ++i) b[i] = load_chunk(w[i] + k, valid);
#pragma unroll
            for (uint32_t i = 0; i < kFewRows; ++i) {
                float v[per];
                to_floats<E>(b[i], v);
#pragma unroll
                for (uint32_t e = 0; e < per; ++e) sum[i] = fmaf(a[e], v[e], sum[i]);
            }
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kFewRows; ++i) {
        float v = wave_sum(sum[i]) + bias[i];
        if (lane == 0 && o0 + i < g.outputs) {
            if (g.residual) v += to_float(((const E *)g.residual)[t * g.residual_stride + o0 + i]);
            ((E *)g.y)[t * g.y_stride + o0 + i] = from_float<E>(v);
        }
    }
}

// ---------------------------------------------------------------------------------
// Rows back to images, gradients of gates and biases
// ---------------------------------------------------------------------------------

// out[t] = residual[t] + the sum of the image's rows, in the order of its slots.  Rows are float32, so that an answer is rounded once.
// 16000 images, two rows of 1024 and a residual each: 42 us for 197 MB (4.7 TB/s: what a copy reaches).
template <typename E>
__global__ __launch_bounds__(256) void k_combine(const float *rows, const int32_t *place, uint32_t images, uint32_t chosen, uint32_t cols,
                                                 const E *residual, uint64_t residual_stride, E *out, uint64_t out_stride)
{
    const uint64_t n = (uint64_t)blockIdx.x * 256 + threadIdx.x, stride = ((uint64_t)cols + 3) / 4 * 4;
    const uint64_t t = n / (stride / 4);
    const uint32_t c = (uint32_t)(n - t * (stride / 4)) * 4;
    if (t >= images) return;
    float v[4] = {0, 0, 0, 0};
    if (residual)
        for (uint32_t e = 0; e < 4; ++e)
            if (c + e < cols) v[e] = to_float(residual[t * residual_stride + c + e]);
    for (uint32_t s = 0; s < chosen; ++s)
        if (place[t * chosen + s] >= 0) {
            const v4f r = *(const v4f *)(rows + (t * chosen + s) * stride + c);
            for (int e = 0; e < 4; ++e) v[e] += r[e];
        }
    E *const to = out + t * out_stride + c;
    if (c + 4 <= cols) {
        store_four(to, v);
    } else {
        for (uint32_t e = 0; e < 4; ++e)
            if (c + e < cols) to[e] = from_float<E>(v[e]);
    }
}

// d gate of a slot = dy . (W2 f(a) + b2) = sum of its row's parts + dy . b2; a wave per slot.
template <typename E>
__global__ __launch_bounds__(256) void k_gate_gradients(const float *partial, uint32_t parts, const int32_t *place, const int32_t *owner,
                                                        uint64_t slots, uint32_t chosen, const E *dy, uint64_t dy_stride,
                                                        uint32_t cols, const E *bias, E *out)
{
    const uint64_t slot = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63;
    if (slot >= slots) return;
    const int32_t row = place[slot];
    float v = 0.0f;
    if (row >= 0) {
        for (uint32_t i = lane; i < parts; i += 64) v += partial[(uint64_t)row * parts + i];
        if (bias) {
            const uint64_t neuron = (uint32_t)owner[slot];
            const E *const d = dy + slot / chosen * dy_stride;
            for (uint32_t c = lane; c < cols; c += 64) v += to_float(d[c]) * to_float(bias[neuron * cols + c]);
        }
    }
    v = wave_sum(v);
    if (lane == 0) out[slot] = from_float<E>(v);
}

// ---------------------------------------------------------------------------------
// AdamW
// ---------------------------------------------------------------------------------

constexpr uint32_t kAdamTensors = 32, kAdamRuns = 2, kAdamChunk = 1024 * kAdamRuns;      // tensors of a launch (their table is a kernel argument), values of a block

struct AdamArgs {
    pink_hip_readout_tensor tensor[kAdamTensors];
    uint32_t first_block[kAdamTensors + 1];
    uint32_t count;
    float rate, beta1, rest1, beta2, rest2, c1, c2, epsilon;
};

__device__ __forceinline__ uint32_t adam_tensor(const AdamArgs &g)
{
    uint32_t i = 0;
    while (i + 1 < g.count && blockIdx.x >= g.first_block[i + 1]) ++i;
    return i;
}

// Four neighbours at their own alignment, those from `valid` on zero and not touched.
template <typename V> __device__ __forceinline__ void load_run(V (&v)[4], const V *at, uint32_t valid)
{
    if (valid >= 4) {
        __builtin_memcpy(v, at, sizeof v);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = i < valid ? at[i] : V{};
    }
}

template <typename V> __device__ __forceinline__ void store_run(V *at, const V (&v)[4], uint32_t valid)
{
    if (valid >= 4) {
        __builtin_memcpy(at, v, sizeof v);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (i < valid) at[i] = v[i];
    }
}

__device__ __forceinline__ float first_value(int8_t code, float scale)
{
    const float u = (float)code * (1.0f / 127);
    return (u * fabsf(u)) * scale;
}

__device__ __forceinline__ float second_value(uint8_t code, float scale)
{
    float u = (float)code * (1.0f / 255);
    u = u * u;
    return (u * u) * scale;
}

// A thread has kAdamRuns times four neighbouring values, 1024 apart, so that a wave's access is a run of memory and a block of 256
// codes belongs to a wave.  All that is read is asked for before anything is done with it.  The states follow by sums, products,
// roots and reciprocals that are each rounded (the codes are whole numbers and must not go by how they were computed).  The
// value's own step takes the hardware's root and reciprocal, each off by one unit at most: 2^-22 of a step.  They take subnormal
// numbers for 0, which is as little where epsilon is 2^-38 or more (the root of a subnormal number is below 2^-63).  Below that
// SMALL_EPSILON divides by what is rounded; so a step without a gradient is 0 at any epsilon.
// 224 M values, bfloat16 gradients and copies, 8-bit states: 726 us for 3.6 GB (4.9 TB/s; a copy reaches 4.8); with every root
// rounded it was 821 us and bound by the vector ALU (117 instructions a value, now 80).  44 M values, float32 states: 226 us, 5.4 TB/s.
template <bool CODES, bool SMALL_EPSILON> __global__ __launch_bounds__(256) void k_adamw(const AdamArgs g)
{
    const uint32_t which = adam_tensor(g);
    const pink_hip_readout_tensor &t = g.tensor[which];
    const uint64_t base = (uint64_t)(blockIdx.x - g.first_block[which]) * kAdamChunk + threadIdx.x * 4;

    float p[kAdamRuns][4], d[kAdamRuns][4], m[kAdamRuns][4], v[kAdamRuns][4];
    Bfloat half[kAdamRuns][4];
    int8_t mc[kAdamRuns][4];
    uint8_t vc[kAdamRuns][4];
    float ms[kAdamRuns], vs[kAdamRuns];
    uint32_t valid[kAdamRuns];
    const bool halves = t.gradient_element == PINK_HIP_ELEMENT_BFLOAT;
#pragma unroll
    for (uint32_t n = 0; n < kAdamRuns; ++n) {
        const uint64_t at = base + n * 1024;
        valid[n] = at >= t.size ? 0 : (uint32_t)min((uint64_t)4, t.size - at);
        load_run(p[n], t.value + at, valid[n]);
        if (halves) load_run(half[n], (const Bfloat *)t.gradient + at, valid[n]);
        else load_run(d[n], (const float *)t.gradient + at, valid[n]);
        if constexpr (CODES) {
            load_run(mc[n], (const int8_t *)t.first + at, valid[n]);
            load_run(vc[n], (const uint8_t *)t.second + at, valid[n]);
            ms[n] = valid[n] ? t.first_scale[at / kBlock8] : 0.0f;
            vs[n] = valid[n] ? t.second_scale[at / kBlock8] : 0.0f;
        } else {
            load_run(m[n], (const float *)t.first + at, valid[n]);
            load_run(v[n], (const float *)t.second + at, valid[n]);
        }
    }
#pragma unroll
    for (uint32_t n = 0; n < kAdamRuns; ++n) {
        const uint64_t at = base + n * 1024;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float grad = halves ? to_float(half[n][i]) : d[n][i];
            if constexpr (CODES) {
                m[n][i] = first_value(mc[n][i], ms[n]);
                v[n][i] = second_value(vc[n][i], vs[n]);
            }
            m[n][i] = m[n][i] * g.beta1 + grad * g.rest1;
            v[n][i] = v[n][i] * g.beta2 + (grad * grad) * g.rest2;
            const float step = SMALL_EPSILON ? (m[n][i] * g.c1) / (sqrtf(v[n][i] * g.c2) + g.epsilon)
                                             : (m[n][i] * g.c1) * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[n][i] * g.c2) + g.epsilon);
            p[n][i] = p[n][i] - (step + p[n][i] * t.decay) * g.rate;
        }
        store_run(t.value + at, p[n], valid[n]);
        if (t.rounded) {
            Bfloat b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = from_float<Bfloat>(p[n][i]);
            store_run((Bfloat *)t.rounded + at, b, valid[n]);
        }
        if constexpr (CODES) {
            // (values past the end are zero; magnitudes order as their bits do, and NaN is the largest)
            uint32_t bits_m = 0, bits_v = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bits_m = max(bits_m, __float_as_uint(fabsf(m[n][i])));
                bits_v = max(bits_v, __float_as_uint(fabsf(v[n][i])));
            }
            float most_m = __uint_as_float(wave_max_u32(bits_m)), most_v = __uint_as_float(wave_max_u32(bits_v));
            most_m = most_m < 1.175494351e-38f ? 0.0f : most_m;
            most_v = most_v < 1.175494351e-38f ? 0.0f : most_v;
            const float mi = most_m > 0.0f ? 1.0f / most_m : 0.0f, vi = most_v > 0.0f ? 1.0f / most_v : 0.0f;
            // Codes are defined by rounded roots.  The hardware's are one unit off at most, which moves 127 sqrt(x) by less than 5e-5 and
            // 255 sqrt(sqrt(x)) by less than 1e-4: only values that close to halfway between two codes need the rounded ones
            // (8 of 100 runs, against 16 instructions for each of three roots).
            float ratio_m[4], ratio_v[4], code_m[4], code_v[4];
            bool close = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                ratio_m[i] = fabsf(m[n][i]) * mi;
                ratio_v[i] = fabsf(v[n][i]) * vi;
                const float root_m = __builtin_amdgcn_sqrtf(ratio_m[i]) * 127.0f;
                const float root_v = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(ratio_v[i])) * 255.0f;
                code_m[i] = rintf(root_m);
                code_v[i] = rintf(root_v);
                close = close || !(fabsf(root_m - code_m[i]) <= 0.5f - 5e-5f && fabsf(root_v - code_v[i]) <= 0.5f - 1e-4f);
            }
            if (close) {                                   // (and NaN: code 0 of a scale that is not finite is NaN again)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    code_m[i] = ratio_m[i] >= 0.0f ? rintf(sqrtf(ratio_m[i]) * 127.0f) : 0.0f;
                    code_v[i] = ratio_v[i] >= 0.0f ? rintf(sqrtf(sqrtf(ratio_v[i])) * 255.0f) : 0.0f;
                }
            }
            int8_t mo[4];
            uint8_t vo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mo[i] = (int8_t)(int)copysignf(code_m[i], m[n][i]);
                vo[i] = (uint8_t)(int)(ratio_v[i] > 0.0f ? fmaxf(code_v[i], 1.0f) : code_v[i]);
            }
            store_run((int8_t *)t.first + at, mo, valid[n]);
            store_run((uint8_t *)t.second + at, vo, valid[n]);
            if (valid[n] && (threadIdx.x & 63) == 0) {
                t.first_scale[at / kBlock8] = most_m;
                t.second_scale[at / kBlock8] = most_v;
            }
        } else {
            store_run((float *)t.first + at, m[n], valid[n]);
            store_run((float *)t.second + at, v[n], valid[n]);
        }
    }
}

// 224 M values: 490 us for 2.3 GB (4.6 TB/s).
__global__ __launch_bounds__(256) void k_unpack(const AdamArgs g)
{
    const uint32_t which = adam_tensor(g);
    const pink_hip_readout_tensor &t = g.tensor[which];
    const uint64_t base = (uint64_t)(blockIdx.x - g.first_block[which]) * kAdamChunk + threadIdx.x * 4;
    int8_t mc[kAdamRuns][4];
    uint8_t vc[kAdamRuns][4];
    float ms[kAdamRuns], vs[kAdamRuns];
    uint32_t valid[kAdamRuns];
#pragma unroll
    for (uint32_t n = 0; n < kAdamRuns; ++n) {
        const uint64_t at = base + n * 1024;
        valid[n] = at >= t.size ? 0 : (uint32_t)min((uint64_t)4, t.size - at);
        load_run(mc[n], (const int8_t *)t.first + at, valid[n]);
        load_run(vc[n], (const uint8_t *)t.second + at, valid[n]);
        ms[n] = valid[n] ? t.first_scale[at / kBlock8] : 0.0f;
        vs[n] = valid[n] ? t.second_scale[at / kBlock8] : 0.0f;
    }
#pragma unroll
    for (uint32_t n = 0; n < kAdamRuns; ++n) {
        float m[4], v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            m[i] = first_value(mc[n][i], ms[n]);
            v[i] = second_value(vc[n][i], vs[n]);
        }
        store_run(t.first_values + base + n * 1024, m, valid[n]);
        store_run(t.second_values + base + n * 1024, v, valid[n]);
    }
}

// ---------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------

uint32_t group_size(const pink_hip_readout_config &c) { return (c.neurons + c.groups - 1) / c.groups; }

// What a forward call leaves for the backward one, and where.
struct Saved {
    size_t order, owner, place, offsets, tile_count, tiles, before, after, bytes;
    uint64_t stride;               // of before's and after's rows: whole 16-byte chunks
};

constexpr uint32_t kLeastTileRows = 16, kFewSlots = 512;

Saved saved_layout(const pink_hip_readout *r, uint64_t images)
{
    const pink_hip_readout_config &c = r->cfg;
    const size_t e = element_bytes(r), slots = images * c.chosen;
    Saved s;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    s.stride = (c.hidden + 16 / e - 1) / (16 / e) * (16 / e);
    s.order = take(slots * 4);
    s.owner = take(slots * 4);
    s.place = take(slots * 4);
    s.offsets = take(((size_t)c.neurons + 1) * 4);
    s.tile_count = take(4);
    s.tiles = take((slots / kLeastTileRows + std::min<size_t>(c.neurons, slots)) * sizeof(uint2));
    s.after = take(slots * s.stride * e);
    s.before = take(slots * s.stride * e);
    s.bytes = at;
    return s;
}

uint32_t plan_waves(uint32_t neurons) { return std::max(1u, std::min(16u, 32768u / neurons)); }

// Floats between rows of products that images are summed up from: whole chunks.
uint64_t whole_rows(uint32_t cols) { return ((uint64_t)cols + 3) / 4 * 4; }

struct Work {
    size_t counts, totals, rows, partial, few, saved, bytes;
};

// `saved`: bytes in the place of a caller's buffer (forward calls that keep nothing) or of gradients of `before`.
Work work_layout(const pink_hip_readout *r, uint64_t images, size_t saved)
{
    const pink_hip_readout_config &c = r->cfg;
    const size_t slots = images * c.chosen, plan_blocks = slots / (plan_waves(c.neurons) * 64) + 1;
    Work w;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += align256(bytes);
        return here;
    };
    w.counts = take(plan_blocks * c.neurons * 4);
    w.totals = take((size_t)c.neurons * 4);
    w.rows = take(c.chosen > 1 ? slots * whole_rows(std::max(c.features, c.outputs)) * 4 : 0);       // (one neuron's go straight to the image)
    w.partial = take(slots * ((c.hidden + 31) / 32) * 4);
    w.few = take(std::min<size_t>(slots, kFewSlots) * c.hidden * 4);
    w.saved = take(saved);
    w.bytes = at;
    return w;
}

int check(const pink_hip_readout_config *c, pink_hip_readout *r)
{
    REFUSE(r, !c, "pink_hip_readout: null argument");
    REFUSE(r, c->neurons == 0 || c->neurons > kMaxNeurons, "Number of neurons must be between 1 and 32768");
    REFUSE(r, c->chosen == 0 || c->chosen > kMaxChosen || c->chosen > c->neurons, "Number of chosen neurons must be between 1 and 64 and not larger than the number of neurons");
    REFUSE(r, c->score > PINK_HIP_SCORE_SIGMOID, "unknown score");
    REFUSE(r, c->renormalise > 1, "renormalise must be 0 or 1");
    REFUSE(r, c->groups == 0 || c->groups > kMaxGroups || c->groups > c->neurons, "Number of groups must be between 1 and 1024 and not larger than the number of neurons");
    REFUSE(r, (uint64_t)(c->groups - 1) * group_size(*c) >= c->neurons, "Number of groups leaves a group without neurons");
    REFUSE(r, c->groups_kept == 0 || c->groups_kept > c->groups, "Number of kept groups must be between 1 and the number of groups");
    REFUSE(r, c->activation > PINK_HIP_SILU, "unknown activation");
    REFUSE(r, c->element > PINK_HIP_ELEMENT_BFLOAT, "unknown element type");
    const bool models = c->features || c->hidden || c->outputs;
    REFUSE(r, models && (!c->features || !c->hidden || !c->outputs), "features, hidden and outputs must be all zero or none");
    REFUSE(r, c->features > kMaxSize || c->hidden > kMaxSize || c->outputs > kMaxSize, "features, hidden and outputs must be at most 1048576");
    return PINK_HIP_OK;
}

RouteArgs route_args(const pink_hip_readout *r, const float *distances, uint32_t images, uint64_t stride, const float *sharpness,
                     const float *radius, const float *bias)
{
    const pink_hip_readout_config &c = r->cfg;
    RouteArgs g = {};
    g.distances = distances;
    g.stride = stride ? stride : c.neurons;
    g.sharpness = sharpness;
    g.radius = radius;
    g.bias = bias;
    g.images = images;
    g.neurons = c.neurons;
    g.chosen = c.chosen;
    g.groups = c.groups;
    g.groups_kept = c.groups_kept;
    g.group_size = group_size(c);
    g.sigmoid = c.score == PINK_HIP_SCORE_SIGMOID;
    g.renormalise = c.renormalise;
    return g;
}

// Rows of a product's tiles, by how many rows a neuron has on average: the weights are read once for each tile of rows, and a tile
// that is mostly empty multiplies for nothing.  Measured forward (us): tiles of 16 / 64 rows, bfloat16 1024 x 512 x 1024 of 100 neurons,
// 12 rows a neuron 70 / 72, 24 rows 93 / 78; float32 2025 x 200 x 45 of 331 neurons, 12 rows 171 / 284, 24 rows 238 / 288, 36 rows 313 / 290.
// Tiles of 64 / 128 rows, bfloat16, 36 rows 83 / 85, 64 rows 103 / 94, 96 rows 128 / 99; float32's stay ahead in 64 past that bound
// (64 rows 377 / 638, 160 rows 728 / 941; training 1269 / 1560 and 2446 / 2544).  bfloat16's largest tiles halve what a CU fetches for
// each product; measured with 640 rows a neuron, 1936 x 1024: 475 us in tiles of 256 x 256 against 550 in 128 x 128; with 320 rows,
// 512 x 1024: 84 against 95, and 102 against 99 for 1024 x 512.
uint32_t tile_rows(const pink_hip_readout *r, uint64_t slots)
{
    const uint64_t neurons = std::min<uint64_t>(r->cfg.neurons, slots);
    if (slots <= 24 * neurons) return 16;
    if (slots <= 64 * neurons) return 64;
    return slots >= 256 * neurons && r->cfg.element == PINK_HIP_ELEMENT_BFLOAT ? 256 : 128;
}

// Are the operands whole chunks at their alignment?  (`saved` and the workspace have both; what lies past a row's end there is
// readable.)
template <typename E, int OP> bool is_direct(const ProductArgs &g)
{
    constexpr uint32_t per = 16 / sizeof(E);
    const auto whole = [](const void *at, uint64_t stride) { return ((uintptr_t)at & 15) == 0 && stride % per == 0; };
    bool direct = whole(g.p, g.p_stride) && whole(g.q, g.q_stride);
    if (OP == kHidden || OP == kAnswer || OP == kBackHidden || OP == kBackInput) direct = direct && g.q_matrix % per == 0;
    if (OP == kHidden || OP == kAnswer) direct = direct && g.depth % per == 0;
    if (OP == kBackHidden) direct = direct && g.depth % per == 0 && g.cols % per == 0;
    if (OP == kBackInput) direct = direct && g.cols % per == 0;          // (its rows are padded with zeros)
    if (OP == kGradFirst) direct = direct && g.cols % per == 0;
    if (OP == kGradSecond) direct = direct && g.rows % per == 0;
    return direct;
}

template <typename E, int OP, int PR, int QC, int PW, int QW, int M, int DEEP, bool DIRECT>
int product_of_tile(pink_hip_readout *r, ProductArgs &g, uint64_t slots)
{
    constexpr bool grad = OP == kGradFirst || OP == kGradSecond;
    g.col_tiles = grad && !g.out ? 1 : (g.cols + QC - 1) / QC;
    g.row_tiles = grad ? (g.rows + PR - 1) / PR : 0;
    const uint64_t tiles = grad ? (uint64_t)r->cfg.neurons * g.row_tiles : slots / PR + std::min<uint64_t>(r->cfg.neurons, slots);
    const uint64_t blocks = tiles * g.col_tiles;
    REFUSE(r, too_many(blocks + kFillBlocks, 64 * PW * QW), "too many images for one call");
    g.slots = (uint32_t)slots;
    const uint32_t more = (OP == kAnswer || OP == kBackInput) && g.place ? kFillBlocks : 0;
    k_product<E, OP, PR, QC, PW, QW, M, DEEP, DIRECT><<<(uint32_t)blocks + more, 64 * PW * QW, 0, r->stream>>>(g);
    return launched(r, "k_product");
}

template <typename E, int OP, bool DIRECT> int product_as(pink_hip_readout *r, ProductArgs &g, uint64_t slots)
{
    constexpr bool half = sizeof(E) == 2;
    if constexpr (OP == kGradFirst || OP == kGradSecond) {
        // Matrices of few rows (the second layer of a handful of outputs): tiles of as few.
        if (g.rows <= 32) return product_of_tile<E, OP, 32, 128, 1, 4, 32, 1, DIRECT>(r, g, slots);
        // Few rows a neuron: writing the gradients is what there is to do, and small tiles spread it over more blocks.  A training step in small /
        // large tiles (us): float32 784 x 96 x 40 of 64 neurons, 16 rows a neuron 61 / 68, 64 rows 112 / 130; where large tiles are many
        // they are ahead at any number of rows, which the rule does not go by (bfloat16 1936 x 1024 x 256 of 100, 16 rows 467 / 441, 64 rows
        // 612 / 583).  The largest tiles (590 against 640 us for 1024 x 1936 of 100 neurons) where there are enough of them to go round.
        if (slots <= 64 * (uint64_t)r->cfg.neurons) return product_of_tile<E, OP, 64, 64, 2, 2, 16, 1, DIRECT>(r, g, slots);
        if constexpr (half && DIRECT) {
            const uint64_t tiles = (uint64_t)r->cfg.neurons * ((g.rows + 255) / 256) * ((g.cols + 255) / 256);
            if (g.out && g.rows >= 256 && tiles >= 1024) return product_of_tile<E, OP, 256, 256, 2, 4, 32, 1, DIRECT>(r, g, slots);
        }
        return product_of_tile<E, OP, 128, 128, 2, 2, 32, 1, DIRECT>(r, g, slots);
    } else {
        // Few rows a neuron: reading the weights is what there is to do; a stage takes 512 bytes of a row so that enough of it is
        // under way.
        const uint32_t rows = tile_rows(r, slots);
        if (rows > 16 && g.cols <= 32) {                   // results of few columns: tiles of as few
            if (rows == 64) return product_of_tile<E, OP, 64, 32, 2, 1, 32, 2, DIRECT>(r, g, slots);
            if (rows == 128) return product_of_tile<E, OP, 128, 32, 4, 1, 32, 1, DIRECT>(r, g, slots);
            return product_of_tile<E, OP, 256, 32, 4, 1, 32, 1, DIRECT>(r, g, slots);
        }
        switch (rows) {
        case 16:                                           // (short sums, as the backward pass has: more blocks at once instead)
            if constexpr (OP == kBackHidden || OP == kBackInput) return product_of_tile<E, OP, 16, 64, 1, 4, 16, 2, DIRECT>(r, g, slots);
            else return product_of_tile<E, OP, 16, 32, 1, 2, 16, 4, DIRECT>(r, g, slots);
        case 64: return product_of_tile<E, OP, 64, 64, 2, 2, 32, 2, DIRECT>(r, g, slots);
        case 256:                                          // (what passes through registers leaves fewer for sums)
            if constexpr (half && DIRECT) return product_of_tile<E, OP, 256, 256, 2, 4, 32, 1, DIRECT>(r, g, slots);
            else if constexpr (half) return product_of_tile<E, OP, 256, 128, 4, 2, 32, 1, DIRECT>(r, g, slots);
            [[fallthrough]];
        default: return product_of_tile<E, OP, 128, 128, 2, 2, 32, 1, DIRECT>(r, g, slots);
        }
    }
}

template <typename E, int OP> int product(pink_hip_readout *r, ProductArgs &g, uint64_t slots)
{
    return is_direct<E, OP>(g) ? product_as<E, OP, true>(r, g, slots) : product_as<E, OP, false>(r, g, slots);
}

int plan(pink_hip_readout *r, const int32_t *neuron, uint32_t slots, char *saved, const Saved &s, const Work &w)
{
    const pink_hip_readout_config &c = r->cfg;
    char *const work = (char *)r->work;
    PlanArgs g = {};
    g.neuron = neuron;
    g.slots = slots;
    g.neurons = c.neurons;
    g.tile_rows = tile_rows(r, slots);
    g.counts = (uint32_t *)(work + w.counts);
    g.order = (uint32_t *)(saved + s.order);
    g.owner = (int32_t *)(saved + s.owner);
    g.place = (int32_t *)(saved + s.place);
    g.offsets = (uint32_t *)(saved + s.offsets);
    g.tile_count = (uint32_t *)(saved + s.tile_count);
    g.tiles = (uint2 *)(saved + s.tiles);
    const uint32_t waves = plan_waves(c.neurons), per_block = waves * 64, blocks = (slots + per_block - 1) / per_block;
    const size_t lds = (size_t)waves * c.neurons * 4;
    if (blocks <= kPerWave<2>) {
        // as many waves as there are slots for, or a thread for each neuron
        const uint32_t with_slots = (slots + 64 * kPerWave<2> - 1) / (64 * kPerWave<2>), all = std::min(16u, std::max(with_slots, (c.neurons + 63) / 64));
        k_plan<2><<<1, all * 64, (size_t)with_slots * c.neurons * 4, r->stream>>>(g);
        return launched(r, "k_plan");
    }
    k_plan<0><<<blocks, waves * 64, lds, r->stream>>>(g);
    TRY(launched(r, "k_plan"));
    k_plan_offsets<<<1, 1024, 0, r->stream>>>(g, blocks, (uint32_t *)(work + w.totals));
    TRY(launched(r, "k_plan_offsets"));
    k_plan<1><<<blocks, waves * 64, lds, r->stream>>>(g);
    return launched(r, "k_plan");
}

template <typename E>
int combine(pink_hip_readout *r, const float *rows, const int32_t *place, uint32_t images, uint32_t cols, const void *residual,
            uint64_t residual_stride, void *out, uint64_t out_stride)
{
    const uint64_t blocks = (images * (whole_rows(cols) / 4) + 255) / 256;
    REFUSE(r, too_many(blocks, 256), "too many images for one call");
    k_combine<E><<<(uint32_t)blocks, 256, 0, r->stream>>>(rows, place, images, r->cfg.chosen, cols, (const E *)residual, residual_stride, (E *)out, out_stride);
    return launched(r, "k_combine");
}

// Slots by themselves read their neuron's weights each, tiles once for a neuron; sorting and tiles cost some 10 us.  Measured (us, slots by
// themselves / tiles): 100 neurons of 1.1 MB, bfloat16, 64 slots 13.5 / 21, 512 slots 34 / 28; of 4.5 MB, 64 slots 51 / 54, 128 slots
// 87 / 72; 331 neurons of 1.7 MB, float32, 64 slots 26 / 51, 256 slots 73 / 90, 512 slots 130 / 119.
bool is_few(const pink_hip_readout *r, uint64_t slots)
{
    const pink_hip_readout_config &c = r->cfg;
    const uint64_t bytes = ((uint64_t)c.features + c.outputs) * c.hidden * element_bytes(r);
    return slots <= 64 || (slots <= kFewSlots && (4 * slots <= 3 * (uint64_t)c.neurons || slots * bytes <= 64u << 20));
}

template <typename E>
int experts(pink_hip_readout *r, const void *x, uint32_t images, uint64_t x_stride, const int32_t *neuron, const float *gates,
            const pink_hip_readout_weights &weights, const void *residual, uint64_t residual_stride, void *y, uint64_t y_stride, void *keep)
{
    const pink_hip_readout_config &c = r->cfg;
    const Saved s = saved_layout(r, images);
    const Work w = work_layout(r, images, keep ? 0 : s.bytes);
    TRY(grow(r, w.bytes));
    char *const work = (char *)r->work, *const saved = keep ? (char *)keep : work + w.saved;
    const uint32_t slots = images * c.chosen;
    if (!keep && is_few(r, slots)) {
        const FewArgs f = {x, x_stride, neuron, gates, weights.first, weights.first_bias, weights.second, weights.second_bias, residual,
                           residual_stride, y_stride, c.neurons, c.chosen, c.features, c.hidden, c.outputs, c.activation,
                           (float *)(work + w.few), y};
        constexpr uint32_t rows = 4 * kFewRows;
        k_few_hidden<E><<<dim3((c.hidden + rows - 1) / rows, slots), 256, 0, r->stream>>>(f);
        TRY(launched(r, "k_few_hidden"));
        k_few_answer<E><<<dim3((c.outputs + rows - 1) / rows, images), 256, 0, r->stream>>>(f);
        return launched(r, "k_few_answer");
    }
    TRY(plan(r, neuron, slots, saved, s, w));

    ProductArgs g = {};
    g.order = (const uint32_t *)(saved + s.order);
    g.offsets = (const uint32_t *)(saved + s.offsets);
    g.tiles = (const uint2 *)(saved + s.tiles);
    g.tile_count = (const uint32_t *)(saved + s.tile_count);
    g.chosen = c.chosen;
    g.activation = c.activation;
    g.gates = gates;
    g.p = x;
    g.p_stride = x_stride;
    g.q = weights.first;
    g.q_stride = c.features;
    g.q_matrix = (uint64_t)c.hidden * c.features;
    g.depth = c.features;
    g.cols = c.hidden;
    g.bias = weights.first_bias;
    g.out = keep ? saved + s.before : nullptr;
    g.out_after = saved + s.after;
    g.out_stride = s.stride;
    TRY((product<E, kHidden>(r, g, slots)));
    g.p = saved + s.after;
    g.p_stride = s.stride;
    g.q = weights.second;
    g.q_stride = c.hidden;
    g.q_matrix = (uint64_t)c.outputs * c.hidden;
    g.depth = c.hidden;
    g.cols = c.outputs;
    g.bias = weights.second_bias;
    if (c.chosen == 1) {
        g.place = (const int32_t *)(saved + s.place);
        g.residual = residual;
        g.residual_stride = residual_stride;
        g.out = y;
        g.out_stride = y_stride;
        return product<E, kAnswer>(r, g, slots);
    }
    g.out = work + w.rows;
    g.out_stride = whole_rows(c.outputs);
    TRY((product<E, kAnswer>(r, g, slots)));
    return combine<E>(r, (const float *)(work + w.rows), (const int32_t *)(saved + s.place), images, c.outputs, residual, residual_stride, y, y_stride);
}

template <typename E>
int experts_backward(pink_hip_readout *r, const void *x, uint32_t images, uint64_t x_stride, const float *gates,
                     const pink_hip_readout_weights &weights, const void *keep, const void *dy, uint64_t dy_stride,
                     const pink_hip_readout_gradients &out, uint64_t dx_stride)
{
    const pink_hip_readout_config &c = r->cfg;
    const Saved s = saved_layout(r, images);
    const uint32_t slots = images * c.chosen;
    const Work w = work_layout(r, images, slots * s.stride * element_bytes(r));
    TRY(grow(r, w.bytes));
    char *const work = (char *)r->work;
    const char *const saved = (const char *)keep;
    const int32_t *const place = (const int32_t *)(saved + s.place);
    void *const dbefore = work + w.saved;                  // slots x stride

    ProductArgs g = {};
    g.order = (const uint32_t *)(saved + s.order);
    g.offsets = (const uint32_t *)(saved + s.offsets);
    g.tiles = (const uint2 *)(saved + s.tiles);
    g.tile_count = (const uint32_t *)(saved + s.tile_count);
    g.chosen = c.chosen;
    g.activation = c.activation;
    g.gates = gates;
    if (out.gates || out.features || out.first || out.first_bias) {
        g.p = dy;
        g.p_stride = dy_stride;
        g.q = weights.second;
        g.q_stride = c.hidden;
        g.q_matrix = (uint64_t)c.outputs * c.hidden;
        g.depth = c.outputs;
        g.cols = c.hidden;
        g.before = saved + s.before;
        g.after = saved + s.after;
        g.out = dbefore;
        g.out_stride = s.stride;
        g.partial = (float *)(work + w.partial);
        TRY((product<E, kBackHidden>(r, g, slots)));
    }
    if (out.gates) {
        REFUSE(r, too_many(((uint64_t)slots + 3) / 4, 256), "too many images for one call");
        k_gate_gradients<E><<<(uint32_t)(((uint64_t)slots + 3) / 4), 256, 0, r->stream>>>(
            g.partial, g.col_tiles, place, (const int32_t *)(saved + s.owner), slots, c.chosen, (const E *)dy, dy_stride, c.outputs,
            (const E *)weights.second_bias, (E *)out.gates);
        TRY(launched(r, "k_gate_gradients"));
    }
    if (out.features) {
        g.p = dbefore;
        g.p_stride = s.stride;
        g.q = weights.first;
        g.q_stride = c.features;
        g.q_matrix = (uint64_t)c.hidden * c.features;
        g.depth = c.hidden;
        g.cols = c.features;
        if (c.chosen == 1) {
            g.place = place;
            g.out = out.features;
            g.out_stride = dx_stride;
            TRY((product<E, kBackInput>(r, g, slots)));
        } else {
            g.out = work + w.rows;
            g.out_stride = whole_rows(c.features);
            TRY((product<E, kBackInput>(r, g, slots)));
            TRY(combine<E>(r, (const float *)(work + w.rows), place, images, c.features, nullptr, 0, out.features, dx_stride));
        }
    }
    if (out.first || out.first_bias) {
        g.p = dbefore;
        g.p_stride = s.stride;
        g.q = x;
        g.q_stride = x_stride;
        g.rows = c.hidden;
        g.cols = c.features;
        g.out = out.first;
        g.out_bias = out.first_bias;
        g.out_stride = c.features;
        TRY((product<E, kGradFirst>(r, g, slots)));
    }
    if (out.second || out.second_bias) {
        g.p = dy;
        g.p_stride = dy_stride;
        g.q = saved + s.after;
        g.q_stride = s.stride;
        g.rows = c.outputs;
        g.cols = c.hidden;
        g.out = out.second;
        g.out_bias = out.second_bias;
        g.out_stride = c.hidden;
        TRY((product<E, kGradSecond>(r, g, slots)));
    }
    return PINK_HIP_OK;
}

// Slots of a call are counted in 31 bits.
int check_images(pink_hip_readout *r, uint32_t images)
{
    REFUSE(r, (uint64_t)images * r->cfg.chosen > 0x7fffffffu, "too many images for one call");
    return PINK_HIP_OK;
}

// Tensors in launches of at most kAdamTensors.
template <typename Check, typename Launch>
int over_tensors(pink_hip_readout *r, const pink_hip_readout_tensor *tensors, uint32_t count, AdamArgs &g, const Check &ok, const Launch &launch)
{
    for (uint32_t i = 0; i < count; ++i)
        if (tensors[i].size) {
            TRY(ok(tensors[i]));
            REFUSE(r, too_many((tensors[i].size + kAdamChunk - 1) / kAdamChunk, 256), "too many values in one tensor");
        }
    uint64_t blocks = 0;
    g.count = 0;
    for (uint32_t i = 0; i <= count; ++i) {
        const uint64_t more = i < count ? (tensors[i].size + kAdamChunk - 1) / kAdamChunk : 0;
        if (g.count && (i == count || g.count == kAdamTensors || too_many(blocks + more, 256))) {
            g.first_block[g.count] = (uint32_t)blocks;
            launch((uint32_t)blocks);
            TRY(launched(r, "k_adamw"));
            g.count = 0;
            blocks = 0;
        }
        if (!more) continue;
        g.tensor[g.count] = tensors[i];
        g.first_block[g.count++] = (uint32_t)blocks;
        blocks += more;
    }
    return PINK_HIP_OK;
}

}  // namespace

extern "C" {

const char *pink_hip_readout_last_error(const pink_hip_readout *r) { return r ? r->err : g_readout_error; }

int pink_hip_readout_check(const pink_hip_readout_config *cfg) { return check(cfg, nullptr); }

int pink_hip_readout_create(pink_hip_readout **out, const pink_hip_readout_config *cfg)
{
    if (!out) return fail(nullptr, PINK_HIP_EINVAL, "pink_hip_readout_create: null argument");
    *out = nullptr;
    TRY(check(cfg, nullptr));
    HIP_TRY(nullptr, hipSetDevice(cfg->device));
    // the forms whose LDS goes by the number of neurons
    const int lds = (int)(kMaxNeurons * 4 + kMaxGroups * 4);
    HIP_TRY(nullptr, hipFuncSetAttribute((const void *)k_route_block, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    HIP_TRY(nullptr, hipFuncSetAttribute((const void *)k_balance, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    HIP_TRY(nullptr, hipFuncSetAttribute((const void *)k_plan<0>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    HIP_TRY(nullptr, hipFuncSetAttribute((const void *)k_plan<1>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    HIP_TRY(nullptr, hipFuncSetAttribute((const void *)k_plan<2>, hipFuncAttributeMaxDynamicSharedMemorySize, lds));
    pink_hip_readout *r = new (std::nothrow) pink_hip_readout();
    if (!r) return fail(nullptr, PINK_HIP_ENOMEM, "pink_hip_readout_create: out of memory");
    r->cfg = *cfg;
    const hipError_t e = hipStreamCreateWithFlags(&r->own, hipStreamNonBlocking);
    if (e != hipSuccess) {
        delete r;
        return fail(nullptr, PINK_HIP_EDEVICE, "hipStreamCreateWithFlags", hipGetErrorString(e));
    }
    r->stream = r->own;
    *out = r;
    return PINK_HIP_OK;
}

void pink_hip_readout_destroy(pink_hip_readout *r)
{
    if (!r) return;
    (void)hipSetDevice(r->cfg.device);
    if (r->stream != r->own) (void)hipStreamSynchronize(r->stream);
    (void)hipStreamSynchronize(r->own);
    if (r->work) (void)hipFree(r->work);
    while (Former *const kept = r->former) {
        (void)hipFree(kept->work);
        r->former = kept->next;
        delete kept;
    }
    (void)hipStreamDestroy(r->own);
    delete r;
}

int pink_hip_readout_set_stream(pink_hip_readout *r, void *hip_stream)
{
    if (!r) return PINK_HIP_EINVAL;
    const hipStream_t next = hip_stream == PINK_HIP_OWN_STREAM ? r->own : (hipStream_t)hip_stream;
    if (next == r->stream) return PINK_HIP_OK;
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    HIP_TRY(r, hipStreamSynchronize(r->stream));           // the workspace is one stream's at a time
    r->stream = next;
    return PINK_HIP_OK;
}

int pink_hip_readout_synchronize(pink_hip_readout *r)
{
    if (!r) return PINK_HIP_EINVAL;
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    HIP_TRY(r, hipStreamSynchronize(r->stream));
    return PINK_HIP_OK;
}

int pink_hip_readout_route(pink_hip_readout *r, const float *distances, uint32_t images, uint64_t stride, const float *sharpness,
                           const float *radius, const float *bias, int32_t *neuron, float *gates)
{
    if (!r) return PINK_HIP_EINVAL;
    if (images == 0) return PINK_HIP_OK;
    REFUSE(r, !distances || !sharpness || !radius || !neuron || !gates, "pink_hip_readout_route: null argument");
    REFUSE(r, stride && stride < r->cfg.neurons, "pink_hip_readout_route: rows of distances overlap");
    TRY(check_images(r, images));
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    RouteArgs g = route_args(r, distances, images, stride, sharpness, radius, bias);
    g.neuron = neuron;
    g.gates = gates;
    const uint32_t candidates = std::max(g.neurons, g.groups_kept * g.group_size);
    const bool by_block = candidates > 2048 || g.groups > 64;
    REFUSE(r, too_many(by_block ? images : (images + 3) / 4, 256), "too many images for one call");
    if (by_block) {
        k_route_block<<<images, 256, (g.neurons + (g.groups > 1 ? g.groups : 0)) * 4, r->stream>>>(g);
        return launched(r, "k_route_block");
    }
    const uint32_t lds = g.groups > 1 ? 4 * (g.groups * (g.group_size | 1) + 64) * 4 : 0, blocks = (images + 3) / 4;
    const uint32_t over_size = g.groups > 1 ? (uint32_t)((1ull << 32) / g.group_size + 1) : 0;
    // Registers for every 64 neurons; with groups the candidates are fewer, and where 8 registers hold them that is
    // what taking them out of 16000 x 1600 distances in 8 of 40 groups goes through.
    const bool few = g.groups > 1 && g.groups_kept * g.group_size <= 512;
    const auto run = [&](auto j) {
        constexpr int J = decltype(j)::value;
        constexpr int C = J < 8 ? J : 8;
        const bool full = !g.renormalise && !g.sigmoid;
        if (few && full) k_route_wave<J, C, true><<<blocks, 256, lds, r->stream>>>(g, over_size);
        else if (few) k_route_wave<J, C, false><<<blocks, 256, lds, r->stream>>>(g, over_size);
        else if (full) k_route_wave<J, J, true><<<blocks, 256, lds, r->stream>>>(g, over_size);
        else k_route_wave<J, J, false><<<blocks, 256, lds, r->stream>>>(g, over_size);
    };
    const uint32_t registers = (candidates + 63) / 64;
    if (registers <= 2) run(std::integral_constant<int, 2>());
    else if (registers <= 4) run(std::integral_constant<int, 4>());
    else if (registers <= 6) run(std::integral_constant<int, 6>());
    else if (registers <= 8) run(std::integral_constant<int, 8>());
    else if (registers <= 12) run(std::integral_constant<int, 12>());
    else if (registers <= 16) run(std::integral_constant<int, 16>());
    else if (registers <= 20) run(std::integral_constant<int, 20>());
    else if (registers <= 24) run(std::integral_constant<int, 24>());
    else if (registers <= 28) run(std::integral_constant<int, 28>());
    else run(std::integral_constant<int, 32>());
    return launched(r, "k_route_wave");
}

int pink_hip_readout_route_backward(pink_hip_readout *r, const float *distances, uint32_t images, uint64_t stride, const float *sharpness,
                                    const float *radius, const float *bias, const int32_t *neuron, const float *gates,
                                    const void *gate_gradients, float *ddistances, float *dsharpness, float *dradius)
{
    if (!r) return PINK_HIP_EINVAL;
    const uint32_t neurons = r->cfg.neurons;
    REFUSE(r, images && (!distances || !sharpness || !radius || !neuron || !gates || !gate_gradients), "pink_hip_readout_route_backward: null argument");
    REFUSE(r, stride && stride < neurons, "pink_hip_readout_route_backward: rows of distances overlap");
    TRY(check_images(r, images));
    if (!ddistances && !dsharpness && !dradius) return PINK_HIP_OK;
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    RouteBackwardArgs a = {};
    a.r = route_args(r, distances, images, stride, sharpness, radius, bias);
    a.r.neuron = const_cast<int32_t *>(neuron);
    a.r.gates = const_cast<float *>(gates);
    a.gate_gradients = gate_gradients;
    a.distance_gradients = ddistances;
    a.want_sums = dsharpness || dradius;
    a.chunk = std::max(4u, std::min(kChunkMost, images / 256));
    a.chunk = std::max(a.chunk, (images + 65534) / 65535);               // (the grid's second dimension)
    REFUSE(r, a.chunk > kChunkMost, "too many images for one call");
    const uint32_t chunks = (images + a.chunk - 1) / a.chunk;
    TRY(grow(r, std::max<size_t>(1, (size_t)chunks * neurons * 8)));
    a.sharpness_part = (float *)r->work;
    a.radius_part = a.sharpness_part + (size_t)chunks * neurons;
    if (images) {
        const dim3 grid((neurons + 255) / 256, chunks);
        const size_t lds = (size_t)a.chunk * a.r.chosen * 8;
        if (r->cfg.element == PINK_HIP_ELEMENT_BFLOAT) k_route_backward<Bfloat><<<grid, 256, lds, r->stream>>>(a);
        else k_route_backward<float><<<grid, 256, lds, r->stream>>>(a);
        TRY(launched(r, "k_route_backward"));
    }
    if (!a.want_sums) return PINK_HIP_OK;
    k_route_sums<<<(neurons + 63) / 64, 1024, 0, r->stream>>>(a.sharpness_part, a.radius_part, chunks, neurons, dsharpness, dradius);
    return launched(r, "k_route_sums");
}

int pink_hip_readout_balance(pink_hip_readout *r, const int32_t *neuron, uint32_t images, float rate, float *bias, int32_t *load)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, (images && !neuron) || !bias, "pink_hip_readout_balance: null argument");
    TRY(check_images(r, images));
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    k_balance<<<1, 1024, r->cfg.neurons * 4, r->stream>>>(neuron, (uint64_t)images * r->cfg.chosen, r->cfg.neurons, rate, bias, load);
    return launched(r, "k_balance");
}

int pink_hip_readout_reserve(pink_hip_readout *r, uint32_t images)
{
    if (!r) return PINK_HIP_EINVAL;
    TRY(check_images(r, images));
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    const size_t parts = ((size_t)images / 4 + 1) * r->cfg.neurons * 8;
    return grow(r, std::max(parts, r->cfg.features ? work_layout(r, images, saved_layout(r, images).bytes).bytes : 0));
}

size_t pink_hip_readout_saved_bytes(pink_hip_readout *r, uint32_t images)
{
    return !r || !r->cfg.features || (uint64_t)images * r->cfg.chosen > 0x7fffffffu ? 0 : saved_layout(r, images).bytes;
}

int pink_hip_readout_experts(pink_hip_readout *r, const void *x, uint32_t images, uint64_t x_stride, const int32_t *neuron, const float *gates,
                             const pink_hip_readout_weights *weights, const void *residual, uint64_t residual_stride, void *y,
                             uint64_t y_stride, void *saved)
{
    if (!r) return PINK_HIP_EINVAL;
    const pink_hip_readout_config &c = r->cfg;
    if (!c.features) return fail(r, PINK_HIP_ESTATE, "pink_hip_readout_experts: the handle was made without models");
    if (images == 0) return PINK_HIP_OK;
    REFUSE(r, !x || !neuron || !gates || !weights || !weights->first || !weights->second || !y, "pink_hip_readout_experts: null argument");
    x_stride = x_stride ? x_stride : c.features;
    y_stride = y_stride ? y_stride : c.outputs;
    residual_stride = residual_stride ? residual_stride : c.outputs;
    REFUSE(r, x_stride < c.features || y_stride < c.outputs || residual_stride < c.outputs, "pink_hip_readout_experts: rows overlap");
    REFUSE(r, (uintptr_t)saved & 255, "pink_hip_readout_experts: saved must be aligned to 256 bytes");
    TRY(check_images(r, images));
    HIP_TRY(r, hipSetDevice(c.device));
    if (c.element == PINK_HIP_ELEMENT_BFLOAT)
        return experts<Bfloat>(r, x, images, x_stride, neuron, gates, *weights, residual, residual_stride, y, y_stride, saved);
    return experts<float>(r, x, images, x_stride, neuron, gates, *weights, residual, residual_stride, y, y_stride, saved);
}

int pink_hip_readout_experts_backward(pink_hip_readout *r, const void *x, uint32_t images, uint64_t x_stride, const float *gates,
                                      const pink_hip_readout_weights *weights, const void *saved, const void *dy, uint64_t dy_stride,
                                      const pink_hip_readout_gradients *out, uint64_t dx_stride)
{
    if (!r) return PINK_HIP_EINVAL;
    const pink_hip_readout_config &c = r->cfg;
    if (!c.features) return fail(r, PINK_HIP_ESTATE, "pink_hip_readout_experts_backward: the handle was made without models");
    REFUSE(r, !out, "pink_hip_readout_experts_backward: null argument");
    const size_t e = element_bytes(r);
    HIP_TRY(r, hipSetDevice(c.device));
    if (images == 0) {                                     // nothing was chosen: the weights' gradients are zero
        const auto clear = [&](void *at, uint64_t n) {
            if (at) k_clear<<<1024, 256, 0, r->stream>>>((uint8_t *)at, n * e);
        };
        clear(out->first, (uint64_t)c.neurons * c.hidden * c.features);
        clear(out->first_bias, (uint64_t)c.neurons * c.hidden);
        clear(out->second, (uint64_t)c.neurons * c.outputs * c.hidden);
        clear(out->second_bias, (uint64_t)c.neurons * c.outputs);
        return launched(r, "k_clear");
    }
    REFUSE(r, !x || !gates || !weights || !weights->first || !weights->second || !saved || !dy, "pink_hip_readout_experts_backward: null argument");
    x_stride = x_stride ? x_stride : c.features;
    dx_stride = dx_stride ? dx_stride : c.features;
    dy_stride = dy_stride ? dy_stride : c.outputs;
    REFUSE(r, x_stride < c.features || dx_stride < c.features || dy_stride < c.outputs, "pink_hip_readout_experts_backward: rows overlap");
    REFUSE(r, (uintptr_t)saved & 255, "pink_hip_readout_experts_backward: saved must be aligned to 256 bytes");
    TRY(check_images(r, images));
    if (c.element == PINK_HIP_ELEMENT_BFLOAT)
        return experts_backward<Bfloat>(r, x, images, x_stride, gates, *weights, saved, dy, dy_stride, *out, dx_stride);
    return experts_backward<float>(r, x, images, x_stride, gates, *weights, saved, dy, dy_stride, *out, dx_stride);
}

int pink_hip_readout_adamw(pink_hip_readout *r, const pink_hip_readout_tensor *tensors, uint32_t count, uint32_t state_bits, uint64_t step,
                           float learning_rate, float beta_first, float beta_second, float epsilon)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, count && !tensors, "pink_hip_readout_adamw: null argument");
    REFUSE(r, state_bits != 8 && state_bits != 32, "pink_hip_readout_adamw: states have 8 or 32 bits");
    REFUSE(r, step == 0, "pink_hip_readout_adamw: steps count from 1");
    REFUSE(r, !(beta_first >= 0.0f && beta_first < 1.0f && beta_second >= 0.0f && beta_second < 1.0f), "pink_hip_readout_adamw: betas must be in [0, 1)");
    REFUSE(r, !(epsilon > 0.0f), "pink_hip_readout_adamw: epsilon must be larger than 0");
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    AdamArgs g = {};
    g.rate = learning_rate;
    g.beta1 = beta_first;
    g.beta2 = beta_second;
    g.rest1 = 1.0f - beta_first;
    g.rest2 = 1.0f - beta_second;
    g.c1 = (float)(1.0 / (1.0 - std::pow((double)beta_first, (double)step)));
    g.c2 = (float)(1.0 / (1.0 - std::pow((double)beta_second, (double)step)));
    g.epsilon = epsilon;
    return over_tensors(
        r, tensors, count, g,
        [&](const pink_hip_readout_tensor &t) -> int {
            REFUSE(r, !t.value || !t.gradient || !t.first || !t.second, "pink_hip_readout_adamw: null argument");
            REFUSE(r, state_bits == 8 && (!t.first_scale || !t.second_scale), "pink_hip_readout_adamw: 8-bit states need scales");
            REFUSE(r, t.gradient_element > PINK_HIP_ELEMENT_BFLOAT, "unknown element type");
            return PINK_HIP_OK;
        },
        [&](uint32_t blocks) {
            const bool small = epsilon < 0x1p-38f;
            if (state_bits == 8 && small) k_adamw<true, true><<<blocks, 256, 0, r->stream>>>(g);
            else if (state_bits == 8) k_adamw<true, false><<<blocks, 256, 0, r->stream>>>(g);
            else if (small) k_adamw<false, true><<<blocks, 256, 0, r->stream>>>(g);
            else k_adamw<false, false><<<blocks, 256, 0, r->stream>>>(g);
        });
}

int pink_hip_readout_unpack(pink_hip_readout *r, const pink_hip_readout_tensor *tensors, uint32_t count)
{
    if (!r) return PINK_HIP_EINVAL;
    REFUSE(r, count && !tensors, "pink_hip_readout_unpack: null argument");
    HIP_TRY(r, hipSetDevice(r->cfg.device));
    AdamArgs g = {};
    return over_tensors(
        r, tensors, count, g,
        [&](const pink_hip_readout_tensor &t) -> int {
            REFUSE(r, !t.first || !t.second || !t.first_scale || !t.second_scale || !t.first_values || !t.second_values, "pink_hip_readout_unpack: null argument");
            return PINK_HIP_OK;
        },
        [&](uint32_t blocks) { k_unpack<<<blocks, 256, 0, r->stream>>>(g); });
}

}  // extern "C"
