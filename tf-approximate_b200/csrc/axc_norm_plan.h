// How group norm's kernels cut up their tensors, and a thread's way through its part.  Plain arithmetic, in a header of its own so that it can be checked without a GPU
// over any number of sizes: the workspace's size, the shared memory and the launches come from here.
#pragma once
#include <stddef.h>

#ifdef __CUDACC__
#define AXC_BOTH __host__ __device__ __forceinline__
#else
#define AXC_BOTH inline
#endif

namespace axc {

constexpr int kNormThreads = 256;              // of a block, at most
constexpr int kNormCluster = 8;                // blocks that share a span, at most
constexpr long long kNormSmem = 226 * 1024;    // of a block, at most

struct NormShape {
    long long samples, places, channels, groups;
    int size;                                  // bytes of a value
    bool aligned;                              // every tensor starts on 16 bytes
    long long each() const { return channels / groups; }
    long long values() const { return samples * places * channels; }
};

// Resident: a span, which is a sample's channels of one or several whole groups, stays in the shared memory of a cluster of `blocks` blocks between
// the sums over it and what is computed of them.  Else the tensors are read twice, in blocks of `span` channels and a share of the places each.
struct NormPlan {
    bool resident;
    int vec;                                   // values that a thread moves at a time: 16 bytes of them, or one
    int threads, span, blocks;
    long long shares;                          // not resident: blocks that share a sample's places
    unsigned smem;
};

inline long long norm_gcd(long long a, long long b)
{
    while (b) {
        const long long t = a % b;
        a = b;
        b = t;
    }
    return a;
}

// Threads of `threads` that take part, so that each keeps its `vec` channels from one step to the next: as many as are a multiple of what the
// channels' order repeats after.  0: it repeats after more than all of them.
inline int norm_active(int threads, int span, int vec)
{
    const long long period = span / norm_gcd(span, vec);
    return period > threads ? 0 : int(threads / period * period);
}

// Steps that the threads take for the places of a block, one more where a sample starts inside 16 bytes
inline long long norm_steps(long long places, int span, int vec, int active)
{
    const long long all = places * span + vec - 1, each = (long long)active * vec;
    return (all + each - 1) / each;
}

AXC_BOTH size_t norm_up16(size_t bytes) { return (bytes + 15) / 16 * 16; }

// Vectors of a line where the lanes of a warp can add up what they have of the same channels, else 0: a power of two, with two lines in a warp at least
inline int norm_lanes(int span, int vec, int threads)
{
    const int period = span % vec ? 0 : span / vec;
    return vec > 1 && period > 0 && period <= 16 && (period & (period - 1)) == 0 && threads % 32 == 0 ? period : 0;
}

// Pairs of sums that a resident block's threads leave each other: one for each thread where its channels are of one group (forward), for each
// channel and warp where the lanes add up theirs (backward), else for each channel of each thread; a place more for every copy of the span.
inline long long norm_entries(int span, int vec, int threads, int active, long long each, bool backward)
{
    if (!backward && vec > 1 && each % vec == 0) return active + (long long)active * vec / span;
    if (backward && norm_lanes(span, vec, threads)) return (long long)threads / 32 * (span + 1);
    return (long long)active * vec + (long long)active * vec / span;
}

// Shared memory of a resident block: `kept` bytes for each value, the entries, pairs of sums of single channels (backward), four floats for each
// group (a pair for the cluster's blocks to read, a pair of results).
inline long long norm_smem(long long places, int span, int vec, int threads, int active, int kept, long long each, bool backward)
{
    return norm_steps(places, span, vec, active) * active * vec * kept + 48 + norm_entries(span, vec, threads, active, each, backward) * 8 + (long long)span * 8 * backward +
           span / each * 16;
}

// Channels at a time where the tensors are read twice
inline int norm_columns(const NormShape &s, int *vec)
{
    const int wide = 16 / s.size;
    *vec = s.aligned && (s.channels % wide == 0 || norm_active(kNormThreads, int(s.channels < (1 << 20) ? s.channels : (1 << 20)), wide) > 0) ? wide : 1;
    const long long most = (long long)kNormThreads * *vec;
    if (s.channels % *vec) return int(s.channels);            // lines that start anywhere: whole ones
    return int(s.channels < most ? s.channels : most);
}

// `kept`: bytes that stay in shared memory for each value; `moved`: bytes read and written for each.
//
// The estimate, in us: all bytes at memory's rate, or the blocks' own times in as many rounds as the SMs take them, whichever is more, and one block's
// time.  A block takes 3 us for its start, its two exchanges and its end, 1 more in a cluster, and its bytes at what an SM moves with the blocks that
// fit on it (20 bytes a ns for each, 44 at most).  Pieces of a line below 64 bytes are charged for the rest of what memory moves.
inline NormPlan norm_plan(const NormShape &s, int kept, int moved, bool backward, int sms)
{
    NormPlan best = {};
    double least = 1e300;
    const int wide = 16 / s.size;
    const long long each = s.each();
    for (int v = 0; v < 2; ++v) {
        const int vec = v == 0 ? wide : 1;
        if (vec > 1 && !s.aligned) continue;
        for (long long k = 1; k <= s.groups; ++k) {
            if (s.groups % k) continue;
            const long long span = each * k;
            if (span > (long long)kNormThreads * vec) break;
            if (span < s.channels && (span % vec || s.channels % vec)) continue;
            for (int threads = 64; threads <= kNormThreads; threads *= 2) {
                const int active = norm_active(threads, int(span), vec);
                if (!active) continue;
                for (int blocks = 1; blocks <= kNormCluster && blocks <= s.places; ++blocks) {
                    const long long places = (s.places + blocks - 1) / blocks;
                    if ((blocks - 1) * places >= s.places) continue;           // the last one has none
                    if (places * span > (1ll << 20)) continue;
                    const long long smem = norm_smem(places, int(span), vec, threads, active, kept, each, backward);
                    if (smem > kNormSmem) continue;
                    const double line = double(span) * s.size, waste = span == s.channels || line >= 64 ? 1.0 : line >= 32 ? 1.15 : 32 / line;
                    long long fit = kNormSmem / (smem + 1024);
                    if (fit > (backward ? 512 : 768) / threads) fit = (backward ? 512 : 768) / threads;       // registers
                    const double units = double(s.samples) * double(s.groups / k) * blocks;
                    // a thread has four accesses on their way
                    double rate = double(fit) * threads * vec * s.size * 4 / 800.0;
                    if (rate > 44) rate = 44;
                    const double bytes = double(places) * double(span) * moved * waste * (vec == 1 ? 2.0 : 1.0);
                    const double own = 3.0 + (blocks > 1 ? 1.0 : 0.0) + bytes * double(fit) / rate / 1000.0;
                    const double rounds = units / (double(sms) * double(fit)), cover = units < sms ? units / sms : 1.0;
                    const double memory = double(s.values()) * moved * waste / (6.5e6 * cover);
                    const double time = (rounds * own > memory ? rounds * own : memory) + own * (rounds < 1 ? 1.0 - rounds + 1e-3 : 0.5);
                    if (time < least) {
                        least = time;
                        best = {true, vec, threads, int(span), blocks, 0, unsigned(smem)};
                    }
                }
            }
        }
    }
    NormPlan swept = {};
    swept.span = norm_columns(s, &swept.vec);
    swept.threads = kNormThreads;
    // six blocks for every SM, of 32 KiB at least and a million values at most
    const long long across = s.samples * ((s.channels + swept.span - 1) / swept.span), most = s.places * swept.span * s.size / (32 * 1024) + 1;
    long long shares = ((long long)sms * 6 + across - 1) / (across ? across : 1);
    if (shares > most) shares = most;
    if (shares > s.places) shares = s.places;
    const long long fewest = (s.places * swept.span >> 20) + 1;
    if (shares < fewest) shares = fewest;
    if (shares < 1) shares = 1;
    const long long per = s.places > 0 ? (s.places + shares - 1) / shares : 1;
    swept.shares = s.places > 0 ? (s.places + per - 1) / per : 1;
    // Read twice: all bytes and those that are read again at 70 % of memory's rate (single values at a fourth of that), or 3 us for each of the two
    // passes' blocks, 3 of which (backward 2) an SM takes at a time, whichever is more; between the passes 4.1 us for each sample's groups, a block each, 8 an SM; and
    // three launches.  (Without the blocks' times 200704 x 1 x 256 bf16 in 32 groups took 23.5 ms instead of 0.5, 16384 x 16 x 64 in 8 groups 629 us instead of 50.)
    const int again = backward ? (moved / s.size == 5 ? 3 : 2) : 1;
    const double bytes = double(s.values()) * (moved + again * s.size) / (4.6e6 * (swept.vec > 1 ? 1.0 : 0.25));
    const double blocks = 2 * 3.0 * double(across) * double(swept.shares) / (double(sms) * (backward ? 2 : 3)), join = 4.1 * double(s.samples) * double(s.groups) / (8.0 * sms);
    if (best.resident && least <= 14.0 + (bytes > blocks ? bytes : blocks) + join) return best;
    return swept;
}

// Bytes of scratch: pairs of fp32 sums for every sample and channel, and share; group sums behind them
inline size_t norm_pad(size_t bytes) { return (bytes + 255) / 256 * 256; }
inline size_t norm_part_bytes(const NormShape &s, const NormPlan &p)
{
    return p.resident ? 0 : norm_pad(size_t(s.samples) * size_t(p.shares) * size_t(s.channels) * 8);
}
inline size_t norm_sums_bytes(const NormShape &s) { return norm_pad(size_t(s.samples) * size_t(s.channels) * 8); }
inline size_t norm_group_bytes(const NormShape &s) { return norm_pad(size_t(s.samples) * size_t(s.groups) * 8); }

// n / by for n by < 2^32, by one multiplication
struct Divider {
    unsigned by, magic;
    AXC_BOTH unsigned of(unsigned n) const
    {
#ifdef __CUDA_ARCH__
        return magic ? __umulhi(n, magic) : n;
#else
        return magic ? unsigned((unsigned long long)n * magic >> 32) : n;
#endif
    }
};
inline Divider divider(unsigned by) { return {by, by > 1 ? unsigned(((1ull << 32) + by - 1) / by) : 0u}; }

// A span as the kernels have it: its channels and groups, the threads that take part, the values that they take in a step, lines of a step, sets of
// entries (see Entries)
struct Span {
    int channels, active, each, lines, copies;
    Divider by_channels, by_each, by_copies;
};
inline Span span_of(int channels, int active, int vec)
{
    const int each = active * vec;
    return {channels, active, each, each / channels, each / channels, divider(unsigned(channels)), divider(unsigned(each)), divider(unsigned(each / channels))};
}

// ---- in the kernels ------------------------------------------------------------------------------------------------------------
// A thread's way through the places and channels of its block: `count` vectors, the j-th with the values o + j * each .. of the block's own
// (place by place, `total` of them), at at + j * step from the sample's start.  Those from `first` to `end` are whole; one before and one
// behind them may stick out of the block's values.
template <int V>
struct Walk {
    int o, each, count, total, first, end;
    long long at, step;
    AXC_BOTH Walk(int thread, const Span &s, int shift, int places, long long channels, long long place0, int channel0)
    {
        each = s.each;
        o = thread * V - shift;
        total = places * s.channels;
        count = thread < s.active && o < total ? int(s.by_each.of(unsigned(total - 1 - o))) + 1 : 0;
        if (s.channels == channels) {
            at = place0 * channels + o;
            step = each;
        } else {
            const int line = int(s.by_channels.of(unsigned(o)));
            at = (place0 + line) * channels + channel0 + (o - line * s.channels);
            step = s.lines * channels;
        }
        first = V > 1 && count > 0 && !whole(0) ? 1 : 0;
        end = V > 1 && count > first && !whole(count - 1) ? count - 1 : count;
    }
    AXC_BOTH bool whole(int j) const
    {
        if (V == 1) return true;
        const int s = o + j * each;
        return s >= 0 && s + V <= total;
    }
    AXC_BOTH bool has(int j, int i) const
    {
        const int s = o + j * each + i;
        return s >= 0 && s < total;
    }
};
// Thread t's channel i is entry t * V + i; a span's channel l has the entries (l + shift) mod span + k * span, the k-th copy of it.  In shared
// memory each copy is one place further on, or the copies of a channel would all be in the same banks.
struct Entries {
    int span, shift, copies, each, rest, base;
    AXC_BOTH Entries(const Span &s, int shift_, int total)
    {
        span = s.channels;
        shift = shift_;
        each = s.each;
        copies = s.copies;
        base = int(s.by_each.of(unsigned(total)));
        rest = total - base * each;
    }
    AXC_BOTH int first_entry(int l) const
    {
        int e = l + shift;
        while (e >= span) e -= span;
        return e;
    }
    AXC_BOTH int place(int entry, int copy) const { return entry + copy; }
    // values that were added up in it
    AXC_BOTH float values(int entry) const
    {
        int o = entry - shift;
        if (o < 0) o += each;
        return float(base + (o < rest ? 1 : 0));
    }
};
AXC_BOTH int entry_places(const Span &s) { return s.each + s.copies; }

// The channels of a thread's values, counted from the span's first, and their groups (of `by_group` channels) counted the same way
template <int V>
AXC_BOTH void local_channels(const Walk<V> &w, const Span &s, const Divider &by_group, int (&local)[V], int (&group)[V])
{
    int l = w.o;
    if (V > 1)
        while (l < 0) l += s.channels;
    l -= int(s.by_channels.of(unsigned(l))) * s.channels;
    int g = int(by_group.of(unsigned(l))), d = l - g * int(by_group.by);
    for (int i = 0; i < V; ++i) {
        local[i] = l;
        group[i] = g;
        ++l;
        if (++d == int(by_group.by)) d = 0, ++g;
        if (l == s.channels) l = g = d = 0;
    }
}

}  // namespace axc
