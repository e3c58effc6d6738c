// Walks of all threads of all blocks for random shapes: every value once, none outside, every channel's sum from its own entries, and the
// shared memory that the kernel lays out is what the plan asks for.  Built and run by test_norm_plan.py.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <vector>

#include "axc_norm_plan.h"

using namespace axc;

static unsigned long long g_state = 88172645463325252ull;
static long long pick(long long lo, long long hi)
{
    g_state ^= g_state << 13;
    g_state ^= g_state >> 7;
    g_state ^= g_state << 17;
    return lo + (long long)(g_state % (unsigned long long)(hi - lo + 1));
}
#define CHECK(x)                                                                                                                                   \
    do {                                                                                                                                           \
        if (!(x)) {                                                                                                                                \
            std::printf("%s: %lld x %lld x %lld, %lld groups, size %d aligned %d: span %d blocks %d threads %d vec %d shares %lld\n", #x, s.samples, \
                        s.places, s.channels, s.groups, s.size, int(s.aligned), p.span, p.blocks, p.threads, p.vec, p.shares);                     \
            std::exit(1);                                                                                                                          \
        }                                                                                                                                          \
    } while (0)

template <int V>
static void block(const NormShape &s, const NormPlan &p, const Span &sp, long long sample, long long place0, int places, int channel0, std::vector<unsigned char> &seen,
                  long long steps)
{
    const int active = sp.active, span = sp.channels;
    const int shift = V == 1 || span < s.channels ? 0 : int((sample * s.places + place0) * s.channels & (V - 1));
    const Entries E(sp, shift, places * span);
    CHECK(places * (long long)span <= (1 << 20) + span);
    std::vector<int> count(size_t(active) * V), channel(size_t(active) * V, -1);
    CHECK(active > 0 && active <= p.threads && (active * V) % span == 0);
    for (int t = 0; t < p.threads; ++t) {
        const Walk<V> w(t, sp, shift, places, s.channels, place0, channel0);
        CHECK(steps < 0 || w.count <= steps);
        CHECK(t < active || w.count == 0);
        int local[V], group[V];
        local_channels<V>(w, sp, p.resident ? divider(unsigned(s.each())) : sp.by_channels, local, group);
        CHECK(w.count == (t < active && w.o < w.total ? (w.total - 1 - w.o) / w.each + 1 : 0));
        for (int j = 0; j < w.count; ++j) {
            const long long first = sample * s.places * s.channels + w.at + j * w.step;
            if (w.whole(j)) CHECK(first % V == 0 || V == 1);
            CHECK(j == 0 || j == w.count - 1 || w.whole(j));
            for (int i = 0; i < V; ++i) {
                if (!w.has(j, i)) {
                    CHECK(!w.whole(j));
                    continue;
                }
                CHECK(first + i >= sample * s.places * s.channels && first + i < (sample + 1) * s.places * s.channels);
                const int c = int((first + i) % s.channels);
                CHECK(c == channel0 + local[i]);
                CHECK(!p.resident || c / s.each() == (channel0 + group[i] * s.each()) / s.each());
                ++seen[size_t(first + i)];
                ++count[size_t(t) * V + i];
                channel[size_t(t) * V + i] = c - channel0;
            }
        }
    }
    std::vector<unsigned char> used(size_t(active) * V);
    for (int l = 0; l < span; ++l)
        for (int k = 0; k < E.copies; ++k) {
            const int e = E.first_entry(l) + k * span;
            CHECK(e >= 0 && e < active * V && !used[e]);
            CHECK(e / span == k && E.place(e, k) == e + k && E.place(e, k) < entry_places(sp));
            used[e] = 1;
            CHECK(channel[e] == -1 || channel[e] == l);
            CHECK(int(E.values(e)) == count[e]);
        }
    CHECK(E.copies * span == active * V);
}

template <int V>
static void whole(const NormShape &s, const NormPlan &p, bool residual, int sums)
{
    std::vector<unsigned char> seen(size_t(s.values()));
    const int spans = int((s.channels + p.span - 1) / p.span);
    for (long long n = 0; n < s.samples; ++n)
        for (int c = 0; c < spans; ++c) {
            const int channel0 = c * p.span;
            if (p.resident) {
                CHECK(s.channels % p.span == 0 && p.span % s.each() == 0 && p.blocks >= 1 && p.blocks <= s.places);
                const int active = norm_active(p.threads, p.span, p.vec), groups = int(p.span / s.each());
                const Span sp = span_of(p.span, active, p.vec);
                const long long steps = norm_steps((s.places + p.blocks - 1) / p.blocks, p.span, p.vec, active);
                const size_t slots = size_t(steps) * active * p.vec;
                // as the kernels lay it out
                const size_t data = (sums ? residual ? 3 : 2 : 1) * norm_up16(slots * s.size);
                if (sums && norm_lanes(p.span, p.vec, p.threads)) CHECK(active == p.threads && s.channels % p.vec == 0);
                else if (!sums && V > 1 && s.each() % V == 0) CHECK(entry_places(span_of(p.span / V, active, 1)) == norm_entries(p.span, p.vec, p.threads, active, s.each(), false));
                else CHECK(entry_places(sp) == norm_entries(p.span, p.vec, p.threads, active, s.each(), sums));
                CHECK(data + size_t(norm_entries(p.span, p.vec, p.threads, active, s.each(), sums)) * 8 + size_t(p.span) * 8 * sums + size_t(groups) * 16 <= p.smem && p.smem <= kNormSmem);
                const long long per = (s.places + p.blocks - 1) / p.blocks;
                CHECK(per * (p.blocks - 1) < s.places);
                for (int r = 0; r < p.blocks; ++r) {
                    const long long p0 = r * per, p1 = p0 + per < s.places ? p0 + per : s.places;
                    block<V>(s, p, sp, n, p0, int(p1 - p0), channel0, seen, steps);
                }
            } else {
                const int span = int(s.channels - channel0 < p.span ? s.channels - channel0 : p.span);
                const Span sp = span_of(span, norm_active(p.threads, span, p.vec), p.vec);
                CHECK(entry_places(sp) <= 2 * kNormThreads * V);
                const long long per = (s.places + p.shares - 1) / p.shares;
                CHECK(per * (p.shares - 1) < s.places);
                for (long long h = 0; h < p.shares; ++h) {
                    const long long p0 = h * per, p1 = p0 + per < s.places ? p0 + per : s.places;
                    block<V>(s, p, sp, n, p0, int(p1 - p0), channel0, seen, -1);
                }
            }
        }
    for (unsigned char c : seen) CHECK(c == 1);
}

int main(int argc, char **argv)
{
    const int rounds = argc > 1 ? std::atoi(argv[1]) : 300;
    int resident = 0, twice = 0, single = 0, loose = 0;
    for (int i = 0; i < rounds; ++i) {
        NormShape s;
        const bool large = i % 4 == 0;
        s.groups = pick(1, i % 3 ? 12 : 300);
        s.channels = s.groups * pick(1, i % 5 ? 24 : 2500 / s.groups + 1);
        s.places = pick(1, large ? 4000000 / s.channels + 1 : 300);
        s.samples = pick(1, large ? 2 : 5);
        s.size = pick(0, 1) ? 2 : 4;
        s.aligned = pick(0, 4) != 0;
        for (int backward = 0; backward < 2; ++backward) {
            const bool residual = pick(0, 1);
            const NormPlan p = norm_plan(s, (backward ? residual ? 3 : 2 : 1) * s.size, (backward ? residual ? 5 : 3 : residual ? 3 : 2) * s.size, backward, 148);
            ++(p.resident ? resident : twice);
            if (p.vec == 1) ++single;
            else if (s.channels % p.vec) ++loose;
            if (p.vec == 8) whole<8>(s, p, residual, backward);
            else if (p.vec == 4) whole<4>(s, p, residual, backward);
            else whole<1>(s, p, residual, backward);
        }
    }
    std::printf("resident %d, twice %d, single values %d, loose lines %d\n", resident, twice, single, loose);
    return resident && twice && single && loose ? 0 : 2;
}
