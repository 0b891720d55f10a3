// The beam selection's lists of candidates on the CPU: a workgroup's waves restated lane by lane with the library's own words, bound and
// list size (gq_beam.h), over rows of signed zeros, few values, and lanes that hold nothing but passing logits. Prints for each number of
// logits a lane and of beams the most entries a wave puts into its list beside the list's size, whether the best n_beam are among them,
// and the pattern.
#include "gq_beam.h"

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

using namespace gq;

namespace {
struct Wave {
    std::vector<std::vector<std::pair<float, int>>> lane;  // (logit, token) of each lane
};

// A chunk's logits dealt to the waves as the kernel deals them, in pieces of four.
std::vector<Wave> deal(const std::vector<float> & x, int per) {
    const int n = int(x.size());
    std::vector<Wave> w(4);
    for (auto & y : w) y.lane.resize(64);
    for (int tid = 0; tid < 256; ++tid) {
        auto & l = w[tid / 64].lane[tid % 64];
        for (int j = 0; j < per; ++j) {
            const int t = 4 * (256 * (j >> 2) + tid) + (j & 3);
            if (t < n) l.push_back({x[t], t});
        }
    }
    return w;
}

// The tokens that the wave lists.
std::vector<std::pair<float, int>> listed(const Wave & w, int k, int ch) {
    uint32_t top[64], high = 0, low = UINT_MAX;
    for (int l = 0; l < 64; ++l) {
        float m = -INFINITY;
        for (auto & e : w.lane[l]) m = e.first > m || (e.first == m && std::signbit(m)) ? e.first : m;  // +0 over -0, as the hardware's maximum
        top[l] = w.lane[l].empty() ? 0 : beam_order(m);
        high = std::max(high, top[l]);
        low = std::min(low, top[l]);
    }
    int n;
    const uint32_t lo = beam_bound([&](uint32_t y) { return int(std::count_if(top, top + 64, [&](uint32_t t) { return t >= y; })); }, k, low, high, n);
    std::vector<std::pair<float, int>> out;
    if (n <= k + BEAM_SLACK && lo > beam_order(-INFINITY)) {
        const float bound = beam_number(lo);
        for (auto & l : w.lane)
            for (auto & e : l)
                if (e.first >= bound) out.push_back(e);
        return out;
    }
    int until = INT_MAX;
    if (n > k + BEAM_SLACK) {
        int mine[64], above = 0;
        for (int l = 0; l < 64; ++l) {
            mine[l] = INT_MAX;
            if (top[l] == lo)
                for (auto & e : w.lane[l])
                    if (beam_order(e.first) == lo) mine[l] = std::min(mine[l], e.second);
            above += top[l] > lo;
        }
        int a = -1, b = ch;
        while (b - a > 1) {
            const int mid = a + (b - a) / 2;
            if (above + std::count_if(mine, mine + 64, [&](int t) { return t <= mid; }) >= k) b = mid;
            else a = mid;
        }
        until = b;
    }
    for (auto & l : w.lane)
        for (auto & e : l)
            if (beam_order(e.first) > lo || (beam_order(e.first) == lo && e.second <= until)) out.push_back(e);
    return out;
}

bool better(const std::pair<float, int> & a, const std::pair<float, int> & b) {
    return a.first > b.first || (a.first == b.first && a.second < b.second);
}
}  // namespace

int main() {
    std::mt19937 rng(1);
    for (int per : {8, 32})
        for (int k = 1; k <= BEAM_MAX; ++k) {
            const int ch = 256 * per;
            int most = 0, pattern = -1;
            bool all = true;
            const auto run = [&](const std::vector<float> & x, int what) {
                for (const Wave & w : deal(x, per)) {
                    auto out = listed(w, k, ch);
                    const int n = (int(out.size()) + 7) / 8 * 8;  // as many are written
                    if (n > most) {
                        most = n;
                        pattern = what;
                    }
                    std::vector<std::pair<float, int>> want;
                    for (auto & l : w.lane) want.insert(want.end(), l.begin(), l.end());
                    std::sort(want.begin(), want.end(), better);
                    // in the kernel's order, entries go by word and token
                    std::sort(out.begin(), out.end(), [](auto & a, auto & b) {
                        const uint32_t x = beam_order(a.first), y = beam_order(b.first);
                        return x > y || (x == y && a.second < b.second);
                    });
                    const size_t m = std::min(want.size(), size_t(k));
                    all = all && out.size() >= m && std::equal(want.begin(), want.begin() + long(m), out.begin(),
                                                               [](auto & a, auto & b) { return a.second == b.second; });
                }
            };
            std::vector<float> x(static_cast<size_t>(ch));
            for (int few : {1, k, k + 2, k + BEAM_SLACK}) {  // +0 in so many lanes of each wave, -0 elsewhere
                std::fill(x.begin(), x.end(), -0.0f);
                for (int w = 0; w < 4; ++w)
                    for (int l = 0; l < std::min(few, 64); ++l) x[size_t(4 * (64 * w + l) + 3)] = 0.0f;
                run(x, 0);
                std::fill(x.begin(), x.end(), 0.0f);  // and the other way round
                for (int l = 0; l < std::min(few, 64); ++l) x[size_t(4 * l)] = -0.0f;
                run(x, 1);
            }
            for (int first = 0; first < 4; ++first)  // all of lanes first .. first + k + 3 above the rest
                for (int lanes : {k, k + BEAM_SLACK, k + BEAM_SLACK + 1})
                    for (int same = 0; same < 2; ++same) {
                        for (float & y : x) y = -5.0f - float(rng() % 1000) / 256;
                        for (int l = first; l < std::min(first + lanes, 64); ++l) {
                            for (int j = 0; j < per; ++j) {
                                const int t = 4 * (256 * (j >> 2) + l) + (j & 3);
                                x[size_t(t)] = same ? 2.0f : 2.0f + float(rng() % 1000) / 256;
                            }
                        }
                        run(x, 2 + first);
                    }
            for (int n : {1, 5, 63, 256, 700, ch}) {  // few values, short rows, masks
                for (int what = 0; what < 3; ++what) {
                    x.resize(static_cast<size_t>(std::min(n, ch)));
                    for (float & y : x) {
                        const int r = int(rng() % 5);
                        y = what == 0 ? float(r - 2) * (rng() % 2 ? 1.0f : -1.0f) * 0.5f : what == 1 ? (r ? -INFINITY : -0.0f) : float(rng() % 4096) / 64 - 32;
                    }
                    run(x, 6 + what);
                }
            }
            std::printf("%d %d %d %d %d %d\n", per, k, most, beam_list(k, per), int(all), pattern);
        }
    return 0;
}
