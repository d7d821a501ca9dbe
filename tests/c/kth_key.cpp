// Rows of keys with ties of every extent through csrc/kth_key.h: whether the threshold
// lets the k first through, and no more than can be sorted. Prints the rows looked at
// and the wrong ones.
#include "../../wpc-engine_amd/csrc/kth_key.h"

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

using wpcg::KthKey;

static const int MOST = 256;
static unsigned long long rows, wrong;

// The order of a float as the kernel has it; 0: no key.
static uint32_t order_of(float v)
{
    if (!(v > -INFINITY)) return 0;
    v += 0.0f;
    uint32_t b;
    memcpy(&b, &v, 4);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// `lower`: an order that the k-th key's is not below.
static void check(const std::vector<uint32_t>& key, int k, uint32_t lower)
{
    const int places = (int)key.size();
    uint32_t least = 0xffffffffu;
    for (uint32_t o : key)
        if (o >= std::max(lower, 1u)) least = std::min(least, o);
    const auto from = [&](uint32_t o) {
        return (int)std::count_if(key.begin(), key.end(), [&](uint32_t x) { return x >= o; });
    };
    const auto at = [&](uint32_t o, int p) { return (int)std::count(key.begin(), key.begin() + p + 1, o); };
    if (from(std::max(lower, 1u)) <= MOST) return;  // these are sorted as they are
    const KthKey t = wpcg::kth_key(k, MOST, least, places, from, at);
    std::vector<int> order(places);
    for (int i = 0; i < places; i++) order[i] = i;
    std::stable_sort(order.begin(), order.end(), [&](int a, int b) { return key[a] > key[b]; });
    const auto through = [&](int i) { return key[i] != 0 && (key[i] > t.order || (key[i] == t.order && i <= t.place)); };
    int n = 0;
    for (int i = 0; i < places; i++) n += through(i);
    bool ok = n >= k && n <= MOST;
    for (int i = 0; i < k; i++) ok &= through(order[i]);
    rows++;
    if (!ok && wrong++ < 5) std::printf("wrong: %d places, k %d, %d through, order %08x place %d\n", places, k, n, t.order, t.place);
}

// The candidates that the kernel would look at: all, and with what lies below the best
// of k of them already left out.
static void check_row(const std::vector<float>& row, int k)
{
    std::vector<uint32_t> key(row.size());
    for (size_t i = 0; i < row.size(); i++) key[i] = order_of(row[i]);
    std::vector<uint32_t> sorted = key;
    std::sort(sorted.rbegin(), sorted.rend());
    if ((int)sorted.size() < k || sorted[k - 1] == 0) return;
    check(key, k, 0);
    check(key, k, sorted[std::min(sorted.size() - 1, (size_t)3 * k)]);
    check(key, k, sorted[k - 1]);
}

int main()
{
    std::mt19937 rng(7);
    const auto upto = [&](int n) { return (int)(rng() % (unsigned)n); };
    std::normal_distribution<float> normal;
    const float values[] = {0.0f, 2.0f, 1.0f, -1.0f, -0.0f, 4.0f, -3.4028235e38f, 1e-40f};
    for (int turn = 0; turn < 4000; turn++) {
        const int v = 257 + upto(2800), k = 1 + upto(64);
        std::vector<float> x(v);
        // rounded normals, of steps that make few or many ties
        const float step = std::exp2((float)(upto(12) - 8)), width = std::exp2((float)(upto(6) - 2));
        for (float& a : x) a = std::nearbyint(normal(rng) * width / step) * step;
        check_row(x, k);
        // a run of one value, some above it and all others below, anywhere in the row
        const float tie = values[upto(8)], low = turn % 3 ? -1e4f : -INFINITY;
        const int run = std::min(v, 1 + upto(400)), begin = upto(v - run + 1);
        for (float& a : x) a = turn % 2 ? low : tie - 1.0f - std::fabs(normal(rng));
        for (int i = 0; i < run; i++) x[begin + i] = tie;
        for (int i = upto(k + 2); i > 0; i--) x[upto(v)] = std::fabs(tie) + 1.0f + (float)upto(3);
        check_row(x, k);
        // neighbouring values, and each value alike
        for (float& a : x) a = 1.0f + std::exp2(-23.0f) * (float)upto(5);
        check_row(x, k);
        for (float& a : x) a = tie;
        check_row(x, k);
        if (turn % 4 == 0) {  // all different
            for (int i = 0; i < v; i++) x[i] = (float)(i - v / 2);
            std::shuffle(x.begin(), x.end(), rng);
            check_row(x, k);
        }
    }
    std::printf("%llu rows, %llu wrong\n", rows, wrong);
    return wrong != 0;
}
