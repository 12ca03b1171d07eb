// The warps of the 8-bit product kernel, played through on the host: the text
// of csrc/f8_mm.cu between its first role and the end of its last (roles.inc),
// its structures (structs.inc), its barriers' set-up (init.inc) and its
// descriptors (desc.inc) are compiled as they stand, one fibre for each warp of
// each CTA of a cluster, in random order.  What the device does is modelled
// here: barriers with arrivals and bytes, copies that land late, products that
// run late and in their thread's order, arrivals on their way to a CTA.
//
//   f8_roles SHAPE SEED FAULT    SHAPE: 0 128 x 128, 1 128 x 256, 2 pair, 3 shared contraction; +4 transposed
//                                FAULT 1: a wait of a random warp runs out at a random moment
//
// Checked: an operand holds the block that the product means, from its issue to
// its end; sums are read after their products and before the next ones; every
// tile is stored once with the sums it should have; nothing is stuck; and when
// all warps have come to the kernel's end, no copy, product or arrival that the
// end of a CTA would cut off is under way.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>
#include <unistd.h>

#include <math.h>

#include <deque>
#include <functional>
#include <map>
#include <random>
#include <string>
#include <type_traits>
#include <vector>

#define __device__
#define __host__
#define __forceinline__ inline
struct int4 { int x, y, z, w; };
struct float2 { float x, y; };
static int4 make_int4(int x, int y, int z, int w) { return {x, y, z, w}; }
static float2 make_float2(float x, float y) { return {x, y}; }
static float __uint_as_float(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static uint32_t __float_as_uint(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
static float2 __ffma2_rn(float2 a, float2 b, float2 c) { return {a.x * b.x + c.x, a.y * b.y + c.y}; }
static float2 __fmul2_rn(float2 a, float2 b) { return {a.x * b.x, a.y * b.y}; }
static float __ldg(const float *p) { return *p; }
static int __all_sync(unsigned, int v) { return v; }
static unsigned __reduce_max_sync(unsigned, unsigned v) { return v; }
static int __any_sync(unsigned, int v) { return v; }
static void __syncwarp() {}
enum { SHC_SRC_F32 = 0, SHC_SRC_F16 = 1, SHC_SRC_BF16 = 30, kF8Block = 128 };
struct CUtensorMap { char what; };

#include "structs.inc"

[[noreturn]] static void fail(const std::string &s) {
    printf("%s\n", s.c_str());
    fflush(stdout);
    _exit(1);
}
static void check(bool ok, const char *s) {
    if (!ok) fail(s);
}

// ---------------------------------------------------------------- fibres and events

static std::mt19937_64 rng;
static unsigned pick(unsigned n) { return (unsigned)(rng() % n); }
static ucontext_t g_main;
struct Fibre {
    ucontext_t ctx;
    std::vector<char> stack;
    std::function<void()> body;
    bool over = false, cut = false;  // cut: its next wait runs out
    int cta = 0;
};
static std::vector<Fibre *> g_fibres;
static Fibre *g_now;
static void yield() { swapcontext(&g_now->ctx, &g_main); }
static void run_fibre() {
    g_now->body();
    g_now->over = true;
    swapcontext(&g_now->ctx, &g_main);
}
// Under way in any order; `ordered`: a plain store or arrival, which the
// cluster barrier at the kernel's end waits for by itself.
struct Event { std::function<void()> what; bool ordered; };
static std::vector<Event> g_events;
static void later(std::function<void()> f, bool ordered = false) { g_events.push_back({f, ordered}); }

// ---------------------------------------------------------------- a CTA

struct Bar {
    int count = 0, pending = 0;
    int64_t bytes = 0;
    uint64_t phase = 0;
    void settle() {
        if (pending == 0 && bytes == 0) phase++, pending = count;
    }
    void arrive() { check(--pending >= 0, "a barrier gets more arrivals than it counts"); settle(); }
    bool passes(uint32_t parity) const { return (phase & 1) != parity; }
};
struct Tag { char map; int x, y, z; };
struct Sum { int c = -1, row0 = 0, col0 = 0, expert = 0, steps = 0; };
struct Cta {
    Control ctl;
    std::map<const void *, Bar> bars;
    std::map<uint32_t, Tag> ring;  // what lies at a copy's destination
    std::map<uint32_t, int> landing;
    std::vector<float> slots;
    std::map<uint32_t, Sum> tmem;
    std::map<uint32_t, int> waiting;  // products on their way to an accumulator
    int copies = 0;
};
static std::vector<Cta> g_cta;
static constexpr uint32_t kRing = 1024, kCtl = 0x40000;
static uint32_t smem_u32(const void *p) {
    for (size_t i = 0; i < g_cta.size(); i++) {
        const char *b = reinterpret_cast<const char *>(&g_cta[i].ctl), *q = static_cast<const char *>(p);
        if (q >= b && q < b + sizeof(Control)) return (uint32_t)(i << 24) + kCtl + (uint32_t)(q - b);
    }
    fail("an address outside shared memory");
}
static Cta &cta_at(uint32_t addr) { return g_cta[addr >> 24]; }
static Bar &bar_at(uint32_t addr) {
    Cta &c = cta_at(addr);
    auto it = c.bars.find(reinterpret_cast<char *>(&c.ctl) + ((addr & 0xFFFFFF) - kCtl));
    check(it != c.bars.end(), "not a barrier");
    return it->second;
}
static Cta &here() { return g_cta[g_now->cta]; }
static void mbar_init(unsigned long long *b, unsigned count) {
    Bar &x = here().bars[b];
    x.count = x.pending = (int)count;
}
static void mbar_arrive(unsigned long long *b) { bar_at(smem_u32(b)).arrive(); }
static uint32_t in_leader(uint32_t a) { return a & 0xFFFFFF; }
static bool elect_one() { return true; }

static void give_up() {
    for (auto &c : g_cta) {
        int *a = &c.ctl.abort;
        if (&c == &here()) *a = 1;
        else later([a] { *a = 1; }, true);
    }
}
static bool bar_wait(unsigned long long *b, uint32_t parity, volatile int *abort, int *) {
    for (;;) {
        yield();
        if (bar_at(smem_u32(b)).passes(parity)) return true;
        if (*abort) return false;
        if (g_now->cut) {
            g_now->cut = false;
            give_up();
            return false;
        }
    }
}
static bool warp_wait(unsigned long long *b, uint32_t parity, volatile int *abort, int *s) { return bar_wait(b, parity, abort, s); }
static void wait_drain(unsigned long long *b, uint32_t parity) {
    do yield();
    while (!bar_at(smem_u32(b)).passes(parity));
}
static void expect_tx(unsigned long long *b, uint32_t bytes) {
    Bar &x = bar_at(smem_u32(b));
    x.bytes += bytes;
    x.arrive();
}
static uint32_t meet(Control &ctl, uint32_t rank, uint32_t issued) {
    check(&ctl == &here().ctl && (int)rank == g_now->cta, "meets for another CTA");
    Cta &other = g_cta[rank ^ 1];
    later([&other, issued] { other.ctl.issued = issued; other.bars[&other.ctl.met].arrive(); }, true);
    wait_drain(&ctl.met, 0);
    return ctl.issued;
}
template <int PAIR>
static void arrive_cluster(uint32_t bar) {
    if (PAIR == 2) later([bar] { bar_at(bar).arrive(); }, true);
    else bar_at(bar).arrive();
}

// ---------------------------------------------------------------- copies, products, sums

static const MmArgs *g_args;
struct Tile { int expert, row0, row_end, col0; };
static std::vector<Tile> g_tiles;
template <int BN, int PAIR>
struct Tiles {
    size_t at = 0;
    explicit Tiles(const MmArgs &) {}
    bool next(Tile &t) {
        if (at == g_tiles.size()) return false;
        t = g_tiles[at++];
        return true;
    }
};

static void copy(uint32_t dst, Tag tag, uint32_t bar, int bytes) {
    Cta *c = &cta_at(dst);
    check(c == &here(), "copies to another CTA");
    c->ring.erase(dst & 0xFFFFFF);
    c->landing[dst & 0xFFFFFF]++;
    c->copies++;
    later([=] {
        c->ring[dst & 0xFFFFFF] = tag;
        c->landing[dst & 0xFFFFFF]--;
        c->copies--;
        Bar &b = bar_at(bar);
        b.bytes -= bytes;
        b.settle();
    });
    yield();
}
template <int PAIR>
static void tma_2d(uint32_t dst, const CUtensorMap *m, uint32_t bar, int x, int y) {
    copy(dst, {m->what, x, y, 0}, bar, g_args->a_box * kTileK);
}
template <int PAIR>
static void tma_3d(uint32_t dst, const CUtensorMap *m, uint32_t bar, int x, int y, int z) {
    copy(dst, {m->what, x, y, z}, bar, 128 * kTileK);
}

#include "desc.inc"
#include "scales.inc"

static Tag operand(Cta &c, uint64_t desc) {
    const uint32_t at = (uint32_t)(desc & 0x3FFF) << 4;
    auto it = c.ring.upper_bound(at);
    check(it != c.ring.begin(), "an operand that was never loaded");
    --it;
    check(!c.landing[it->first], "an operand that is being loaded");
    check(at - it->first < 128 * 128, "an operand that was never loaded");
    return it->second;
}
static bool g_trans;
static const Tile &tile_of(int row, int col) {
    for (const Tile &t : g_tiles)
        if (t.row0 == row && t.col0 <= col && col < t.col0 + 256) {
            const Tile *best = &t;
            for (const Tile &u : g_tiles)
                if (u.row0 == row && u.col0 <= col && u.col0 > best->col0) best = &u;
            return *best;
        }
    fail("no such tile");
}
struct Product { uint32_t d; uint64_t a, b; bool add; int pair; unsigned long long *commit; };
static std::map<Fibre *, std::deque<Product>> g_products;
// Where a wait runs out, the arrivals of one thread's commits come to a CTA in
// the order of the commits (the last one's then stands for all); elsewhere
// they may overtake one another.
static bool g_in_order;
static std::map<std::pair<Fibre *, int>, std::deque<uint32_t>> g_way;
static Sum means(const Product &q) {
    Sum s;
    for (int r = 0; r < q.pair; r++) {
        Cta &c = g_cta[g_cta.size() == 1 || q.pair == 1 ? g_now ? (size_t)g_now->cta : 0 : (size_t)r];
        const Tag b = operand(c, q.b);
        check(b.map == 'w', "not a weight");
        const int cb = (g_trans ? b.y : b.x) / 128, col = g_trans ? b.x : b.y;
        if (r == 0) {
            const Tag a = operand(c, q.a);
            check(a.map == 'a', "not rows");
            s.c = a.x / 128, s.row0 = a.y;
            s.col0 = tile_of(s.row0, col).col0;
            s.expert = b.z;
        }
        check(cb == s.c, "operands of two blocks");
        check(b.z == tile_of(s.row0, col).expert && tile_of(s.row0, col).col0 == s.col0, "operands of two tiles");
    }
    return s;
}
static bool same(const Sum &a, const Sum &b) { return a.c == b.c && a.row0 == b.row0 && a.col0 == b.col0 && a.expert == b.expert; }
static void run_product(Fibre *f) {
    std::deque<Product> &q = g_products[f];
    Product x = q.front();
    q.pop_front();
    g_now = f;
    if (x.commit) {
        const uint32_t at = smem_u32(x.commit);
        for (int r = 0; r < x.pair; r++) {
            const uint32_t to = x.pair == 2 ? ((uint32_t)r << 24) | (at & 0xFFFFFF) : at;
            if (!g_in_order) {
                later([to] { bar_at(to).arrive(); });
                continue;
            }
            std::deque<uint32_t> &way = g_way[{f, r}];
            way.push_back(to);
            later([&way] {
                const uint32_t first = way.front();
                way.pop_front();
                bar_at(first).arrive();
            });
        }
    } else {
        const Sum s = means(x);
        for (int r = 0; r < x.pair; r++) {
            Cta &c = x.pair == 2 ? g_cta[r] : g_cta[f->cta];
            c.waiting[x.d]--;
            Sum &to = c.tmem[x.d];
            if (!x.add) to = s, to.steps = 1;
            else check(same(to, s), "a sum of two blocks"), to.steps++;
        }
    }
    g_now = nullptr;
}
template <int PAIR>
static void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t, bool add) {
    const Product q{d, a, b, add, PAIR, nullptr};
    means(q);
    for (int r = 0; r < PAIR; r++) (PAIR == 2 ? g_cta[r] : here()).waiting[d]++;
    g_products[g_now].push_back(q);
}
template <int PAIR>
static void mma_commit(unsigned long long *b) {
    g_products[g_now].push_back({0, 0, 0, false, PAIR, b});
    yield();
}
static void fence_before() {}
static void fence_after() {}

// Sums are whole numbers times g_unit, scales whole numbers times powers of two,
// so that everything is exact: in f32's range, and with products of scales below and above it.
static float g_unit = 1.0f;
static float value(const Sum &s, int c) { return g_unit * (float)(1 + (c * 7 + s.row0 / 32 * 3 + s.col0 / 64 * 5 + s.expert) % 31); }
static void tmem_ld16(uint32_t addr, uint32_t r[16]) {
    const uint32_t d = (addr & 0xFFFF) / 128 * 128;
    const Sum s = here().tmem[d];
    check(s.steps == 4 && !here().waiting[d], "sums read while they are made");
    for (int i = 0; i < 16; i++) r[i] = __float_as_uint(value(s, s.c));
    yield();
}
static void tmem_wait_ld(uint32_t *) {}

static std::vector<float> g_sa, g_sb;
static std::map<std::pair<int, int>, int> g_stored;  // (row, column) of a warp's pieces
static float wanted(int row, int col, int c0, int c1, int pair_rows) {
    const int row0 = row - row % pair_rows;
    const Tile *t = nullptr;
    for (const Tile &u : g_tiles)
        if (u.row0 <= row && row < u.row_end && u.row0 + pair_rows > row && u.col0 <= col && (!t || u.col0 > t->col0)) t = &u;
    check(t, "a row of no tile");
    (void)row0;
    Sum s;
    s.row0 = t->row0, s.col0 = t->col0, s.expert = t->expert;
    double v = 0;
    for (int c = c0; c < c1; c++)
        v += (double)value(s, c) * ((double)g_sa[(size_t)row * g_args->a_scale_stride + c] *
                            g_sb[t->expert * g_args->w_scale_expert + (col < g_args->out ? col / 128 : t->col0 / 128) * g_args->w_scale_out +
                                 c * g_args->w_scale_in]);
    return (float)v;
}
static int g_tm;  // rows of a tile
template <int DT>
static void store_rows(const MmArgs &p, const CUtensorMap *, uint32_t, const float2 acc[32], int row0, int row_end, int col0) {
    check(row0 < row_end, "rows of nobody stored");
    if (col0 >= p.out) return;
    const float w = wanted(row0, col0, 0, p.blocks_c, g_tm);
    for (int i = 0; i < 32; i++) check(acc[i].x == w && acc[i].y == w, "wrong sums stored");
    g_stored[{row0, col0}]++;
    yield();
}
static void store_wait() {}
static void st_shared(uint32_t addr, float v) {
    Cta &c = cta_at(addr);
    check(&c == &here(), "sums left in another CTA");
    check(c.copies == 0, "sums left in a ring that copies come to");
    for (auto &w : c.waiting) check(w.second == 0, "sums left in a ring that products read");
    const uint32_t at = ((addr & 0xFFFFFF) - kRing) / 4, row = at % kTileM, col = at / kTileM;
    const Tile &t = g_tiles.at(0);
    const int part = g_now->cta, c0 = g_args->blocks_c * part / g_args->split, c1 = g_args->blocks_c * (part + 1) / g_args->split;
    if (t.col0 + (int)col < g_args->out) check(v == wanted(t.row0 + row, t.col0 + col, c0, c1, g_tm), "wrong sums left to be joined");
    g_stored[{t.row0 + (int)row, t.col0 + (int)col}]++;
}

// ---------------------------------------------------------------- the kernel's own text

template <int BN, int PAIR, bool TRANS, bool SPLIT>
static void kernel(int cta, int warp, const MmArgs &p) {
    using S = Shape<BN, PAIR>;
    Cta &me = g_cta[cta];
    Control &ctl = me.ctl;
    const struct { int x; } threadIdx{warp * 32};
    const int lane = 0, rank = PAIR == 2 ? cta : 0, part = SPLIT ? cta : 0;
    const uint32_t ring = ((uint32_t)cta << 24) + kRing, tmem = 0;
    const int c_begin = SPLIT ? p.blocks_c * part / p.split : 0;
    const int blocks = SPLIT ? p.blocks_c * (part + 1) / p.split - c_begin : p.blocks_c;
    const uint32_t stages = ring + S::kStages * S::kStageBytes;
    float *const slots = me.slots.data();
    volatile int *abort = &ctl.abort;
    const CUtensorMap map_a{'a'}, map_w{'w'}, map_d{'d'};
    (void)threadIdx, (void)lane, (void)part, (void)map_d;
#include "roles.inc"
}
template <int BN, int PAIR>
static void set_up(Control &ctl) {
    using S = Shape<BN, PAIR>;
    const struct { int x; } threadIdx{0};
#include "init.inc"
}

template <int BN, int PAIR, bool TRANS, bool SPLIT>
static void play(bool fault) {
    using S = Shape<BN, PAIR>;
    check(S::kSmem <= 227 * 1024, "more shared memory than there is");
    MmArgs p{};
    const int ctas = SPLIT ? (pick(2) ? 2 : 4) : PAIR;
    g_tm = kTileM * PAIR;
    g_trans = TRANS;
    p.split = SPLIT ? ctas : 1;
    const int choices[] = {1, 2, 3, 4, 5, 7, 8, 9, 12, 13, 33};
    p.blocks_c = SPLIT ? ctas * 2 + (int)pick(9) : choices[pick(11)];
    p.out = SPLIT ? 128 - 64 * (int)pick(2) : BN * 2 - (int)pick(2) * (BN / 2 + 60);
    p.n_experts = SPLIT ? 1 : 3;
    p.a_box = pick(2) ? 128 : 32;
    // tiles in the kernel's order, experts of ragged length
    const int lengths[] = {1, 33, 100, 128, 129, 200, 256, 300, 512};
    int row = 0;
    for (int e = 0; e < p.n_experts; e++) {
        const int n = SPLIT ? 1 + (int)pick(128) : lengths[pick(9)], first = row;
        for (int col = 0; col < p.out; col += BN)
            for (int r = first; r < first + n; r += g_tm) {
                g_tiles.push_back({e, r, first + n, col});
                if (SPLIT) break;
            }
        // what a CTA takes of them: a persistent grid's every third, say, or all
        row = first + (n + 511) / 512 * 512;
    }
    if (!SPLIT && pick(3) == 0) {
        std::vector<Tile> some;
        for (const Tile &t : g_tiles)
            if (pick(3) == 0) some.push_back(t);
        if (pick(20)) g_tiles = some.empty() ? std::vector<Tile>{g_tiles[0]} : some;
        else g_tiles.clear();  // offsets that leave this CTA nothing
    }
    p.n_rows = row;
    p.a_scale_stride = p.blocks_c;
    const int nb = (p.out + 127) / 128;
    p.w_scale_expert = nb * p.blocks_c, p.w_scale_out = p.blocks_c, p.w_scale_in = 1;
    g_sa.resize((size_t)row * p.blocks_c);
    g_sb.resize((size_t)p.n_experts * nb * p.blocks_c);
    for (float &v : g_sa) v = (float)(1 + pick(4));
    for (float &v : g_sb) v = (float)(1 + pick(4));
    const int range = (int)pick(3);  // the product of two scales: an ordinary number, a subnormal one, an infinite one
    g_unit = range == 2 ? 0x1p-18f : 1.0f;
    for (float &v : g_sa) v = ldexpf(v, range == 1 ? -80 : range == 2 ? 68 : 0);
    for (float &v : g_sb) v = ldexpf(v, range == 1 ? -60 : range == 2 ? 60 : 0);
    p.a_scales = g_sa.data(), p.w_scales = g_sb.data();
    const int types[] = {SHC_SRC_F32, SHC_SRC_F16, SHC_SRC_BF16};
    p.dst_type = types[pick(3)];
    g_args = &p;

    g_cta.resize(ctas);
    for (int c = 0; c < ctas; c++) {
        memset(&g_cta[c].ctl, 0, sizeof(Control));
        g_cta[c].slots.assign(kSlots * S::kSlotBytes / 4, -1.0f);
        Fibre f;
        f.cta = c;
        g_now = &f;
        set_up<BN, PAIR>(g_cta[c].ctl);
    }
    for (int c = 0; c < ctas; c++)
        for (int w = 0; w < S::kThreads / 32; w++) {
            Fibre *f = new Fibre;
            f->cta = c;
            f->stack.resize(256 * 1024);
            f->body = [c, w, &p] { kernel<BN, PAIR, TRANS, SPLIT>(c, w, p); };
            getcontext(&f->ctx);
            f->ctx.uc_stack.ss_sp = f->stack.data();
            f->ctx.uc_stack.ss_size = f->stack.size();
            f->ctx.uc_link = nullptr;
            makecontext(&f->ctx, run_fibre, 0);
            g_fibres.push_back(f);
        }
    // a product warp may be given few turns, or the copies, and so on
    std::vector<unsigned> weight(g_fibres.size());
    for (auto &w : weight) w = 1 + pick(4) * pick(8);
    const unsigned event_weight = 1 + pick(40), product_weight = 1 + pick(40);
    const uint64_t fault_at = fault ? 1 + pick(pick(2) ? 400 : 8000) : 0;
    for (uint64_t step = 1;; step++) {
        check(step < 5000000, "stuck");  // four times what the longest runs take
        if (step == fault_at) g_fibres[pick((unsigned)g_fibres.size())]->cut = true;
        size_t live = 0;
        for (Fibre *f : g_fibres) live += !f->over;
        if (!live) break;
        unsigned total = event_weight + product_weight;
        for (size_t i = 0; i < g_fibres.size(); i++) total += g_fibres[i]->over ? 0 : weight[i];
        unsigned at = pick(total);
        if (at < event_weight) {
            if (g_events.empty()) continue;
            const size_t i = pick((unsigned)g_events.size());
            auto e = g_events[i].what;
            g_events.erase(g_events.begin() + i);
            e();
            continue;
        }
        at -= event_weight;
        if (at < product_weight) {
            std::vector<Fibre *> some;
            for (auto &q : g_products)
                if (!q.second.empty()) some.push_back(q.first);
            if (!some.empty()) run_product(some[pick((unsigned)some.size())]);
            continue;
        }
        at -= product_weight;
        for (size_t i = 0; i < g_fibres.size(); i++) {
            if (g_fibres[i]->over) continue;
            if (at < weight[i]) {
                g_now = g_fibres[i];
                swapcontext(&g_main, &g_now->ctx);
                g_now = nullptr;
                break;
            }
            at -= weight[i];
        }
    }
    // All warps are at the kernel's end.
    for (auto &q : g_products) check(q.second.empty(), "a product is under way when its CTA ends");
    for (auto &e : g_events) check(e.ordered, "a copy or an arrival is under way when a CTA ends");
    bool gave_up = false;
    for (auto &c : g_cta) gave_up |= c.ctl.abort != 0;
    if (gave_up) {
        printf("gave up\n");
        return;
    }
    for (auto &s : g_stored) check(s.second == (SPLIT ? ctas : 1), "stored twice");
    size_t want = 0;
    for (const Tile &t : g_tiles)
        for (int r = t.row0; r < t.row_end && r < t.row0 + g_tm; r += 32)
            for (int col = t.col0; col < t.col0 + BN; col += SPLIT ? 1 : 64) want += SPLIT || col < p.out;
    check(g_stored.size() == want, "tiles left out");
    printf("done\n");
}

int main(int argc, char **argv) {
    if (argc != 4) return 2;
    const int shape = atoi(argv[1]);
    rng.seed((uint64_t)atoll(argv[2]) * 8 + shape);
    const bool fault = g_in_order = atoi(argv[3]) != 0;
    switch (shape) {
    case 0: play<128, 1, false, false>(fault); break;
    case 1: play<256, 1, false, false>(fault); break;
    case 2: play<256, 2, false, false>(fault); break;
    case 3: play<128, 1, false, true>(fault); break;
    case 4: play<128, 1, true, false>(fault); break;
    case 5: play<256, 1, true, false>(fault); break;
    case 6: play<256, 2, true, false>(fault); break;
    default: play<128, 1, true, true>(fault);
    }
    return 0;
}
