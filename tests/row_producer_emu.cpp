// The K and V producers of row_attn.cuh, compiled for the host: the kernel's own
// source block (row_producer_block.inc, cut out by the test) run by 32 threads as
// the lanes of a warp. Warp-wide operations meet at a rendezvous; one that can
// never fill because a lane has left, or waits at another operation, is a
// deadlock and is reported instead of waited for. Slots of the ring are free
// for `grants` waits, then the wait gives up and raises the abort flag, as a
// bounded wait of the kernel does.
//
//   row_producer_emu <tree 0|1> <kv 0|1> <grants>      exit 0: all lanes got out
#include <algorithm>
#include <atomic>
#include <condition_variable>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <thread>
#include <vector>

using std::min;

struct Deadlock {};

struct Warp {
  std::mutex mu;
  std::condition_variable cv;
  int waiting = 0, left = 0, kind = 0;
  long long round = 0;
  bool dead = false;
  uint32_t in[32], out[32];

  void check() {  // every lane has left or waits, but not all of them wait
    if (left > 0 && waiting > 0 && left + waiting == 32) { dead = true; cv.notify_all(); }
  }
  void leave() {
    std::lock_guard<std::mutex> l(mu);
    ++left;
    check();
  }
  // All lanes bring a value and take away every lane's.
  uint32_t meet(int lane, int what, uint32_t v, uint32_t (&all)[32]) {
    std::unique_lock<std::mutex> l(mu);
    if (waiting > 0 && kind != what) { dead = true; cv.notify_all(); }
    if (dead) throw Deadlock();
    kind = what;
    in[lane] = v;
    if (++waiting == 32) {
      std::copy(in, in + 32, out);
      waiting = 0;
      ++round;
      cv.notify_all();
    } else {
      const long long mine = round;
      check();
      cv.wait(l, [&] { return round != mine || dead; });
      if (round == mine) throw Deadlock();
    }
    std::copy(out, out + 32, all);
    return all[lane];
  }
};

Warp g_warp;
thread_local int t_lane;

void __syncwarp() { uint32_t a[32]; g_warp.meet(t_lane, 1, 0, a); }
bool __all_sync(unsigned, bool v) {
  uint32_t a[32];
  g_warp.meet(t_lane, 2, v, a);
  return std::all_of(a, a + 32, [](uint32_t x) { return x != 0; });
}
unsigned __ballot_sync(unsigned, bool v) {
  uint32_t a[32], bits = 0;
  g_warp.meet(t_lane, 3, v, a);
  for (int i = 0; i < 32; ++i) bits |= a[i] << i;
  return bits;
}
template <class T> T __shfl_sync(unsigned, T v, int from) {
  uint32_t a[32];
  g_warp.meet(t_lane, 4, uint32_t(v), a);
  return T(a[from]);
}
int __popc(unsigned v) { return __builtin_popcount(v); }

// ------------------------------------------------ what the block refers to ---
constexpr int D = 128, NK = 2, NV = 3, kDevBadInput = 2;
struct L {
  static constexpr int kHalves = 2;
  static constexpr uint32_t kHalf = 128 * 64 * 2, kTile = 2 * kHalf;
  static constexpr uint32_t kOffK = 0, kOffV = NK * kTile, kOffPages = kOffV + NV * kTile;
  static constexpr uint32_t kPageSlots = 128;
};
struct RowItem { int s, kh, key0, keys, t0, n; };
struct Params {
  int block_log2 = 4, block_size = 16, box_rows = 16, num_pages = 200, layer = 1, bt_len = 0;
  long long page_rows = 64, layer_rows = 32, kv_rows = 16;
  const int *bt = nullptr, *bt_off = nullptr;
  int* status = nullptr;
} p;
int table_entries(const Params& q, int s) { return q.bt_off[s + 1] - q.bt_off[s]; }
void atomicOr(int* to, int v) { __atomic_fetch_or(to, v, __ATOMIC_SEQ_CST); }

std::vector<RowItem> g_items;
volatile int g_abort = 0;
volatile int* abort_flag = &g_abort;
uint8_t smem[L::kOffPages + 2 * L::kPageSlots * 4];
uint64_t k_full[NK], k_empty[NK], v_full[NV], v_empty[NV];
int tmK, tmV;
int g_grants, g_kv;
std::mutex g_mu;
int g_waits = 0;
long long g_expect = 0, g_loaded = 0;
std::atomic<int> g_wrong{0};

void wrong(const char* what) {
  if (!g_wrong.exchange(1)) std::fprintf(stderr, "wrong: %s\n", what);
}
bool next_item(uint32_t ord, RowItem& it) {
  if (ord >= g_items.size()) return false;
  it = g_items[ord];
  return true;
}
void item_done(uint32_t) {}
bool row_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  std::lock_guard<std::mutex> l(g_mu);
  const int n = g_kv ? NV : NK;
  uint64_t* empty = g_kv ? v_empty : k_empty;
  if (bar != empty + g_waits % n || parity != ((uint32_t(g_waits / n) & 1) ^ 1)) wrong("slot");
  if (g_waits == g_grants) { *abort = 1; return false; }
  if (*abort) { wrong("a wait after giving up"); return false; }
  if (g_loaded != g_expect) wrong("a slot's bytes");
  ++g_waits;
  return true;
}
void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  std::lock_guard<std::mutex> l(g_mu);
  if (bar != (g_kv ? v_full : k_full) + (g_waits - 1) % (g_kv ? NV : NK)) wrong("full barrier");
  g_expect += bytes;
}
long long g_box;
void tma_load_2d(void* dst, const void* map, uint64_t* bar, int, int row) {
  std::lock_guard<std::mutex> l(g_mu);
  const uint32_t slot = (g_waits - 1) % (g_kv ? NV : NK);
  const uint64_t at = static_cast<uint8_t*>(dst) - smem;
  const uint64_t tile = (g_kv ? L::kOffV : L::kOffK) + slot * L::kTile;
  if (bar != (g_kv ? v_full : k_full) + slot || map != (g_kv ? &tmV : &tmK)) wrong("barrier or map");
  if (at < tile || at + g_box > tile + L::kTile || row < 0) wrong("place");
  g_loaded += g_box;
  if (g_loaded > g_expect) wrong("loaded before it was announced");
}

template <bool TREE>
void produce(const int warp, const int lane) {
#include "row_producer_block.inc"
}

int main(int argc, char** argv) {
  if (argc != 4) return 2;
  const bool tree = std::atoi(argv[1]) != 0;
  g_kv = std::atoi(argv[2]);
  g_grants = std::atoi(argv[3]);
  // long, short, one of a single ragged tile; pages of 16, the table of the
  // third sequence ends early (those boxes are left out)
  g_items = {{0, 0, 0, 2500, 0, 20}, {1, 0, 2500, 260, 1, 2}, {2, 0, 2760, 70, 0, 1}};
  std::vector<int> bt(160 + 17 + 3), off = {0, 160, 177, 180};
  for (size_t i = 0; i < bt.size(); ++i) bt[i] = int(i * 7 % 200);
  int status = 0;
  p.bt = bt.data();
  p.bt_off = off.data();
  p.bt_len = int(bt.size());
  p.status = &status;
  g_box = (tree ? p.box_rows : 128) * 64 * 2;
  std::atomic<int> stuck{0};
  std::vector<std::thread> lanes;
  for (int i = 0; i < 32; ++i)
    lanes.emplace_back([&, i] {
      t_lane = i;
      try {
        if (tree) produce<true>(g_kv ? 14 : 10, i);
        else produce<false>(g_kv ? 14 : 10, i);
      } catch (const Deadlock&) {
        ++stuck;
      }
      g_warp.leave();
    });
  for (auto& t : lanes) t.join();
  if (stuck) std::fprintf(stderr, "deadlock: %d lanes wait for ones that have left\n", int(stuck));
  if (!stuck && g_loaded != g_expect) wrong("bytes at the end");
  const int tiles = 20 + 2 + 1;
  if (!stuck && g_waits != std::min(g_grants, tiles)) wrong("tiles");
  if (!stuck && tree && g_grants >= tiles && status != kDevBadInput) wrong("status");
  std::printf("%d tiles\n", g_waits);
  return stuck ? 1 : g_wrong ? 3 : 0;
}
