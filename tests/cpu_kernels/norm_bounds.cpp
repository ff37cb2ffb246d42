// dpft_norm.hip on the CPU, its buffers between pages that fault: every entry point at the sizes on stdin
// (N C H W groups), every type, buffers against the page above and against the page below.  Ends with 0 and a
// count if no access leaves its buffer, every barrier is met and every result is written.
#include <signal.h>
#include <sys/mman.h>
#include <unistd.h>

#include <cstdarg>

#include "../../deep_prob_feature_track_amd/csrc/dpft_norm.hip"

static char g_what[512];

namespace cpu {
std::vector<Thread> threads;
ucontext_t scheduler;
int current, alive, arrived, generation;
static std::function<void()> g_kernel;

void fail(const char* why) {
  fprintf(stderr, "%s: %s, workgroup %u thread %d\n", why, g_what, blockIdx.x, current);
  _exit(1);
}
static void entry() {
  g_kernel();
  threads[current].done = true;
  if (--alive && arrived == alive) {
    arrived = 0;
    ++generation;
    for (auto& t : threads) t.sent.clear();
  }
  for (;;) yield();
}
void run(unsigned grid, int n, std::function<void()> kernel) {
  constexpr size_t kStack = 1 << 16;
  static char* stacks = static_cast<char*>(malloc(512 * kStack));
  g_kernel = kernel;
  threads.resize(n);
  gridDim.x = grid;
  for (blockIdx.x = 0; blockIdx.x < grid; ++blockIdx.x) {
    alive = n;
    arrived = 0;
    for (int t = 0; t < n; ++t) {
      threads[t].sent.clear();
      threads[t].done = false;
      getcontext(&threads[t].context);
      threads[t].context.uc_stack.ss_sp = stacks + t * kStack;
      threads[t].context.uc_stack.ss_size = kStack;
      threads[t].context.uc_link = nullptr;
      makecontext(&threads[t].context, entry, 0);
    }
    for (long rounds = 0; alive; ++rounds) {
      if (rounds > 100000000) fail("a wait that does not end");
      for (current = 0; current < n; ++current)
        if (!threads[current].done) swapcontext(&scheduler, &threads[current].context);
    }
  }
}
}  // namespace cpu
cpu::Index blockIdx, gridDim;
ThreadIndex threadIdx;

int dpft_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vfprintf(stderr, fmt, ap);
  va_end(ap);
  return code;
}
int dpft_hip_check(const char*) { return DPFT_OK; }

static void on_fault(int, siginfo_t*, void*) { cpu::fail("access out of range"); }

// 16-byte aligned, at the upper or the lower end of its pages; `blank` around it and, at first, in it.
struct Buffer {
  static constexpr size_t kGuard = 1 << 20;
  char *base, *p;
  size_t n, pages;
  int blank;
  Buffer(size_t bytes, bool upper, int fill) : n(bytes), blank(fill) {
    const size_t held = (std::max<size_t>(n, 1) + 15) / 16 * 16;
    pages = (held + 4095) / 4096 * 4096;
    base = static_cast<char*>(mmap(nullptr, pages + 2 * kGuard, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
    mprotect(base + kGuard, pages, PROT_READ | PROT_WRITE);
    p = base + kGuard + (upper ? pages - held : 0);
    memset(base + kGuard, blank, pages);
  }
  ~Buffer() { munmap(base, pages + 2 * kGuard); }
  bool clean() const {  // nothing written beside it
    for (char* c = base + kGuard; c < base + kGuard + pages; ++c)
      if ((c < p || c >= p + n) && *c != (char)blank) return false;
    return true;
  }
  void clear() { memset(p, blank, n); }
  template <typename T>
  void values(unsigned seed) {
    for (size_t i = 0; i < n / sizeof(T); ++i) {
      seed = seed * 1664525u + 1013904223u;
      reinterpret_cast<T*>(p)[i] = (T)((float)(seed >> 8) / (1 << 23) - 1.0f);
    }
  }
  void values(int type, unsigned seed) {
    if (type == DPFT_TYPE_F32) values<float>(seed);
    else if (type == DPFT_TYPE_BF16) values<__bf16>(seed);
    else values<_Float16>(seed);
  }
  template <typename T>
  bool written() const {  // a blank value is 1.5e16 in fp32 and bf16, 203 in fp16
    for (size_t i = 0; i < n / sizeof(T); ++i)
      if (!(std::fabs((float)reinterpret_cast<T*>(p)[i]) < (std::is_same_v<T, _Float16> ? 150.0f : 1e4f))) return false;
    return true;
  }
  bool written(int type) const {
    return type == DPFT_TYPE_F32 ? written<float>() : type == DPFT_TYPE_BF16 ? written<__bf16>() : written<_Float16>();
  }
};

static void one(int N, int C, int H, int W, int G, int type, bool upper) {
  const size_t n = (size_t)N * C * H * W, size = type ? 2 : 4, blocks = (n + 31) / 32;
  DpftGroupNorm d{};
  d.pixels = (int64_t)H * W;
  d.N = N;
  d.C = C;
  d.groups = G;
  d.act = DPFT_ACT_ELU;
  d.x_type = type;
  d.param_type = type == DPFT_TYPE_F16 ? DPFT_TYPE_BF16 : DPFT_TYPE_F32;
  d.eps = 1e-5f;
  const size_t psize = d.param_type ? 2 : 4, ws_bytes = dpft_group_norm_workspace_size(&d);
  Buffer x(n * size, upper, 0), dy(n * size, upper, 0), w(C * psize, upper, 0), b(C * psize, upper, 0);
  Buffer y(n * size, upper, 0x5a), dx(n * size, upper, 0x5a), dw(C * psize, upper, 0x5a), db(C * psize, upper, 0x5a);
  Buffer mean(N * G * 4, upper, 0x5a), rstd(N * G * 4, upper, 0x5a), q(n, upper, 0x5a), scale(blocks, upper, 0x5a);
  Buffer ws(ws_bytes, upper, 0xff);
  x.values(type, 1);
  dy.values(type, 2);
  w.values(d.param_type, 3);
  b.values(d.param_type, 4);
  auto at = [&](const char* call) {
    snprintf(g_what, sizeof g_what, "N %d C %d H %d W %d groups %d type %d %s, %s", N, C, H, W, G, type, upper ? "upper" : "lower",
             call);
    ws.clear();
  };
  auto check = [&](int rc) {
    if (rc) cpu::fail("refused");
    for (const Buffer* t : {&x, &dy, &w, &b, &y, &dx, &dw, &db, &mean, &rstd, &q, &scale, &ws})
      if (!t->clean()) cpu::fail("a write beside a buffer");
  };
  float *mu = reinterpret_cast<float*>(mean.p), *rs = reinterpret_cast<float*>(rstd.p);
  int8_t* q8 = reinterpret_cast<int8_t*>(q.p);
  uint8_t* s8 = reinterpret_cast<uint8_t*>(scale.p);

  at("forward");
  check(dpft_group_norm_act(&d, x.p, w.p, b.p, y.p, nullptr, nullptr, nullptr, nullptr, ws.p, ws_bytes, nullptr));
  if (!y.written(type)) cpu::fail("a value not written");
  const std::vector<char> y0(y.p, y.p + y.n);
  at("forward with a checkpoint");
  y.clear();
  check(dpft_group_norm_act(&d, x.p, w.p, b.p, y.p, mu, rs, q8, s8, ws.p, ws_bytes, nullptr));
  if (memcmp(y0.data(), y.p, y.n)) cpu::fail("another y");
  const std::vector<char> q0(q.p, q.p + q.n), s0(scale.p, scale.p + scale.n);
  at("checkpoint");
  q.clear();
  scale.clear();
  check(dpft_act_checkpoint(x.p, type, n, q8, s8, nullptr));
  if (memcmp(q0.data(), q.p, q.n) || memcmp(s0.data(), scale.p, scale.n)) cpu::fail("another checkpoint");
  at("restore");
  y.clear();
  check(dpft_act_restore(q8, s8, n, y.p, type, nullptr));
  if (!y.written(type)) cpu::fail("a value not written");
  if (type == DPFT_TYPE_F32 && C % 4 == 0) {
    at("packed");
    y.clear();
    d.flags = DPFT_GN_PACKED;
    check(dpft_group_norm_act(&d, x.p, w.p, b.p, y.p, nullptr, nullptr, nullptr, nullptr, ws.p, ws_bytes, nullptr));
    if (!y.written(type)) cpu::fail("a value not written");
    d.flags = 0;
  }
  for (int want : {7, 1, 2, 4, 0})
    for (bool from_q : {false, true}) {
      at(from_q ? "backward from a checkpoint" : "backward");
      dx.clear();
      dw.clear();
      db.clear();
      check(dpft_group_norm_act_backward(&d, dy.p, from_q ? nullptr : x.p, from_q ? q8 : nullptr, from_q ? s8 : nullptr, w.p, b.p,
                                         mu, rs, want & 1 ? dx.p : nullptr, want & 2 ? dw.p : nullptr,
                                         want & 4 ? db.p : nullptr, ws.p, ws_bytes, nullptr));
      if ((want & 1 && !dx.written(type)) || (want & 2 && !dw.written(d.param_type)) || (want & 4 && !db.written(d.param_type)))
        cpu::fail("a value not written");
    }
}

int main() {
  stack_t own{};
  own.ss_sp = malloc(1 << 16);
  own.ss_size = 1 << 16;
  sigaltstack(&own, nullptr);
  struct sigaction act {};
  act.sa_sigaction = on_fault;
  act.sa_flags = SA_SIGINFO | SA_ONSTACK;
  sigaction(SIGSEGV, &act, nullptr);
  sigaction(SIGBUS, &act, nullptr);
  int N, C, H, W, G, count = 0;
  while (scanf("%d %d %d %d %d", &N, &C, &H, &W, &G) == 5)
    for (int type : {DPFT_TYPE_F32, DPFT_TYPE_BF16, DPFT_TYPE_F16})
      for (bool upper : {true, false}) {
        one(N, C, H, W, G, type, upper);
        ++count;
      }
  printf("%d\n", count);
}
