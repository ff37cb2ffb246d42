// The normalisation's host path and kernels on the CPU on given values, for a test that compares the results.
//   norm_values walk N C H W groups type [workgroups]
//     blocks and workgroups of a sample's tile in the passes: statistics, apply, apply into channel quads, gradients'
//     sums, input gradient; then tiles of the statistics, and 1 where a pass takes the small maps' one launch
//   norm_values run N C H W groups type workgroups act < x dy weight bias > y q scale [packed] dx dw db dx dw db
//     (in memory order, parameters fp32; packed where fp32 and C % 4 == 0; the gradients from x, then from q)
// Workgroups: of the statistics, the gradients' sums, the apply pass and the input gradient, in place of the source's
// own (whose constants the build made variables).  Buffers lie between pages that fault, as in norm_bounds.cpp, whose parts these are.
#define main norm_bounds_main
#include "norm_bounds.cpp"
#undef main

static void get(Buffer& b) {
  if (fread(b.p, 1, b.n, stdin) != b.n) cpu::fail("input cut short");
}
static void put(const Buffer& b) { fwrite(b.p, 1, b.n, stdout); }

static int walk(const DpftGroupNorm& d) {
  if (check(&d) != DPFT_OK) return 1;
  const Walk w[] = {make_walk(d, kDeep, kStatsWorkgroups), make_walk(d, kDeepApply, kApplyWorkgroups),
                    make_walk(d, kDeepApply, kApplyWorkgroups, kPackedSlots), make_walk(d, kDeepSums, kSumsWorkgroups),
                    make_walk(d, kDeepGrad, kGradWorkgroups)};
  for (const Walk& a : w) printf("%d %d ", a.blocks, a.parts);
  printf("%d %d\n", w[0].tiles, (make_slice(d, kSmallHold).cw || make_slice(d, kSmallHold / 2).cw) ? 1 : 0);
  return 0;
}

static int run(DpftGroupNorm d) {
  const size_t n = (size_t)d.N * d.C * d.pixels, size = d.x_type ? 2 : 4, groups = (size_t)d.N * d.groups * 4;
  const size_t ws_bytes = dpft_group_norm_workspace_size(&d);
  if (!ws_bytes) return 1;
  const bool up = true;
  Buffer x(n * size, up, 0), dy(n * size, up, 0), w(d.C * 4, up, 0), b(d.C * 4, up, 0), ws(ws_bytes, up, 0xff);
  Buffer y(n * size, up, 0x5a), y2(n * size, up, 0x5a), mean(groups, up, 0x5a), rstd(groups, up, 0x5a);
  Buffer q(n, up, 0x5a), scale((n + 31) / 32, up, 0x5a), dx(n * size, up, 0x5a), dw(d.C * 4, up, 0x5a), db(d.C * 4, up, 0x5a);
  get(x), get(dy), get(w), get(b);
  auto at = [&](const char* call) {
    snprintf(g_what, sizeof g_what, "%s", call);
    ws.clear();
  };
  auto ok = [&](int rc) {
    if (rc) cpu::fail("refused");
    for (const Buffer* t : {&x, &dy, &w, &b, &ws, &y, &y2, &mean, &rstd, &q, &scale, &dx, &dw, &db})
      if (!t->clean()) cpu::fail("a write beside a buffer");
  };
  float *mu = reinterpret_cast<float*>(mean.p), *rs = reinterpret_cast<float*>(rstd.p);
  int8_t* q8 = reinterpret_cast<int8_t*>(q.p);
  uint8_t* s8 = reinterpret_cast<uint8_t*>(scale.p);
  at("forward");
  ok(dpft_group_norm_act(&d, x.p, w.p, b.p, y2.p, nullptr, nullptr, nullptr, nullptr, ws.p, ws_bytes, nullptr));
  at("forward with a checkpoint");
  ok(dpft_group_norm_act(&d, x.p, w.p, b.p, y.p, mu, rs, q8, s8, ws.p, ws_bytes, nullptr));
  if (memcmp(y.p, y2.p, y.n)) cpu::fail("another y");
  put(y), put(q), put(scale);
  if (d.x_type == DPFT_TYPE_F32 && d.C % 4 == 0) {
    at("packed");
    d.flags = DPFT_GN_PACKED;
    y2.clear();
    ok(dpft_group_norm_act(&d, x.p, w.p, b.p, y2.p, nullptr, nullptr, nullptr, nullptr, ws.p, ws_bytes, nullptr));
    d.flags = 0;
    put(y2);
  }
  for (bool from_q : {false, true}) {
    at(from_q ? "backward from a checkpoint" : "backward");
    dx.clear(), dw.clear(), db.clear();
    ok(dpft_group_norm_act_backward(&d, dy.p, from_q ? nullptr : x.p, from_q ? q8 : nullptr, from_q ? s8 : nullptr, w.p, b.p, mu,
                                    rs, dx.p, dw.p, db.p, ws.p, ws_bytes, nullptr));
    put(dx), put(dw), put(db);
  }
  return 0;
}

int main(int argc, char** argv) {
  stack_t own{};
  own.ss_sp = malloc(1 << 16);
  own.ss_size = 1 << 16;
  sigaltstack(&own, nullptr);
  struct sigaction act {};
  act.sa_sigaction = on_fault;
  act.sa_flags = SA_SIGINFO | SA_ONSTACK;
  sigaction(SIGSEGV, &act, nullptr);
  sigaction(SIGBUS, &act, nullptr);
  const bool runs = argc == 13 && !strcmp(argv[1], "run");
  if (!runs && ((argc != 8 && argc != 12) || strcmp(argv[1], "walk"))) return 2;
  DpftGroupNorm d{};
  d.N = atoi(argv[2]);
  d.C = atoi(argv[3]);
  d.pixels = (int64_t)atoi(argv[4]) * atoi(argv[5]);
  d.groups = atoi(argv[6]);
  d.x_type = atoi(argv[7]);
  if (argc > 8) {
    kStatsWorkgroups = atoi(argv[8]);
    kSumsWorkgroups = atoi(argv[9]);
    kApplyWorkgroups = atoi(argv[10]);
    kGradWorkgroups = atoi(argv[11]);
  }
  d.act = runs ? atoi(argv[12]) : DPFT_ACT_NONE;
  d.eps = 1e-5f;
  return runs ? run(d) : walk(d);
}
