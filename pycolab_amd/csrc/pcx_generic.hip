// pcx_generic.hip -- table-driven step kernel for games whose entities are
// plain Sprites, MazeWalkers (no scrolling) and ordinary Drapes:
//   examples/warehouse_manager.py, examples/extraterrestrial_marauders.py,
//   examples/hello_world.py  (reference: engine.py:583-847 around them).
// gfx950 only.
//
// Same two-phase shape as pcx_scrolly_maze.hip: a workgroup is one
// wavefront that owns 64 consecutive environments.
//   * logic phase, lane == environment: state words are loaded SoA-coalesced,
//     entity state lives in per-lane LDS columns (so the update schedule, the
//     z-order and the entity programs can be walked with ordinary loops over
//     tables), every engine.py:735 repaint is a *snapshot* (sprite cells +
//     curtains) that board/layer probes evaluate lazily;
//   * render phase: occlusion is resolved once per environment, then the wave
//     streams board + layers with coalesced dword stores.
// Curtains are bit-rows (RW words per row) while the logic runs -- np.roll of
// a MarauderDrape or RollingDrape is a rotate -- and are flattened to cell-bit
// vectors for the render phase.

#include "pcx_internal.h"
#include "pcx_crop_window.h"
#include "pcx_stream.h"
#include "pcx_generic_kernel.h"

#include "pcx_rtc.h"  // hiprtc + the cache of code objects, shared with pcx_scrolly_maze.hip

#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>

#include "build/pcx_generic_rtc.inc"  // RTC_NAMES / RTC_SOURCES: this file's device-side headers as text (csrc/Makefile, tools/embed_sources.py)

namespace pcx {
namespace gen {

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

// The header a specialised build includes (PCX_GENERIC_SPEC): Consts member by member in declaration order, then the
// staged tables.  (sizeof is checked so that a member added to Consts cannot be forgotten here.)
static std::string spec_header(const Consts& k, const std::vector<uint32_t>& tab, bool sregs) {
  static_assert(sizeof(Consts) == 4 * (16 + 1 + 3 + 1 + 1 + 7 + 2 + 1 + PCX_MAX_SCROLL_GROUPS + 2 + 2 + 1 + 3 + 2 + 1 + 11 + 14 + 4) + PCX_MAX_CHARS,
                "Consts changed: update spec_header()");
  // (PCX_SPEC_NS: the sprite count for the preprocessor -- pcx_generic_kernel.h decides by it whether the sprites' state lives in registers)
  std::string o = "// generated by GenericBackend (pcx_generic.hip spec_header)\n";
  // (with the sprites in registers: 128 VGPRs -- four waves per SIMD -- instead of 96; LDS admits 8-12 workgroups per CU anyway)
  if (sregs) o += "#define PCX_SPEC_SREGS 1\n#ifndef PCX_X_WPE\n#define PCX_X_WPE 4\n#endif\n";
  o += "static constexpr Consts K = {";
  auto i32 = [&](int32_t v) { o += std::to_string(v); o += ", "; };
  auto u32 = [&](uint32_t v) { o += std::to_string(v); o += "u, "; };
  for (int32_t v : {k.game, k.R, k.C, k.cells, k.pitch, k.QW, k.L, k.NS, k.ND, k.NT, k.n_groups, k.RW, k.FW, k.NW, k.n_actions, k.n_bchars,
                    k.occl, k.n_dir, k.zdyn, k.w_z, k.w_next, k.reward_float, k.l_dir, k.l_zord, k.l_zabove, k.l_zabove_s, k.l_zabove_d, k.l_zq, k.l_ztmp,
                    k.has_scroll, k.w_scroll, k.n_sgroups}) i32(v);
  o += "{";
  for (int g = 0; g < PCX_MAX_SCROLL_GROUPS; ++g) u32(k.group_sprites[g]);
  o += "}, ";
  u32(k.magic_q); u32(k.magic_c);
  for (int32_t v : {k.w_sflags, k.w_drapes, k.ip, k.ix, k.ib, k.tx, k.bolt_mask_all, k.bolt_mask_up, k.box_mask,
                    k.l_things, k.l_z, k.l_sched, k.l_backdrop, k.l_bdmask, k.l_aux, k.l_init, k.l_initd, k.l_laybc, k.l_s2t, k.l_d2t,
                    k.l_pos, k.l_flg, k.l_snap, k.l_cur, k.l_snapd, k.l_flat, k.l_sdesc, k.l_skip, k.l_flatraw, k.l_sdescraw, k.l_corner,
                    k.l_pmask, k.l_pframe, k.l_words, k.l_wcorner, k.l_inbox, k.l_bdcode, k.l_codes}) i32(v);
  o += "{";
  for (int i = 0; i < PCX_MAX_CHARS; ++i) { o += std::to_string((int)k.chars[i]); o += ", "; }
  o += "}};\nstatic constexpr uint32_t TAB[] = {";
  for (size_t i = 0; i < tab.size(); ++i) { if (i % 16 == 0) o += "\n  "; o += std::to_string(tab[i]); o += "u, "; }
  if (tab.empty()) o += "0u";
  o += "};\n";
  return o;
}

// ---- run-time specialisation -----------------------------------------------------------------------------------
// pcx_generic_step is an interpreter: the update schedule, every entity's program, its table entry, the z-order and
// all loop bounds are data.  For ONE template they are constants, and a build of the same source with those constants
// in (pcx_generic_kernel.h PCX_GENERIC_SPEC) lets the compiler evaluate the interpreter away: 38-63 KB of code instead
// of 150, no scratch, 44-96 VGPRs, 1.3-2.6 times faster on the fixtures of tools/generic_timing.py
// (profiles/r04_generic_spec.md).  hiprtc (part of the ROCm runtime; dlopen'ed, no link dependency) compiles it in
// 1-3 s when a large engine is created; the code object is kept in memory per (template, device) and on disk
// ($PCX_JIT_CACHE, default <directory of libpcx.so>/jit_cache), keyed by a hash of everything that goes into it.
// Anything that fails on the way -- no libhiprtc, a compile error, an unwritable cache -- leaves the engine on the
// table-driven build (same results, PCX_DEBUG & 16 prints why); pcx_engine_launch_shape tells which one runs (30 / 31).
namespace rtc {

static const char* const OPTIONS[] = {"--offload-arch=gfx950", "-O3", "-std=c++17", PCX_RTC_NO_PACKED_FP32, "-DPCX_GENERIC_SPEC=\"pcx_generic_spec.h\""};
constexpr int N_OPTIONS = sizeof OPTIONS / sizeof OPTIONS[0];

static const char* const TU = "#include \"pcx_generic_kernel.h\"\n";
static const pcx::rtc::Program PROGRAM = {RTC_NAMES, RTC_SOURCES, RTC_COUNT, TU, "pcx_generic_spec.hip", OPTIONS, N_OPTIONS, "pcx_generic_spec.h", "pcx_generic", "pcx generic"};
using pcx::rtc::fnv;
// PCX_GENERIC_SPEC_DEFS="-DX=1 -DY": extra options of the run-time build (A/B runs of kernel variants on one box: the options are
// part of the cache key, so every variant is its own entry)
static std::vector<char> code_object(const std::string& spec, std::string& why, bool verbose, bool read_cache = true, bool* from_cache = nullptr) {
  const char* extra = getenv("PCX_GENERIC_SPEC_DEFS");
  const char* pw = getenv("PCX_GENERIC_PW");  // the opt-in persistent-worker kernel rides along only when asked for (it doubles the compile time)
  const bool with_pw = pw && atoi(pw) != 0;
  if ((!extra || !*extra) && !with_pw) return pcx::rtc::code_object(PROGRAM, spec, why, verbose, read_cache, from_cache);
  if (!extra) extra = "";
  std::vector<std::string> words;
  if (with_pw) words.emplace_back("-DPCX_GENERIC_WITH_PW=1");
  for (const char* p = extra; *p;) {
    while (*p == ' ') ++p;
    const char* q = p;
    while (*q && *q != ' ') ++q;
    if (q > p) words.emplace_back(p, q);
    p = q;
  }
  std::vector<const char*> opts(OPTIONS, OPTIONS + N_OPTIONS);
  for (const std::string& w : words) opts.push_back(w.c_str());
  pcx::rtc::Program prog = PROGRAM;
  prog.options = opts.data();
  prog.n_options = (int)opts.size();
  return pcx::rtc::code_object(prog, spec, why, verbose, read_cache, from_cache);
}

struct Loaded { hipModule_t mod = nullptr; hipFunction_t fn = nullptr, fn_pw = nullptr; int vgprs = 0; };  // fn_pw: pcx_generic_step_pw (null in code objects of rounds 4-5)

// One module per (constants, device) and process; never unloaded (engines come and go, the code stays).
static const Loaded* load(const std::string& spec, int device, std::string& why, bool verbose) {
  static std::mutex mu;
  static std::map<std::pair<uint64_t, int>, Loaded> mods;
  uint64_t key = fnv(0xCBF29CE484222325ull, spec.data(), spec.size());
  if (const char* extra = getenv("PCX_GENERIC_SPEC_DEFS")) key = fnv(key, extra, strlen(extra));
  if (const char* pw = getenv("PCX_GENERIC_PW")) if (atoi(pw) != 0) key = fnv(key, "pw", 2);
  std::lock_guard<std::mutex> lock(mu);
  auto it = mods.find({key, device});
  if (it != mods.end()) return it->second.fn ? &it->second : nullptr;
  Loaded l;
  for (int attempt = 0; attempt < 2 && !l.fn; ++attempt) {
    bool cached = false;
    const std::vector<char> code = code_object(spec, why, verbose, /*read_cache=*/attempt == 0, &cached);
    if (code.empty()) break;
    l = Loaded{};
    if (hipModuleLoadData(&l.mod, code.data()) != hipSuccess) { why = "hipModuleLoadData failed"; l.mod = nullptr; (void)hipGetLastError(); }
    else if (hipModuleGetFunction(&l.fn, l.mod, "pcx_generic_step") != hipSuccess) { why = "the code object has no pcx_generic_step"; l.fn = nullptr; (void)hipGetLastError(); }
    else if (hipFuncGetAttribute(&l.vgprs, HIP_FUNC_ATTRIBUTE_NUM_REGS, l.fn) != hipSuccess) { l.vgprs = 0; (void)hipGetLastError(); }
    if (l.fn && hipModuleGetFunction(&l.fn_pw, l.mod, "pcx_generic_step_pw") != hipSuccess) { l.fn_pw = nullptr; (void)hipGetLastError(); }
    if (!cached) break;  // (freshly compiled: a second compile would give the same)
  }
  auto& slot = mods[{key, device}];
  slot = l;
  return slot.fn ? &slot : nullptr;
}

}  // namespace rtc

// Waves per workgroup, measured.  How many waves should share a group's render loop depends on the template in ways
// no rule caught (profiles/r04_generic_spec.md: at 262,144 environments warehouse_L0 wants 4, walkers_scroll_groups 2,
// walkers_room 1, hello_world and better_scrolly_custom_B 8 -- up to 1.4 x between the best and the rule's choice), and
// the result does not depend on it, so the engine finds out on its own launches: after WARM step launches on the rule's
// choice every candidate runs REPS launches between two events on the launch stream; once the last of them has
// completed (polled, never waited for) the candidate with the smallest median stays.  Launches under stream capture,
// reset launches and PCX_GENERIC_WAVES leave the tuner alone; PCX_GENERIC_TUNE=0 turns it off.
struct Tuner {
  static constexpr int WARM = 6, REPS = 3, NC = 8;  // (round 6: four wave counts x {owner codes, masks}; `nc` of them are tried)
  int nc = 4;
  int phase = 0;      // step launches seen
  int chosen = 0;     // > 0: settled
  bool off = false, measuring = false;
  hipEvent_t ev[NC * REPS][2] = {};
  bool have_events = false;
  ~Tuner() { drop(); }
  void drop() {
    if (have_events) for (auto& e : ev) { (void)hipEventDestroy(e[0]); (void)hipEventDestroy(e[1]); }
    have_events = false;
  }
  bool done() const { return off || chosen > 0 || phase == 0; }
  void restart() { drop(); phase = 0; chosen = 0; measuring = false; }  // the launch's work changed (an epilogue, fused croppers): measure again
  // waves per workgroup 1, 2, 4, 8 in the low byte; bit 8: the mask-composing render loop instead of owner codes (tried only
  // where a launch may render from codes: nc == 8)
  static int candidate(int i) { return (1 << (i & 3)) | ((i >> 2) << 8); }
  int pick(int rule, const StepArgs& a, hipStream_t s) {
    measuring = false;
    if (chosen > 0) return chosen;
    if (off || a.mode != 0) return rule;
    if (phase == 0) {
      const char* e = getenv("PCX_GENERIC_TUNE");
      if (e && atoi(e) == 0) { off = true; return rule; }
    }
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &cap) != hipSuccess || cap != hipStreamCaptureStatusNone) { (void)hipGetLastError(); return rule; }
    const int i = phase - WARM;
    if (i < 0) { ++phase; return rule; }
    if (i < nc * REPS) {
      if (!have_events) {
        for (auto& e : ev)
          if (hipEventCreate(&e[0]) != hipSuccess || hipEventCreate(&e[1]) != hipSuccess) { (void)hipGetLastError(); off = true; return rule; }
        have_events = true;
      }
      if (hipEventRecord(ev[i][0], s) != hipSuccess) { (void)hipGetLastError(); off = true; return rule; }
      measuring = true;
      return candidate(i / REPS);
    }
    // all measured: settle as soon as the last launch has completed
    if (hipEventQuery(ev[nc * REPS - 1][1]) != hipSuccess) { (void)hipGetLastError(); return rule; }
    float best = 0.0f;
    for (int c = 0; c < nc; ++c) {
      float t[REPS];
      for (int r = 0; r < REPS; ++r)
        if (hipEventElapsedTime(&t[r], ev[c * REPS + r][0], ev[c * REPS + r][1]) != hipSuccess) { (void)hipGetLastError(); off = true; drop(); return rule; }
      for (int x = 0; x < REPS; ++x) for (int y = x + 1; y < REPS; ++y) if (t[y] < t[x]) { const float q = t[x]; t[x] = t[y]; t[y] = q; }
      const float med = t[REPS / 2];
      if (chosen == 0 || med < best) { best = med; chosen = candidate(c); }
    }
    drop();
    const char* dbg = getenv("PCX_DEBUG");
    if (dbg && (atoi(dbg) & 16)) fprintf(stderr, "[pcx generic] waves per workgroup: %d, render loop: %s (the rule said %d; median %.4f ms)\n", chosen & 0xFF, (chosen & 0x100) ? "masks" : nc == 8 ? "owner codes" : "as the launch allows", rule, best);
    return chosen;
  }
  void launched(hipStream_t s) {
    if (!measuring) return;
    const int i = phase - WARM;
    if (hipEventRecord(ev[i][1], s) != hipSuccess) { (void)hipGetLastError(); off = true; }
    ++phase;
    measuring = false;
  }
};

class GenericBackend : public Backend {
 public:
  int init(const pcx_template& t, int64_t batch) override;
  int plan(const pcx_template& t, int64_t batch);
  // include/pcx.h pcx_generic_specialise_check: the specialised build of a planned template, compiled (or found in the cache); no device needed
  int specialise_check(char* log, int64_t log_bytes, int64_t* code_bytes) {
    std::string why;
    const std::vector<char> code = rtc::code_object(spec_header(k_spec_, tab_host_, spec_sregs_), why, false);
    if (log && log_bytes > 0) snprintf(log, (size_t)log_bytes, "%s", why.c_str());
    if (code_bytes) *code_bytes = (int64_t)code.size();
    return code.empty() ? set_error(PCX_E_UNSUPPORTED, "generic backend: no specialised build: %s", why.substr(0, 400).c_str()) : 0;
  }
  int launch(const StepArgs& a, const pcx_buffers& out, hipStream_t s) override;
  int read_things(int64_t env0, int64_t n, pcx_sprite_state* sprites, uint8_t* curtains) override;
  int64_t bytes_per_step() const override {
    return 4 + 8 * (int64_t)k_.NW + (int64_t)(1 + k_.L) * k_.cells + 15;
  }
  int tuner_done() const override { return tuner_.done() && pw_tuner_.done(); }
  const char* kernel_name() const override { return "pcx_generic_step"; }
  int launch_shape() const override { return (spec_ ? 31 : 30) + (last_pw_ ? 2 : 0); }  // include/pcx.h pcx_engine_launch_shape
  // include/pcx.h pcx_engine_set_epilogue: the planar float32 feature array (ObservationToFeatureArray in its default axis
  // order, rendering.py:545-661) out of the render loop -- the board dword is in a register there.  The other kinds
  // (channels last, value array, repainter) stay with the hand-written kernels and the stand-alone pcx_post_* kernels.
  int set_epilogue(const pcx_epilogue_desc* d) override {
    tuner_.restart();
    if (!d) { feat_ = pcx_epilogue_desc{}; return 0; }
    if (d->to_array || d->channels_last)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: only the planar feature array is written by the table-driven kernel");
    if (!k_.occl)  // (without occlusion a layer is the thing's raw mask, not board == character: rendering.py:236-278)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: the feature-array epilogue needs occlusion_in_layers=True");
    if (fused_.on) return set_error(PCX_E_UNSUPPORTED, "generic backend: fused croppers and the feature-array epilogue exclude each other");
    PCX_HIP(hipDeviceSynchronize());  // (no launch in flight may still write the old array)
    feat_ = *d;
    return 0;
  }
  int set_fused_croppers(const crop::FusedCrops* fc) override {
    if (fc && fc->n > 0 && !k_.occl)  // (the windows derive their layers from the board they cut)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: fused croppers need occlusion_in_layers=True");
    if (fc && fc->n > 0 && feat_.out_dev)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: fused croppers and the feature-array epilogue exclude each other");
    tuner_.restart();
    return fused_.set(fc, /*drapes_ok=*/true);  // the raw curtains are bit rows in LDS: a drape's median is at hand
  }
  const int32_t* sprite_track() const override { return track_.ptr; }
  const int32_t* next_chapter_words() const override {
    return k_.w_next >= 0 ? reinterpret_cast<const int32_t*>(state_.ptr + (size_t)k_.w_next * bpad_) : nullptr;
  }
  // include/pcx.h pcx_engine_plot_words / pcx_engine_set_plot_words: the plot words are the state words W_V0..3 ([NW][bpad]
  // rows); what new episodes start with is staged in plot_in_ (allocated by init() with a new Plot's values; part of a checkpoint)
  const int32_t* plot_words() const override { return uses_plot_words_ ? reinterpret_cast<const int32_t*>(state_.ptr + (size_t)W_V0 * bpad_) : nullptr; }
  int set_plot_words(const int32_t* words_host, const uint8_t* mask_host) override {
    if (!uses_plot_words_) return set_error(PCX_E_UNSUPPORTED, "generic backend: this template's programs keep nothing in the Plot");
    std::vector<int32_t> stage((size_t)PCX_PLOT_WORDS * bpad_);
    PCX_HIP(hipDeviceSynchronize());
    PCX_HIP(hipMemcpy(stage.data(), plot_in_.ptr, stage.size() * 4, hipMemcpyDeviceToHost));
    for (int w = 0; w < PCX_PLOT_WORDS; ++w)
      for (int64_t b = 0; b < batch_; ++b)
        if (!mask_host || mask_host[b]) stage[(size_t)w * bpad_ + b] = words_host[(size_t)w * batch_ + b];
    PCX_HIP(hipMemcpy(plot_in_.ptr, stage.data(), stage.size() * 4, hipMemcpyHostToDevice));
    return 0;
  }
  const uint32_t* curtain_bits() const override { return curtains_.ptr; }
  int ensure_curtains() override { return curtains_.ptr ? 0 : curtains_.alloc((size_t)(k_.ND ? k_.ND : 1) * k_.FW * bpad_); }
  int curtain_words() const override { return k_.FW; }
  int64_t batch_pad() const override { return bpad_; }
  void persistent_arrays(std::vector<std::pair<void*, size_t>>& out) override {  // pcx_engine_export_state
    out.push_back({state_.ptr, state_.count * sizeof(uint32_t)});
    out.push_back({track_.ptr, track_.count * sizeof(int32_t)});
    if (plot_in_.ptr) out.push_back({plot_in_.ptr, plot_in_.count * sizeof(int32_t)});  // (what auto-resets after a resume start from)
  }
  int plane_pitch() const override { return k_.pitch; }

 private:
  Consts k_{};
  bool uses_plot_words_ = false;             // the template's programs keep Plot entries in the state words W_V0..3 (examples/ordeal.py)
  int32_t plot_init_[PCX_PLOT_WORDS] = {0, 0, 0, 0};
  DevArray<int32_t> plot_in_;                // [PCX_PLOT_WORDS][bpad], see set_plot_words()
  bool spec_sregs_ = false;  // ... and whether that build keeps the sprites' state in registers (spec_header says so to the kernel)
  Consts k_spec_{};  // the same with the LDS layout of the specialised build (plan(): no flag / snapshot columns); what a launch of spec_ goes by
  int64_t batch_ = 0, bpad_ = 0;
  uint64_t seed_ = 0;
  int64_t env_offset_ = 0;
  int num_cus_ = 256;
  stream::FusedCropsHolder fused_;
  DevArray<uint32_t> tables_, state_, curtains_;
  DevArray<unsigned long long> stats_;  // PCX_DEBUG & 8
  DevArray<int32_t> track_;
  int n_table_words_ = 0;
  std::vector<uint32_t> tab_host_;  // the staged tables as uploaded (the constants of a specialised build)
  pcx_epilogue_desc feat_{};           // pcx_engine_set_epilogue (out_dev null: none)
  const rtc::Loaded* spec_ = nullptr;  // the build of pcx_generic_step specialised for this template, when there is one
  Tuner tuner_;
  int64_t state_unit_ = WAVE, state_row_ = 0;  // the state words' layout (pcx_generic_kernel.h Ptrs): set in init()
  // persistent workers (pcx_generic_kernel.h pcx_generic_step_pw)
  DevArray<uint32_t> work_ctr_;
  ShapeTuner pw_tuner_;
  bool last_pw_ = false, pw_lds_raised_ = false;
  int launch_pw(const StepArgs& a, const pcx_buffers& out, hipStream_t s, Ptrs& P, bool* launched);
  std::vector<int> walker_;
};

// Everything about a template that needs no device: validation, the tables, the state and LDS layouts.
int GenericBackend::plan(const pcx_template& t, int64_t batch) {
  Consts& k = k_;
  batch_ = batch;
  bpad_ = (batch + WAVE - 1) / WAVE * WAVE;
  k.occl = t.occlusion_in_layers != 0;
  k.game = t.game; k.R = t.rows; k.C = t.cols; k.cells = t.rows * t.cols; k.L = t.n_chars;
  k.NS = t.n_sprites; k.ND = t.n_drapes; k.NT = t.n_things; k.n_groups = t.n_groups; k.n_actions = t.n_actions;
  if (k.C > 255 || k.R > 255 || k.L > MAX_L || k.cells > 8192)
    return set_error(PCX_E_UNSUPPORTED, "generic backend: board larger than 255x255 / 8192 cells or more than %d characters", MAX_L);
  if (k.NT > 16)  // the render loop is instantiated for up to 16 things (render_planes<16>)
    return set_error(PCX_E_UNSUPPORTED, "generic backend: %d sprites and drapes, at most 16 are supported", k.NT);
  k.pitch = (k.cells + 3) & ~3;
  k.QW = k.pitch / 4;
  k.RW = (k.C + 31) / 32;
  k.FW = (k.cells + 31) / 32 + 2;
  {
    bool ok = true;
    const uint32_t m = (uint32_t)(((1ull << 32) + k.QW - 1) / k.QW);
    for (uint32_t x = 0; x <= (uint32_t)WAVE * k.QW; ++x)
      if ((uint32_t)(((uint64_t)x * m) >> 32) != x / k.QW) { ok = false; break; }
    if (!ok) return set_error(PCX_E_UNSUPPORTED, "generic backend: board too large for the 32-bit reciprocal");
    k.magic_q = m;
    const uint32_t mc = (uint32_t)(((1ull << 32) + k.C - 1) / k.C);
    for (uint32_t x = 0; x < (uint32_t)k.cells; ++x)
      if ((uint32_t)(((uint64_t)x * mc) >> 32) != x / k.C) { ok = false; break; }
    if (!ok) return set_error(PCX_E_UNSUPPORTED, "generic backend: board too large for the 32-bit reciprocal");
    k.magic_c = mc;
  }
  seed_ = (uint64_t)(uint32_t)t.param[0] | ((uint64_t)(uint32_t)t.param[1] << 32);
  env_offset_ = (int64_t)((uint64_t)(uint32_t)t.param[2] | ((uint64_t)(uint32_t)t.param[3] << 32));

  // things, numbered by z-order position (back to front)
  auto find_sprite = [&](int ch) { for (int s = 0; s < t.n_sprites; ++s) if (t.sprites[s].ch == ch) return s; return -1; };
  auto find_drape = [&](int ch) { for (int d = 0; d < t.n_drapes; ++d) if (t.drapes[d].ch == ch) return d; return -1; };
  auto layer_of = [&](int ch) { for (int i = 0; i < k.L; ++i) if (t.chars[i] == ch) return i; return -1; };
  std::vector<uint32_t> things((size_t)k.NT * T_WORDS, 0), zt(k.NT), sched(k.NT), patterns;
  k.has_scroll = 0;
  k.n_sgroups = 1;
  for (int g = 0; g < PCX_MAX_SCROLL_GROUPS; ++g) k.group_sprites[g] = 0;
  k.ip = k.ix = k.ib = k.tx = -1;
  k.bolt_mask_all = k.bolt_mask_up = k.box_mask = 0;
  for (int z = 0; z < k.NT; ++z) {
    const int ch = t.z_order[z];
    uint32_t* e = &things[(size_t)z * T_WORDS];
    e[T_CH] = ch;
    e[T_LAYER] = layer_of(ch);
    uint32_t above = 0;
    for (int u = z + 1; u < k.NT; ++u) above |= 1u << u;
    e[T_ABOVE] = above;
    int s = find_sprite(ch), d = find_drape(ch);
    if (s >= 0) {
      const pcx_sprite_desc& sd = t.sprites[s];
      e[T_KIND] = 0; e[T_IDX] = s; e[T_PROG] = sd.program;
      e[T_FLAGS] = (sd.is_walker ? TF_WALKER : 0) | (sd.confined ? TF_CONFINED : 0);
      e[T_P0] = sd.param[0]; e[T_P1] = sd.param[1]; e[T_P2] = sd.param[2]; e[T_P3] = sd.param[3];
      memcpy(&e[T_IMP0], sd.impassable, 16);
      if (sd.egocentric) { e[T_FLAGS] |= TF_EGO; k.has_scroll = 1; }
      if (sd.scrolling_group >= PCX_MAX_SCROLL_GROUPS) return set_error(PCX_E_UNSUPPORTED, "generic backend: more than %d scrolling groups", PCX_MAX_SCROLL_GROUPS);
      e[T_GROUP] = sd.scrolling_group;
      k.group_sprites[sd.scrolling_group] |= 1u << s;
      if ((int)sd.scrolling_group + 1 > k.n_sgroups) k.n_sgroups = sd.scrolling_group + 1;
      if (ch == 'P') k.ip = z;
      if (sd.program == PCX_PROG_EM_UPBOLT) { k.bolt_mask_all |= 1 << s; k.bolt_mask_up |= 1 << s; }
      if (sd.program == PCX_PROG_EM_DOWNBOLT) k.bolt_mask_all |= 1 << s;
      if (sd.program == PCX_PROG_WM_BOX) k.box_mask |= 1 << s;
    } else if (d >= 0) {
      const pcx_drape_desc& dd = t.drapes[d];
      e[T_KIND] = 1; e[T_IDX] = d; e[T_PROG] = dd.program; e[T_P0] = dd.param[0]; e[T_P1] = dd.param[1];
      e[T_P2] = dd.param[2]; e[T_P3] = dd.param[3];
      if (dd.scrolling_group >= PCX_MAX_SCROLL_GROUPS) return set_error(PCX_E_UNSUPPORTED, "generic backend: more than %d scrolling groups", PCX_MAX_SCROLL_GROUPS);
      e[T_GROUP] = dd.scrolling_group;
      if ((int)dd.scrolling_group + 1 > k.n_sgroups) k.n_sgroups = dd.scrolling_group + 1;
      if (dd.is_scrolly) {
        if (dd.pattern_rows > 4096 || dd.pattern_cols > 4096 || dd.margin_rows > 255 || dd.margin_cols > 255)
          return set_error(PCX_E_UNSUPPORTED, "generic backend: Scrolly pattern too large");
        const int PRW = (dd.pattern_cols + 31) / 32 + 2;
        e[T_FLAGS] = TF_SCROLLY;
        e[T_PDIM] = (uint32_t)dd.pattern_rows | ((uint32_t)dd.pattern_cols << 16);
        e[T_MARG] = (uint32_t)(dd.have_margins != 0) | ((uint32_t)dd.margin_rows << 8) | ((uint32_t)dd.margin_cols << 16);
        e[T_PRW] = PRW;
        e[T_PAT] = 0x80000000u | (uint32_t)patterns.size();  // relocated once the table layout is known
        for (int r = 0; r < dd.pattern_rows; ++r) {
          std::vector<uint32_t> row(PRW, 0);
          for (int c = 0; c < dd.pattern_cols; ++c)
            if (dd.pattern[(size_t)r * dd.pattern_cols + c]) row[c >> 5] |= 1u << (c & 31);
          patterns.insert(patterns.end(), row.begin(), row.end());
        }
        k.has_scroll = 1;
      } else if (dd.program == PCX_PROG_SCROLLY) {
        return set_error(PCX_E_INVALID, "generic backend: the 'scrolly' program needs a Scrolly drape");
      }
      if (ch == 'X') { k.ix = d; k.tx = z; }
      if (ch == 'B') k.ib = d;
    } else {
      return set_error(PCX_E_INVALID, "generic backend: z_order names an unknown character");
    }
    zt[z] = z;
    if (k.C > 64)  // whole-row rotates and window copies hold a row in 64 bits
      switch (e[T_PROG]) {
        case PCX_PROG_WM_JUDGE: case PCX_PROG_HW_ROLLING: case PCX_PROG_EM_MARAUDER: case PCX_PROG_SCROLLY:
          return set_error(PCX_E_UNSUPPORTED, "generic backend: program %u needs cols <= 64", e[T_PROG]);
        default: break;
      }
    if (k.C > 64 && d >= 0 && t.drapes[d].is_scrolly)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: Scrolly drapes need cols <= 64");
    switch (e[T_PROG]) {
      case PCX_PROG_WM_BOX: case PCX_PROG_WM_JUDGE: case PCX_PROG_WM_PLAYER: case PCX_PROG_HW_ROLLING:
      case PCX_PROG_HW_SLIDING: case PCX_PROG_EM_PLAYER: case PCX_PROG_EM_BUNKER: case PCX_PROG_EM_MARAUDER:
      case PCX_PROG_EM_UPBOLT: case PCX_PROG_EM_DOWNBOLT: case PCX_PROG_STATIC: case PCX_PROG_WALKER:
      case PCX_PROG_SCROLLY: case PCX_PROG_BS_PLAYER: case PCX_PROG_BS_PATROLLER: case PCX_PROG_BS_CASH:
      case PCX_PROG_OD_PLAYER: case PCX_PROG_OD_DRAGONDUCK: case PCX_PROG_OD_SWORD: break;
      default: return set_error(PCX_E_UNSUPPORTED, "generic backend: no device program %u", e[T_PROG]);
    }
  }
  for (int i = 0; i < k.NT; ++i) {
    int zi = -1;
    for (int z = 0; z < k.NT; ++z) if (t.z_order[z] == t.schedule[i]) zi = z;
    if (zi < 0) return set_error(PCX_E_INVALID, "generic backend: schedule names an unknown character");
    sched[i] = (uint32_t)zi | ((uint32_t)t.group_of[i] << 8);
  }
  for (int z = 0; z < k.NT; ++z) {  // programs that look up things['P']
    const uint32_t prog = things[(size_t)z * T_WORDS + T_PROG];
    if ((prog == PCX_PROG_BS_PATROLLER || prog == PCX_PROG_BS_CASH || prog == PCX_PROG_EM_UPBOLT ||
         prog == PCX_PROG_EM_DOWNBOLT || prog == PCX_PROG_WM_BOX || prog == PCX_PROG_OD_DRAGONDUCK || prog == PCX_PROG_OD_SWORD) && k.ip < 0)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: program %u needs a sprite 'P'", prog);
    if ((prog == PCX_PROG_EM_DOWNBOLT) && k.tx < 0)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: program %u needs a drape 'X'", prog);
  }
  if (t.game == PCX_GAME_MARAUDERS && (k.ip < 0 || k.ix < 0))
    return set_error(PCX_E_UNSUPPORTED, "generic backend: marauders needs things 'P' and 'X'");
  if (t.game == PCX_GAME_WAREHOUSE && k.ip < 0)
    return set_error(PCX_E_UNSUPPORTED, "generic backend: warehouse needs a 'P' sprite");

  // backdrop, backdrop-only characters, goal cells ('_') as bit-rows
  std::vector<uint32_t> bd4(k.QW, 0);
  memcpy(bd4.data(), t.backdrop, k.cells);
  k.n_bchars = 0;
  std::vector<uint32_t> bdmask, laybc, s2t(k.NS ? k.NS : 1, 0), d2t(k.ND ? k.ND : 1, 0);
  for (int z = 0; z < k.NT; ++z)
    (things[(size_t)z * T_WORDS + T_KIND] == 0 ? s2t : d2t)[things[(size_t)z * T_WORDS + T_IDX]] = z;
  for (int z = 0; z < k.NT; ++z) {  // walkers: which things' characters are impassable to them (sprites.py:496-511)
    if (things[(size_t)z * T_WORDS + T_KIND] != 0) continue;
    const pcx_sprite_desc& sd = t.sprites[things[(size_t)z * T_WORDS + T_IDX]];
    uint32_t impt = 0;
    for (int u = 0; u < k.NT; ++u) {
      const int ch = t.z_order[u];
      if (ch < 128 && ((sd.impassable[ch >> 3] >> (ch & 7)) & 1)) impt |= 1u << u;
    }
    things[(size_t)z * T_WORDS + T_IMPT] = impt;
  }
  for (int z = 0; z < k.NT; ++z)
    for (int u = z + 1; u < k.NT; ++u) {
      const uint32_t* f = &things[(size_t)u * T_WORDS];
      things[(size_t)z * T_WORDS + (f[T_KIND] == 0 ? T_ABOVE_S : T_ABOVE_D)] |= 1u << f[T_IDX];
    }
  for (int i = 0; i < k.L; ++i) {
    const int ch = t.chars[i];
    if (find_sprite(ch) >= 0 || find_drape(ch) >= 0) continue;
    laybc.push_back(i); k.n_bchars++;
    std::vector<uint32_t> m(k.QW, 0);
    uint8_t* mb = reinterpret_cast<uint8_t*>(m.data());
    for (int c = 0; c < k.cells; ++c) mb[c] = t.backdrop[c] == ch;
    bdmask.insert(bdmask.end(), m.begin(), m.end());
  }
  std::vector<uint32_t> aux((size_t)k.R * k.RW, 0);
  for (int r = 0; r < k.R; ++r)
    for (int c = 0; c < k.C; ++c)
      if (t.backdrop[r * k.C + c] == '_') aux[r * k.RW + (c >> 5)] |= 1u << (c & 31);

  // state layout + initial words
  k.w_sflags = W_SPRITES + k.NS;
  k.w_drapes = k.w_sflags + (k.NS + 3) / 4;
  const int ndw = k.ND * k.R * k.RW;
  k.w_scroll = k.w_drapes + ndw;
  // plot directives: the issuing / moved things as thing ids; a game that changes
  // the z-order keeps it per environment (two state words)
  std::vector<uint32_t> dirs;
  k.n_dir = t.n_directives; k.zdyn = 0;
  bool next_dir = false;
  k.reward_float = t.reward_is_float != 0;
  for (int z = 0; z < k.NT; ++z) {  // examples/ordeal.py: its programs assign next_chapter, change the z-order and keep Plot entries
    const uint32_t prog = things[(size_t)z * T_WORDS + T_PROG];
    if (prog == PCX_PROG_OD_PLAYER || prog == PCX_PROG_OD_DRAGONDUCK) next_dir = true;
    if (prog == PCX_PROG_OD_DRAGONDUCK) k.zdyn = 1;
    if (prog == PCX_PROG_OD_PLAYER || prog == PCX_PROG_OD_DRAGONDUCK || prog == PCX_PROG_OD_SWORD) uses_plot_words_ = true;
  }
  if (k.n_dir < 0 || k.n_dir > PCX_MAX_DIRECTIVES) return set_error(PCX_E_INVALID, "generic backend: bad directive count");
  auto thing_of = [&](int ch) { for (int z = 0; z < k.NT; ++z) if (t.z_order[z] == ch) return z; return -1; };
  for (int i = 0; i < k.n_dir; ++i) {
    const pcx_directive& dv = t.directives[i];
    const int who = thing_of(dv.ch);
    int move = 0, front = 0xFF;
    if (who < 0 || dv.selector <= 0) return set_error(PCX_E_INVALID, "generic backend: malformed directive %d", i);
    const uint32_t wprog = things[(size_t)who * T_WORDS + T_PROG];
    if (wprog != PCX_PROG_WALKER && wprog != PCX_PROG_SCROLLY && wprog != PCX_PROG_STATIC)
      return set_error(PCX_E_UNSUPPORTED, "generic backend: only tabled entities issue plot directives");
    if (dv.kind == PCX_DIR_Z_ORDER) {
      move = thing_of(dv.move_this);
      front = dv.in_front_of ? thing_of(dv.in_front_of) : 0xFF;
      if (move < 0 || front < 0 || move == front)
        return set_error(PCX_E_INVALID, "generic backend: a z-order directive names no Sprite or Drape of this game");
      k.zdyn = 1;
    } else if (dv.kind == PCX_DIR_TERMINATE) {
      if (!(dv.discount >= 0.0f && dv.discount <= 1.0f)) return set_error(PCX_E_INVALID, "Discount must be in range [0,1].");
    } else if (dv.kind == PCX_DIR_NEXT_CHAPTER) {
      if (dv.reward < PCX_CHAPTER_NONE) return set_error(PCX_E_INVALID, "generic backend: a next_chapter directive names chapter %d", dv.reward);
      next_dir = true;
    } else if (dv.kind != PCX_DIR_ADD_REWARD) {
      return set_error(PCX_E_INVALID, "generic backend: unknown directive kind %d", dv.kind);
    }
    uint32_t dbits;
    memcpy(&dbits, &dv.discount, 4);
    dirs.push_back((uint32_t)who | ((uint32_t)dv.kind << 8) | ((uint32_t)move << 16) | ((uint32_t)front << 24));
    dirs.push_back((uint32_t)dv.selector);
    dirs.push_back((uint32_t)dv.reward);
    dirs.push_back(dbits);
  }
  k.w_z = k.w_scroll + (k.has_scroll ? 1 + k.ND + 2 * k.NS : 0);
  k.w_next = next_dir ? k.w_z + (k.zdyn ? 2 : 0) : -1;
  k.NW = k.w_z + (k.zdyn ? 2 : 0) + (next_dir ? 1 : 0);
  std::vector<uint32_t> init(k.NW, 0), initd(ndw ? ndw : 1, 0);
  if (next_dir) init[k.w_next] = (uint32_t)PCX_CHAPTER_UNSET;
  init[W_FRAME] = (uint32_t)-1;
  uint32_t dx_plus1 = 1;
  int32_t v[4] = {0, 0, (int32_t)NEVER, (int32_t)NEVER};
  if (uses_plot_words_) { v[PCX_PLOT_OD_HAS_SWORD] = 0; v[PCX_PLOT_OD_LAST_POSITION] = -1; v[PCX_PLOT_OD_PRIOR_CHAPTER] = -1; v[3] = 0; }  // a new Plot
  memcpy(plot_init_, v, sizeof v);
  for (int d = 0; d < k.ND; ++d) {
    if (t.drapes[d].program == PCX_PROG_EM_MARAUDER) dx_plus1 = (uint32_t)(t.drapes[d].param[0] + 1) & 0xFF;
    if (t.drapes[d].program == PCX_PROG_WM_JUDGE) v[0] = t.drapes[d].param[0];
    for (int r = 0; r < k.R; ++r)
      for (int c = 0; c < k.C; ++c)
        if (t.drapes[d].curtain[r * k.C + c]) initd[(d * k.R + r) * k.RW + (c >> 5)] |= 1u << (c & 31);
  }
  init[W_FLAGS] = dx_plus1 << 8;
  if (k.has_scroll)
    for (int d = 0; d < k.ND; ++d)
      init[k.w_scroll + 1 + d] = ((uint32_t)t.drapes[d].corner_row & 0xFFFFu) | ((uint32_t)t.drapes[d].corner_col << 16);
  for (int j = 0; j < 4; ++j) init[W_V0 + j] = (uint32_t)v[j];
  walker_.assign(k.NS, 0);
  for (int s = 0; s < k.NS; ++s) {
    const pcx_sprite_desc& sd = t.sprites[s];
    walker_[s] = sd.is_walker;
    const int vr = sd.is_walker ? sd.vrow : sd.row, vc = sd.is_walker ? sd.vcol : sd.col;
    init[W_SPRITES + s] = ((uint32_t)vr & 0xFFFFu) | ((uint32_t)vc << 16);
    init[k.w_sflags + (s >> 2)] |= ((uint32_t)(sd.visible != 0) | ((uint32_t)(sd.prior_visible != 0) << 1) |
                                    ((uint32_t)(sd.program == PCX_PROG_BS_PATROLLER && sd.param[0]) << 2)) << (8 * (s & 3));
  }

  // tables -> one buffer staged into LDS, then the per-lane arrays
  std::vector<uint32_t> tab;
  auto place = [&](const std::vector<uint32_t>& v2) { int off = (int)tab.size(); tab.insert(tab.end(), v2.begin(), v2.end()); return off; };
  k.l_things = place(things); k.l_z = place(zt); k.l_sched = place(sched); k.l_backdrop = place(bd4);
  k.l_bdmask = place(bdmask); k.l_aux = place(aux); k.l_init = place(init); k.l_initd = place(initd);
  if (laybc.empty()) laybc.push_back(0);
  k.l_laybc = place(laybc); k.l_s2t = place(s2t); k.l_d2t = place(d2t);
  k.l_dir = place(dirs);
  {
    // owner codes (pcx_stream.h stream_codes; pcx_generic_step_pw): the backdrop's code dwords -- a character's code names its
    // layer plane; plane padding is selector 12 (zero bytes in every plane).  At most 16 characters.
    std::vector<uint32_t> bdcode(k.QW, 0);
    uint8_t* const b = reinterpret_cast<uint8_t*>(bdcode.data());
    const int Lc = k.L;
    for (int c = 0; c < k.pitch; ++c) {
      uint32_t code = Lc <= 8 ? 12u : 0xCCu;
      if (c < k.cells) {
        const uint32_t i = (uint32_t)layer_of(t.backdrop[c]);
        code = Lc <= 8 ? i : i < 8u ? 0xC0u | i : 0x0Cu | ((i - 8u) << 4);
      }
      b[c] = (uint8_t)code;
    }
    k.l_bdcode = place(bdcode);
  }
  {
    const int pat0 = place(patterns);
    for (int z = 0; z < k.NT; ++z) {
      uint32_t& off = tab[k.l_things + (size_t)z * T_WORDS + T_PAT];
      if (tab[k.l_things + (size_t)z * T_WORDS + T_KIND] == 1 && (off & 0x80000000u)) off = pat0 + (off & 0x7FFFFFFFu);
    }
  }
  n_table_words_ = (int)tab.size();
  tab_host_ = tab;
  // The per-lane arrays behind the staged tables.  `sregs`: the layout of the specialised build (round 6: pcx_generic_kernel.h
  // PCX_SREGS keeps every sprite's flag byte and snapshot cell in registers -- their columns are not laid out at all, and
  // l_flg / l_snap alias l_pos, which still receives the position rows of the state load).
  auto layout = [&](Consts& k, bool sregs) {
  int off = (n_table_words_ + 1) & ~1;
  k.l_pos = off; off += k.NS * WAVE;
  k.l_flg = sregs ? k.l_pos : off; if (!sregs) off += k.NS * WAVE;
  k.l_snap = sregs ? k.l_pos : off; if (!sregs) off += k.NS * WAVE;
  k.l_cur = off; off += ndw * WAVE;
  k.l_snapd = off; off += ndw * WAVE;
  k.l_corner = off; if (k.has_scroll) off += k.ND * WAVE;
  k.l_pmask = off; if (k.has_scroll) off += k.NS * WAVE;
  k.l_pframe = off; if (k.has_scroll) off += k.NS * WAVE;
  k.l_zord = off; if (k.zdyn) off += k.NT * WAVE;
  k.l_zabove = off; if (k.zdyn) off += k.NT * WAVE;
  k.l_zabove_s = off; if (k.zdyn) off += k.NT * WAVE;
  k.l_zabove_d = off; if (k.zdyn) off += k.NT * WAVE;
  k.l_ztmp = off; if (k.zdyn) off += (k.NT + 1) * WAVE;
  k.l_zq = off; if (k.zdyn) off += MAX_ZQ * WAVE;
  // owner codes of the group, [64][QW | 1] dwords (pcx_generic_step's render loop since round 6): over everything above, which is
  // dead by the time the logic phase writes them -- the state has been written back, the curtains flattened, the track words stored
  k.l_codes = (k.occl && k.L <= 16 && k.l_bdcode >= 0 && k.QW <= 160) ? k.l_pos : -1;  // (larger boards: 40 KB of codes per group and more -- the mask loop)
  if (k.l_codes >= 0 && off < k.l_codes + WAVE * (k.QW | 1)) off = k.l_codes + WAVE * (k.QW | 1);
  off = (off + 1) & ~1;
  k.l_flat = off; off += k.ND * (k.FW | 1) * WAVE;  // ---- from here on: what the render phase reads
  off = (off + 1) & ~1;
  k.l_sdesc = off; off += 2 * k.NS * WAVE;
  // the inbox of the state load lies over them (the flat vectors and the descriptors are written after the state
  // has been consumed); a template with few things gets the rows it lacks
  k.l_inbox = k.l_flat;
  if (off < k.l_inbox + (IB_ROWS + (k.NS + 3) / 4) * WAVE) off = k.l_inbox + (IB_ROWS + (k.NS + 3) / 4) * WAVE;
  k.l_skip = off; off += WAVE;
  k.l_flatraw = off; if (!k.occl) off += k.ND * (k.FW | 1) * WAVE;
  off = (off + 1) & ~1;
  k.l_sdescraw = off; if (!k.occl) off += 2 * k.NS * WAVE;
  k.l_wcorner = off; off += crop::MAX_FUSED_CROPPERS * WAVE;
  k.l_words = off;
  };
  layout(k, false);
  k_spec_ = k;
  {
    const char* defs = getenv("PCX_GENERIC_SPEC_DEFS");  // (A/B runs: the round-5 build of the kernel needs the round-5 layout)
    // the sprites' state in registers (pcx_generic_kernel.h PCX_SREGS): up to eight sprites, and not the marauders' programs -- they
    // index sprites by a lane's own values, select chains of NS (marauders_custom_A 262,144: 0.318 -> 0.353 ms; profiles/r06_generic.md)
    bool em = false;
    for (int z = 0; z < k.NT; ++z) {
      const uint32_t pr = tab[k.l_things + (size_t)z * T_WORDS + T_PROG];
      em = em || pr == PCX_PROG_EM_PLAYER || pr == PCX_PROG_EM_BUNKER || pr == PCX_PROG_EM_MARAUDER || pr == PCX_PROG_EM_UPBOLT || pr == PCX_PROG_EM_DOWNBOLT;
    }
    spec_sregs_ = !(defs && strstr(defs, "PCX_X_NO_SPRITE_REGS")) && k.NS <= 8 && k.NS > 0 && !em;
    if (spec_sregs_) layout(k_spec_, true);
  }
  const int off = k.l_words;
  for (int i = 0; i < PCX_MAX_CHARS; ++i) k.chars[i] = i < t.n_chars ? t.chars[i] : 0;
  if ((size_t)off * 4 > 160 * 1024)
    return set_error(PCX_E_UNSUPPORTED, "generic backend: template needs %d bytes of LDS per wave", off * 4);
  for (int i = 0; i < PCX_MAX_CHARS; ++i) k_spec_.chars[i] = k.chars[i];
  if (const char* dump = getenv("PCX_GENERIC_DUMP_SPEC")) {  // experiments: the header of a specialised build (see spec_header)
    if (FILE* f = fopen(dump, "w")) { const std::string h = spec_header(k_spec_, tab_host_, spec_sregs_); fwrite(h.data(), 1, h.size(), f); fclose(f); }
  }
  return 0;
}

int GenericBackend::init(const pcx_template& t, int64_t batch) {
  if (int rc0 = plan(t, batch)) return rc0;
  const Consts& k = k_;
  const int off = k.l_words;
  const std::vector<uint32_t>& tab = tab_host_;
  {
    int dev = 0;
    hipDeviceProp_t prop;
    if (hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&prop, dev) == hipSuccess && prop.multiProcessorCount > 0)
      num_cus_ = prop.multiProcessorCount;
  }
  {
    // A specialised build costs seconds of compile time once per template (then a file read): worth it for the
    // batches this engine is for, not for a unit test's few hundred environments.  PCX_GENERIC_JIT=0 / 1: never /
    // always; PCX_GENERIC_JIT_MIN: the smallest batch that gets one (default 4,096: hiprtc takes 1-3 s per template).
    int64_t min_batch = 4096;
    if (const char* e = getenv("PCX_GENERIC_JIT_MIN")) min_batch = atoll(e);
    const char* jit = getenv("PCX_GENERIC_JIT");
    const bool want = jit ? atoi(jit) != 0 : batch >= min_batch;
    const char* dbg = getenv("PCX_DEBUG");
    const bool verbose = dbg && (atoi(dbg) & 16);
    if (want) {
      int dev = 0;
      (void)hipGetDevice(&dev);
      std::string why;
      spec_ = rtc::load(spec_header(k_spec_, tab_host_, spec_sregs_), dev, why, verbose);
      if (spec_ && (size_t)off * 4 > 64 * 1024) {  // more dynamic LDS than the default limit: the module function must be told
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(spec_->fn), hipFuncAttributeMaxDynamicSharedMemorySize, off * 4);
        if (e != hipSuccess) {
          (void)hipGetLastError();
          why = std::string("hipFuncSetAttribute(MaxDynamicSharedMemorySize) on the module function: ") + hipGetErrorString(e);
          spec_ = nullptr;
        }
      }
      if (!spec_ && verbose) fprintf(stderr, "[pcx generic] no specialised kernel: %s\n", why.c_str());
    }
  }
  int rc;
  if ((rc = tables_.upload(tab))) return rc;
  // [NW][bpad].  (Round 6 measured the unit-major alternative -- a unit's NW rows as one contiguous piece, state_unit_ = NW * 64,
  // state_row_ = 64: one 6-10 KB burst and one TLB entry per unit instead of 26-40 scattered rows -- with the kernel side as it is
  // now: 0.1053 / 0.1055 ms on warehouse_L0, 0.0820 / 0.0825 on walkers_scroll_groups, the logic-only launches equal too.  The
  // write-back is not what the logic phase waits for; the host-side readers were not converted.)
  state_unit_ = WAVE; state_row_ = bpad_;
  {
    const char* defs = getenv("PCX_GENERIC_SPEC_DEFS");  // (PCX_X_WB4, a timing experiment of the kernel: room for its 16-byte stores)
    const bool wb4 = defs && strstr(defs, "PCX_X_WB4");
    if ((rc = state_.alloc((size_t)k.NW * bpad_ * (wb4 ? 2 : 1) + (wb4 ? (size_t)bpad_ * 8 : 0)))) return rc;
  }
  if ((rc = track_.alloc((size_t)(k.NS ? k.NS : 1) * bpad_))) return rc;
  if (uses_plot_words_) {  // every episode starts from a new Plot's entries until pcx_engine_set_plot_words says otherwise
    std::vector<int32_t> stage((size_t)PCX_PLOT_WORDS * bpad_);
    for (int w = 0; w < PCX_PLOT_WORDS; ++w) std::fill(stage.begin() + (size_t)w * bpad_, stage.begin() + (size_t)(w + 1) * bpad_, plot_init_[w]);
    if ((rc = plot_in_.upload(stage))) return rc;
  }
  if ((rc = work_ctr_.alloc(16 * 9))) return rc;  // the logic workers' ticket shards and done-count (pcx_stream.h WorkQueue), zeroed here
  return 0;
}

// Persistent workers with decoupled logic / render (pcx_generic_kernel.h pcx_generic_step_pw): plain step launches of batches
// that give every CU several work units.  *launched false: the caller takes pcx_generic_step.
int GenericBackend::launch_pw(const StepArgs& a, const pcx_buffers& out, hipStream_t s, Ptrs& P, bool* launched) {
  *launched = false;
  const int64_t groups = bpad_ / WAVE;
  int min_per_cu = 4;
  if (const char* e = getenv("PCX_GENERIC_PW_MIN")) min_per_cu = atoi(e);
  bool want = a.mode == 0 && a.n_steps == 1 && !fused_.on && !feat_.out_dev && !a.export_curtains && (a.debug & ~(2 | 8 | 16 | 32)) == 0 &&
              groups >= (int64_t)num_cus_ * min_per_cu && (!spec_ || spec_->fn_pw) && k_.occl && k_.L <= 16;
  // Opt-in (PCX_GENERIC_PW=1).  Measured (profiles/r06_generic.md): decoupling does what it should -- the render workers' owner-code
  // loop streams a unit in 3-4 us, two of them keep up with six logic workers -- but the launch stays bound by the LOGIC side,
  // units_per_CU x T / n_logic: a logic worker's copy of the per-lane arrays is as big as a group's in pcx_generic_step, its
  // hand-over slot comes on top, so fewer contexts step at once (6 against 9-16), and T grows by the code generation and by the
  // worker's own write-back queueing behind the plane stores (30 -> 41 us on warehouse_L0).  warehouse_L0 262,144: 0.104-0.106 ms
  // either way; walkers_scroll_groups 0.104 against 0.079; marauders_custom_A 0.352 against 0.318.  Kept as a tested launch shape
  // for what comes next (smaller per-lane arrays), not as the default.
  if (const char* e = getenv("PCX_GENERIC_PW")) want = want && atoi(e) != 0; else want = false;
  if (!want) return 0;
  const Consts& k = spec_ ? k_spec_ : k_;
  const int lw = (k.l_wcorner - k.l_pos + 1) & ~1, slot = (WAVE * (k.QW | 1) + WAVE + 1) & ~1;  // a worker's per-lane arrays; its hand-over slot
  // candidates: {logic workers, render workers, workgroups per CU}
  struct Cand { int nl, nr, per_cu; };
  static const Cand cands[ShapeTuner::NC] = {{6, 2, 1}, {4, 2, 1}, {3, 1, 2}, {8, 2, 1}};
  const bool knobs = getenv("PCX_GENERIC_PW_LOGIC") || getenv("PCX_GENERIC_PW_RENDER") || getenv("PCX_GENERIC_PW_PER_CU") ||
                     (getenv("PCX_GENERIC_TUNE") && atoi(getenv("PCX_GENERIC_TUNE")) == 0);
  if (knobs || (a.debug & ~16)) pw_tuner_.off = true;
  const Cand& c = cands[pw_tuner_.pick(a, s)];
  int nl = c.nl, nr = c.nr, per_cu = c.per_cu;
  if (const char* e = getenv("PCX_GENERIC_PW_LOGIC")) { const int v = atoi(e); if (v >= 1 && v <= 14) nl = v; }
  if (const char* e = getenv("PCX_GENERIC_PW_RENDER")) { const int v = atoi(e); if (v >= 1 && v <= 8) nr = v; }
  if (const char* e = getenv("PCX_GENERIC_PW_PER_CU")) { const int v = atoi(e); if (v >= 1 && v <= 4) per_cu = v; }
  // what fits: per workgroup the tables, nl copies of the per-lane arrays and as many hand-over slots, the flags; per CU 160 KB
  auto words_for = [&](int n) { return (size_t)k.l_pos + (size_t)n * (lw + slot) + (size_t)n + 2; };
  const size_t room = ((size_t)160 * 1024 / (size_t)per_cu) & ~(size_t)255;
  while (nl > 1 && words_for(nl) * 4 > room) --nl;
  if (words_for(nl) * 4 > room) return 0;
  if (nr > nl) nr = nl;
  if (nl + nr > 16) nr = 16 - nl;
  const size_t lds = words_for(nl) * 4;
  int64_t wgs = (int64_t)num_cus_ * per_cu;
  if (const char* e = getenv("PCX_GENERIC_PW_GRID")) { const int v = atoi(e); if (v >= 1) wgs = v; }  // (tests: few workgroups, many units each)
  const int64_t want_wgs = (groups + nl - 1) / nl;
  if (wgs > want_wgs) wgs = want_wgs;
  stream::WorkArgs wa;
  wa.ctr = work_ctr_.ptr;
  wa.n_units = (uint32_t)groups;
  wa.dynamic = wgs * nl < groups && groups >= (int64_t)num_cus_ * 8;
  if (const char* e = getenv("PCX_GENERIC_PW_DYNAMIC")) wa.dynamic = atoi(e) != 0 && wgs * nl < groups;
  if (getenv("PCX_GENERIC_PW_GRID") || getenv("PCX_GENERIC_PW_DYNAMIC")) pw_tuner_.off = true;
  wa.lock = 0;
  PwArgs w{wa, nl, nr, lw, k.l_pos + nl * lw, slot, k.l_pos + nl * (lw + slot)};
  if (lds > 64 * 1024 && !pw_lds_raised_) {
    if (spec_) {
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(spec_->fn_pw), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
      if (e != hipSuccess) { (void)hipGetLastError(); return 0; }
    } else {
      PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(pcx_generic_step_pw), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    }
    pw_lds_raised_ = true;
  }
  if (spec_) {
    void* params[] = {const_cast<Consts*>(&k), &P, const_cast<StepArgs*>(&a), const_cast<pcx_buffers*>(&out), &w};
    PCX_HIP(hipModuleLaunchKernel(spec_->fn_pw, (unsigned)wgs, 1, 1, (unsigned)((nl + nr) * WAVE), 1, 1, (unsigned)lds, s, params, nullptr));
  } else {
    hipLaunchKernelGGL(pcx_generic_step_pw, dim3((unsigned)wgs), dim3((nl + nr) * WAVE), lds, s, k_, P, a, out, w);
  }
  PCX_HIP(hipGetLastError());
  pw_tuner_.launched(s);
  *launched = true;
  return 0;
}

int GenericBackend::launch(const StepArgs& a, const pcx_buffers& out, hipStream_t s) {
  if (a.export_curtains && !curtains_.ptr) {
    int rc = curtains_.alloc((size_t)(k_.ND ? k_.ND : 1) * k_.FW * bpad_);
    if (rc) return rc;
  }
  if ((a.debug & 8) && !stats_.ptr) {
    int rc = stats_.alloc(128);
    if (rc) return rc;
  }
  if (stats_.ptr) PCX_HIP(hipMemsetAsync(stats_.ptr, 0, 128 * sizeof(unsigned long long), s));
  Ptrs P{tables_.ptr, n_table_words_, state_.ptr, state_unit_, state_row_, track_.ptr, curtains_.ptr, batch_, bpad_, stats_.ptr, seed_, env_offset_,
         feat_.out_dev, feat_.depth, feat_.skip_layers, {}, 0, plot_in_.ptr};
  if (feat_.out_dev) memcpy(P.feat_ch, feat_.chars, sizeof P.feat_ch);
  // Plain steps may render from owner codes (pcx_generic_kernel.h render_codes); fused croppers cut their windows from the curtain
  // bit vectors and the feature epilogue rides the mask loop.  Whether they DO is measured together with the waves per workgroup
  // (Tuner: hello_world 262,144 environments 0.319 -> 0.230 ms with codes, better_scrolly_maze_L1 0.114 -> 0.135: the logic lane
  // writes QW code dwords per environment, the mask loop composes them on all lanes); PCX_GENERIC_CODES=0 / 1 decides by hand.
  const bool codes_ok = !fused_.on && !feat_.out_dev && !(a.debug & 4) && (spec_ ? k_spec_ : k_).l_codes >= 0;
  int codes_forced = -1;
  if (const char* e = getenv("PCX_GENERIC_CODES")) codes_forced = atoi(e) != 0;
  {
    bool launched = false;
    if (int rc = launch_pw(a, out, s, P, &launched)) return rc;
    last_pw_ = launched;
    if (launched) goto stats;
  }
  {
  // (the window corners of fused croppers are the layout's last array: without croppers it is not asked for)
  const Consts& kl = spec_ ? k_spec_ : k_;
  size_t lds = (size_t)(fused_.on ? kl.l_words : kl.l_wcorner) * 4;
  // Waves per workgroup (they share the render loop of the group's 64 environments).  The kernel's 95 VGPRs let
  // five waves onto a SIMD (20 per CU), so of the `fit` workgroups LDS has room for only 20 / n are resident with n
  // waves each -- and the logic phase (one wave per workgroup, VALU-bound) is what the kernel mostly waits for.
  // Measured at 262,144 environments (profiles/r03_tuning.md): warehouse_L0 (fit 10) 1/2/4/8 waves 0.172 / 0.162 /
  // 0.205 / 0.331 ms; walkers_scroll_groups (fit 8) 0.171 / 0.152 / 0.236 / 0.443; hello_world (fit 6, four times
  // the bytes to stream) 2 waves 0.42, 4 waves 0.33.  Hence: the most waves that still keep about 80 % of `fit`
  // workgroups resident.  When the batch has fewer groups than the chip has room for, 8 waves split the render loop.
  const int64_t groups = bpad_ / WAVE;
  const int fit = (int)((160 * 1024) / (lds ? lds : 1)) > 0 ? (int)((160 * 1024) / (lds ? lds : 1)) : 1;
  int nwaves = fit <= 2 ? 8 : fit <= 6 ? 4 : 2;
  if (spec_ && spec_->vgprs > 0) {  // the same rule with the specialised build's own register count
    const int alloc = (spec_->vgprs + 7) & ~7, per_simd = 512 / alloc < 8 ? 512 / alloc : 8, per_cu = 4 * (per_simd > 0 ? per_simd : 1);
    nwaves = 5 * per_cu >= 8 * 4 * fit ? 8 : 5 * per_cu >= 4 * 4 * fit ? 4 : 2;
  }
  int forced = 0;
  if (const char* e = getenv("PCX_GENERIC_WAVES")) { const int v = atoi(e); if (v >= 1 && v <= 8) forced = v; }
  tuner_.nc = codes_ok && codes_forced < 0 ? 8 : 4;
  bool masks = !codes_ok;
  if (forced) nwaves = forced;
  else if (groups < (int64_t)num_cus_ * (fit < 4 ? fit : 4)) { nwaves = 8; masks = true; }  // the chip is underfilled: split the render loop further (all lanes compose: masks)
  else { const int c = tuner_.pick(nwaves, a, s); nwaves = c & 0xFF; masks = masks || (c & 0x100); }  // ... and where it is not, the rule is only the first guess (see Tuner)
  if (codes_forced >= 0) masks = !codes_forced;
  P.use_codes = codes_ok && !masks;
  if (lds > 64 * 1024)
    PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(pcx_generic_step), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
  if (spec_) {
    const crop::FusedCrops* fcp = fused_.ptr();
    void* params[] = {const_cast<Consts*>(&kl), &P, const_cast<StepArgs*>(&a), const_cast<pcx_buffers*>(&out), &fcp};
    PCX_HIP(hipModuleLaunchKernel(spec_->fn, (unsigned)groups, 1, 1, (unsigned)(nwaves * WAVE), 1, 1, (unsigned)lds, s, params, nullptr));
  } else {
    hipLaunchKernelGGL(pcx_generic_step, dim3((unsigned)groups), dim3(nwaves * WAVE), lds, s, k_, P, a, out, fused_.ptr());
  }
  PCX_HIP(hipGetLastError());
  tuner_.launched(s);
  }
stats:
  if (stats_.ptr) {  // debugging aid: where the logic phase spends its cycles (lane 0 of every group)
    unsigned long long h[128];
    PCX_HIP(hipStreamSynchronize(s));
    PCX_HIP(hipMemcpy(h, stats_.ptr, sizeof h, hipMemcpyDeviceToHost));
    static int printed = 0;
    if (printed++ % 32 == 8) {
      const double n = (double)(h[69] ? h[69] : 1);
      fprintf(stderr, "[pcx generic] cycles per group: load %.0f, update groups %.0f, write-back %.0f, occlusion %.0f (flat vectors %.0f, curtain pairs %.0f, sprite cells %.0f, resolve %.0f, descriptors + track %.0f), logic total %.0f; by program id mod 8:",
              h[64] / n, h[65] / n, h[66] / n, h[68] / n, h[70] / n, (h[71] - h[70]) / n, (h[72] - h[71]) / n, (h[73] - h[72]) / n,
              (h[68] - h[73]) / n, h[67] / n);
      for (int p = 0; p < 8; ++p) if (h[p]) fprintf(stderr, " %d:%.0f", p, h[p] / n);
      fprintf(stderr, "\n");
    }
  }
  return 0;
}

int GenericBackend::read_things(int64_t env0, int64_t n, pcx_sprite_state* sprites, uint8_t* curtains) {
  const Consts& k = k_;
  std::vector<uint32_t> st((size_t)k.NW * n);
  PCX_HIP(hipDeviceSynchronize());
  for (int w = 0; w < k.NW; ++w)
    PCX_HIP(hipMemcpy(st.data() + (size_t)w * n, state_.ptr + (size_t)w * bpad_ + env0, n * 4, hipMemcpyDeviceToHost));
  auto word = [&](int w, int64_t i) { return st[(size_t)w * n + i]; };
  for (int64_t i = 0; i < n; ++i) {
    if (sprites)
      for (int s = 0; s < k.NS; ++s) {
        pcx_sprite_state& o = sprites[i * k.NS + s];
        memset(&o, 0, sizeof o);
        const uint32_t pw = word(W_SPRITES + s, i);
        o.vrow = (int16_t)(pw & 0xFFFF); o.vcol = (int16_t)(pw >> 16);
        const bool on = o.vrow >= 0 && o.vrow < k.R && o.vcol >= 0 && o.vcol < k.C;
        o.row = on ? o.vrow : 0; o.col = on ? o.vcol : 0;
        o.visible = (word(k.w_sflags + (s >> 2), i) >> (8 * (s & 3))) & 1;
      }
    if (curtains)
      for (int d = 0; d < k.ND; ++d)
        for (int r = 0; r < k.R; ++r)
          for (int c = 0; c < k.C; ++c)
            curtains[((size_t)i * k.ND + d) * k.cells + r * k.C + c] =
                (word(k.w_drapes + (d * k.R + r) * k.RW + (c >> 5), i) >> (c & 31)) & 1;
  }
  return 0;
}

}  // namespace gen

Backend* make_generic_backend() { return new gen::GenericBackend(); }

int generic_specialise_check(const pcx_template& t, char* log, int64_t log_bytes, int64_t* code_bytes) {
  gen::GenericBackend b;
  if (int rc = b.plan(t, 64)) return rc;
  return b.specialise_check(log, log_bytes, code_bytes);
}

}  // namespace pcx
