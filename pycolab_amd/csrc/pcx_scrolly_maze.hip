// pcx_scrolly_maze.hip -- fused step kernel for the scrolly_maze game family
// (reference: pycolab/examples/scrolly_maze.py driven by engine.py:583-847,
// prefab_parts/sprites.py MazeWalker, prefab_parts/drapes.py Scrolly and
// protocols/scrolling.py).  Written for gfx950 only.
//
// One launch = one Engine.play() for every environment of the batch.
//
// Mapping to the hardware:
//   * a workgroup is ONE wavefront and owns 64 consecutive environments;
//   * phase A, lane == environment: the per-environment state (a dozen
//     32-bit words, SoA over the batch, so every load/store is a coalesced
//     256-byte wave access) is stepped through the three update groups.  The
//     intermediate repaints of engine.py:735 are never materialised: the few
//     board cells MazeWalker._check_motion looks at are evaluated lazily from
//     a register snapshot of "what the last repaint would have shown";
//   * phase A leaves, in LDS, each environment's two drape curtains as R
//     bit-rows and its sprite cells;
//   * phase B, the wavefront streams the observation: 64 lanes walk the
//     (environment, 4-cell group) space, each lane composes one board dword
//     in z-order from LDS, derives the L layer dwords from it with byte-wise
//     SWAR compares, and stores 1+L dwords; a wave store covers 256
//     contiguous bytes of one plane.  Nothing is read back from HBM.
//
// Shared, immutable template data (wall pattern and coin pattern as bit-rows,
// backdrop) is staged into LDS once per workgroup from L2.  Per-environment
// coins are a bitmask over the template's coins in row-major order (coins only
// disappear), 12 bytes for level 0 instead of a 4005-cell pattern; the id of the
// coin at a pattern cell is a popcount over the coin pattern's bit-rows, so a
// board probe is a handful of independent LDS reads -- no list to walk.

#include "pcx_internal.h"
#include "pcx_scrolly_maze_kernel.h"
#include "pcx_rtc.h"  // hiprtc + the cache of code objects, shared with pcx_generic.hip

#include <cstdarg>
#include <cstdlib>
#include <cstring>
#include <map>
#include <mutex>

#include "build/pcx_scrolly_rtc.inc"  // RTC_NAMES / RTC_SOURCES: this file's device-side headers as text (csrc/Makefile, tools/embed_sources.py)

namespace pcx {
namespace sm {

// ---- run-time specialisation (round 6) ---------------------------------------------------------------------------
// The instances with a level's constants compiled in (template parameter LV: 6,300 instructions and a 9 us logic phase per
// unit instead of 15,300 and 17-23 us; the cooperative small-batch instance 5,900 instead of 13,600) existed for the three
// shipped levels only -- pcx_sm_shipped.h.  A level of one's own on the example's 10x30 board with its 'abcP' cast (a new
// entry of scrolly_maze.py's MAZES_ART, scrolly_maze.py:212-242) now gets the same two instances at pcx_engine_create:
// hiprtc compiles pcx_scrolly_maze_kernel.h with the engine's own Consts as the header PCX_SM_SPEC (pcx_rtc.h: dlopen'ed
// hiprtc, code objects cached per (constants, device) in the process and on disk under $PCX_JIT_CACHE).  Engines of
// PCX_SM_JIT_MIN = 4,096 environments and more (PCX_SM_JIT=0 / 1: never / always); anything that fails on the way leaves
// the engine on the run-time-constants instances (same results; PCX_DEBUG & 16 says why); pcx_engine_launch_shape 7 = the
// persistent shape on a run-time build.
namespace jit {

static const char* const OPTIONS[] = {"--offload-arch=gfx950", "-O3", "-std=c++17", PCX_RTC_NO_PACKED_FP32, "-DPCX_SM_SPEC=\"pcx_sm_spec.h\""};
static const char* const TU = "#include \"pcx_scrolly_maze_kernel.h\"\n";
static const rtc::Program PROGRAM = {RTC_NAMES, RTC_SOURCES, RTC_COUNT, TU, "pcx_sm_spec.hip", OPTIONS, sizeof OPTIONS / sizeof OPTIONS[0], "pcx_sm_spec.h", "pcx_scrolly_maze", "pcx scrolly_maze"};

// The header a run-time build includes: the Consts as the persistent shape launches them and as init() leaves them, as words
// (tools/gen_sm_shipped.py writes pcx_sm_shipped.h the same way).  `persistent_ok`: the persistent shape can take this
// level at all (ScrollyMazeBackend::ps_shape: at most four coin words) -- otherwise only the cooperative instance is built.
// `other_shape`: not the example's board and cast -- ONE instance with the shape as template arguments (pcx_scrolly_maze_kernel.h
// PCX_SM_SPEC_SHAPE) instead of the persistent + cooperative pair.
static std::string spec_header(const Consts& persistent, const Consts& plain, bool persistent_ok, bool other_shape = false, bool unoccluded = false) {
  std::string o = "// generated by ScrollyMazeBackend (pcx_scrolly_maze.hip jit::spec_header)\n#define PCX_SM_SPEC_N " + std::to_string(CONSTS_WORDS) + "\n";
  if (!persistent_ok) o += "#define PCX_SM_SPEC_NO_PS 1\n";
  if (other_shape) {
    char buf[160];
    snprintf(buf, sizeof buf, "#define PCX_SM_SPEC_SHAPE %d, %d, %d, %d, %d, %d\n#define PCX_SM_SPEC_UNOCC %s\n", plain.NS, plain.R, plain.C, plain.L, plain.ip, plain.ie,
             unoccluded ? "true" : "false");
    o += buf;
  }
  auto words = [&](const char* name, const Consts& k) {
    uint32_t w[CONSTS_WORDS];
    memcpy(w, &k, sizeof k);
    o += "#define "; o += name; o += " \\\n ";
    char buf[16];
    for (int i = 0; i < CONSTS_WORDS; ++i) {
      snprintf(buf, sizeof buf, " 0x%08Xu%s", w[i], i + 1 < CONSTS_WORDS ? "," : "");
      o += buf;
      if (i % 8 == 7 && i + 1 < CONSTS_WORDS) o += " \\\n ";
    }
    o += "\n";
  };
  words("PCX_SM_SPEC_WORDS", persistent);
  words("PCX_SM_SPEC_PLAIN_WORDS", plain);
  return o;
}

// the two instances' names in the code object (Itanium mangling of pcx_scrolly_maze_kernel.h's explicit instantiations)
#define PCX_SM_MANGLED(targs) "_ZN3pcx2sm21pcx_scrolly_maze_stepI" targs "EEEvNS0_6ConstsENS0_4PtrsENS_8StepArgsE11pcx_buffersNS_6stream12EpilogueArgsEPKNS_4crop10FusedCropsE"
static const char* const FN_PS = PCX_SM_MANGLED("Li4ELi10ELi30ELi8ELi3ELi3ELb0ELb0ELb0ELb1ELi3ELi7");
static const char* const FN_COOP = PCX_SM_MANGLED("Li4ELi10ELi30ELi8ELi3ELi3ELb0ELb1ELb0ELb0ELi0ELi8");
#undef PCX_SM_MANGLED
static bool has_symbol(const std::vector<char>& code, const char* name) {  // (symbol names are plain text in the ELF string table)
  const size_t n = strlen(name);
  for (size_t i = 0; i + n <= code.size(); ++i) if (code[i] == name[0] && memcmp(&code[i], name, n) == 0) return true;
  return false;
}
// ... and of the one instance of another shape: the template arguments in Itanium's spelling (a negative value is `n<digits>`)
static std::string fn_shape(const Consts& k, bool unoccluded) {
  auto lit = [](int v) { return std::string("Li") + (v < 0 ? "n" + std::to_string(-v) : std::to_string(v)) + "E"; };
  return "_ZN3pcx2sm21pcx_scrolly_maze_stepI" + lit(k.NS) + lit(k.R) + lit(k.C) + lit(k.L) + lit(k.ip) + lit(k.ie) + (unoccluded ? "Lb1E" : "Lb0E") +
         "Lb0ELb0ELb0ELi0ELi9EEEvNS0_6ConstsENS0_4PtrsENS_8StepArgsE11pcx_buffersNS_6stream12EpilogueArgsEPKNS_4crop10FusedCropsE";
}
struct Loaded { hipModule_t mod = nullptr; hipFunction_t fn = nullptr, fn_coop = nullptr, fn_shape = nullptr; };  // fn: null when the level cannot take the persistent shape; fn_shape: the instance of another shape (then the only one)

// One module per (constants, device) and process; never unloaded (engines come and go, the code stays).
static const Loaded* load(const std::string& spec, int device, std::string& why, bool verbose, const std::string& shape_name = std::string()) {
  static std::mutex mu;
  static std::map<std::pair<uint64_t, int>, Loaded> mods;
  const uint64_t key = rtc::fnv(0xCBF29CE484222325ull, spec.data(), spec.size());
  std::lock_guard<std::mutex> lock(mu);
  auto it = mods.find({key, device});
  if (it != mods.end()) return (it->second.fn_coop || it->second.fn_shape) ? &it->second : nullptr;
  Loaded l;
  if (!shape_name.empty()) {  // another shape: one instance
    for (int attempt = 0; attempt < 2 && !l.fn_shape; ++attempt) {
      bool cached = false;
      const std::vector<char> code = rtc::code_object(PROGRAM, spec, why, verbose, /*read_cache=*/attempt == 0, &cached);
      if (code.empty()) break;
      l = Loaded{};
      if (hipModuleLoadData(&l.mod, code.data()) != hipSuccess) { why = "hipModuleLoadData failed"; l.mod = nullptr; (void)hipGetLastError(); }
      else if (hipModuleGetFunction(&l.fn_shape, l.mod, shape_name.c_str()) != hipSuccess) { why = "the code object does not hold the instance under the expected name"; l.fn_shape = nullptr; (void)hipGetLastError(); }
      if (!cached) break;
    }
    auto& slot = mods[{key, device}];
    slot = l;
    return slot.fn_shape ? &slot : nullptr;
  }
  for (int attempt = 0; attempt < 2 && !l.fn_coop; ++attempt) {  // (a cache entry that does not load is compiled again and replaced)
    bool cached = false;
    const std::vector<char> code = rtc::code_object(PROGRAM, spec, why, verbose, /*read_cache=*/attempt == 0, &cached);
    if (code.empty()) break;
    l = Loaded{};
    if (hipModuleLoadData(&l.mod, code.data()) != hipSuccess) { why = "hipModuleLoadData failed"; l.mod = nullptr; (void)hipGetLastError(); }
    else if (hipModuleGetFunction(&l.fn_coop, l.mod, FN_COOP) != hipSuccess) { why = "the code object does not hold the cooperative instance under the expected name"; l.fn_coop = nullptr; (void)hipGetLastError(); }
    if (l.fn_coop && hipModuleGetFunction(&l.fn, l.mod, FN_PS) != hipSuccess) { l.fn = nullptr; (void)hipGetLastError(); }
    if (!cached) break;  // (freshly compiled: a second compile would give the same)
  }
  auto& slot = mods[{key, device}];
  slot = l;
  return slot.fn_coop ? &slot : nullptr;
}

}  // namespace jit


// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

static uint32_t magic20(uint32_t divisor, uint32_t max_numerator, bool* ok) {
  uint32_t m = ((1u << 20) + divisor - 1) / divisor;
  *ok = true;
  for (uint32_t x = 0; x <= max_numerator; ++x)
    if (((uint64_t)x * m) >> 20 != x / divisor || (uint64_t)x * m > 0xFFFFFFFFull) { *ok = false; break; }
  return m;
}

class ScrollyMazeBackend : public Backend {
 public:
  int init(const pcx_template& t, int64_t batch) override;
  int launch(const StepArgs& a, const pcx_buffers& out, hipStream_t s) override;
  int read_things(int64_t env0, int64_t n, pcx_sprite_state* sprites, uint8_t* curtains) override;
  int64_t bytes_per_step() const override {
    // Algorithmic HBM bytes of one env-step in this layout:
    // read: action 4 + state words 4*NW; write: state words that change every
    // step 4*(NW-CW) (the coin mask is rewritten only on a pickup) + planes
    // (1+L)*cells + results (reward 4, reward_set 1, discount 4, done 1,
    // frame 4, error 1).
    return 4 + 4 * (int64_t)k_.NW + 4 * (int64_t)(k_.NW - k_.CW) + (int64_t)(1 + k_.L) * k_.cells + 15;
  }
  int tuner_done() const override { return tuner_.done(); }
  const char* kernel_name() const override { return "pcx_scrolly_maze_step"; }
  int launch_shape() const override { return last_shape_; }
  // Does a single step of this batch run in the cooperative launch shape (launch(): few groups per CU)?
  bool coop_shape() const {
    const bool shipped_shape = !unoccluded_ && k_.NS == 4 && k_.R == 10 && k_.C == 30 && k_.L == 8 && k_.ip == 3 && k_.ie == 3;
    int coop_below = 4;  // (as in launch(); with fused croppers a workgroup is always one group)
    if (const char* e = getenv("PCX_COOP_BELOW")) coop_below = atoi(e);
    return shipped_shape && bpad_ / WAVE < (int64_t)num_cus_ * coop_below;
  }
  // Does a plain step of the shipped shape take the persistent launch shape (3; 0: one workgroup per group)?  From four
  // units per CU up, i.e. wherever the cooperative shape does not apply (round 4: 6-23 % faster than shape 0 from 131,072
  // to 2,097,152 environments on the same box, slower at 65,536; round 5, with the 9 us logic phase: 0.045 against 0.052
  // ms at 65,536 too -- profiles/r05_tuning.md); PCX_SM_SHAPE=0 / 3 forces one for A/B runs.
  int ps_shape(const StepArgs& a) const {
    int shape = 3;
    bool asked = false;
    if (const char* e = getenv("PCX_SM_SHAPE")) { shape = atoi(e) == 3 ? 3 : 0; asked = true; }
    if (a.mode != 0 || (a.debug & ~(5 | 16)) != 0 || epi_.out || fused_.on || k_.CW > 4 || k_.NW > PS_IB_ACTION) shape = 0;
    if (!asked && bpad_ / WAVE < (int64_t)num_cus_ * 4) shape = 0;
    return shape;
  }
  // The Consts a persistent launch hands to the kernel: the workers' LDS buffers are sized by the unit (units of 32 or 16
  // environments let more workers share a CU).
  Consts ps_consts(int unit) const {
    Consts kk = k_;
    kk.lds_ps_buf_words = unit * (((k_.QW + 1) / 2) | 1) + WAVE;  // (owner codes as nibbles: the kernel's CODE_PITCH for NIB)
    kk.lds_ps_words1 = kk.lds_ps_buf0 + kk.lds_ps_buf_words;
    kk.lds_ps_wave_words = kk.lds_ps_words1 - kk.lds_ps_inbox;  // a worker's {inbox, coin masks, buffer}
    return kk;
  }
  void set_plan_only() { plan_only_ = true; }
  const Consts& consts() const { return k_; }
  bool shipped_shape() const { return !unoccluded_ && k_.NS == 4 && k_.R == 10 && k_.C == 30 && k_.L == 8 && k_.ip == 3 && k_.ie == 3; }
  bool persistent_ok() const { return k_.CW <= 4 && k_.NW <= PS_IB_ACTION; }  // (ps_shape: what the persistent shape's inbox holds)
  // another board or cast that a static-shape instance can be built for at run time: whole dwords per plane (the static-shape code
  // paths count SR * SC / 4 of them), one to six sprites, occluded layers (the raw-mask render path has only ever been
  // instantiated with a run-time shape: its static-shape build compiles and is WRONG -- tests/test_scrolly_specialised.py found it)
  bool other_shape_ok() const { return !shipped_shape() && !unoccluded_ && k_.NS >= 1 && k_.NS <= MAX_NS && k_.cells % 4 == 0 && k_.R >= 1 && k_.C >= 1; }
  std::string spec_text() const { return jit::spec_header(ps_consts(WAVE), k_, persistent_ok(), !shipped_shape(), unoccluded_); }
  // include/pcx.h pcx_scrolly_maze_specialise_check: the run-time build of a planned template, compiled (or found in the cache); no device needed
  int specialise_check(char* log, int64_t log_bytes, int64_t* code_bytes) {
    if (log && log_bytes > 0) log[0] = 0;
    if (code_bytes) *code_bytes = 0;
    if (!shipped_shape() && !other_shape_ok())
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: no run-time build for this shape (planes of whole dwords, one to six sprites); it keeps the shape-generic instance");
    if (baked_lv(k_, false))
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: a shipped level -- its instances with the constants compiled in are part of the library (pcx_sm_shipped.h)");
    std::string why;
    const std::string spec = spec_text();
    if (const char* dump = getenv("PCX_SM_DUMP_SPEC")) {  // tests: the header of a run-time build
      if (FILE* f = fopen(dump, "w")) { fputs(spec.c_str(), f); fclose(f); }
    }
    const std::vector<char> code = rtc::code_object(jit::PROGRAM, spec, why, false);
    if (log && log_bytes > 0) snprintf(log, (size_t)log_bytes, "%s", why.c_str());
    if (code_bytes) *code_bytes = (int64_t)code.size();
    if (code.empty()) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: no run-time build: %s", why.substr(0, 400).c_str());
    if (shipped_shape() ? (!jit::has_symbol(code, jit::FN_COOP) || (persistent_ok() && !jit::has_symbol(code, jit::FN_PS)))
                        : !jit::has_symbol(code, jit::fn_shape(k_, unoccluded_).c_str())) {
      if (log && log_bytes > 0) snprintf(log, (size_t)log_bytes, "the code object does not hold the instances under the names jit::load looks up");
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: the run-time build does not hold the instances under the expected names");
    }
    return 0;
  }
  // Which compiled-in instance (pcx_sm_shipped.h) has these launch-time Consts, word for word?  LV of the kernel, 0: none.
  // `persistent`: the constants as the persistent shape launches them (odd LV) or as init() leaves them (even LV).
  // PCX_SM_BAKED=0: never (A/B runs, tests of the run-time instance)
  static int baked_lv(const Consts& kk, bool persistent) {
    if (!SHIPPED_VALID) return 0;
    if (const char* e = getenv("PCX_SM_BAKED")) if (atoi(e) == 0) return 0;
    for (int lv = persistent ? 1 : 2; lv < N_BAKED; lv += 2) {
      if (lv == 5) continue;
      const Consts baked = consts_from_words(SHIPPED_WORDS[lv]);
      Consts x = kk;  // (the unit-dependent layout words travel as kernel arguments)
      x.lds_ps_buf_words = baked.lds_ps_buf_words; x.lds_ps_words1 = baked.lds_ps_words1; x.lds_ps_wave_words = baked.lds_ps_wave_words;
      if (memcmp(&x, &baked, sizeof x) == 0) return lv;
    }
    return 0;
  }
  // the epilogue / fused croppers have no multi-step instance; small batches: the cooperative shape walks up to 256 steps
  // per launch; large batches of the shipped shape: the persistent workers walk up to 64 (a launch of 64 steps of
  // 1,048,576 environments is ~35 ms: error polls and host-side cancellation stay that fine-grained)
  int max_fused_steps() const override {
    if (epi_.out || fused_.on) return 1;
    if (fused_ok_) return 256;
    StepArgs probe;
    const bool shipped_shape = !unoccluded_ && k_.NS == 4 && k_.R == 10 && k_.C == 30 && k_.L == 8 && k_.ip == 3 && k_.ie == 3;
    if (const char* f = getenv("PCX_FUSE_STEPS")) if (atoi(f) == 0) return 1;
    // ... where walking the steps inside the launch pays (profiles/r06_stepn_crossover.txt: a multi-step launch keeps every worker on
    // its own units -- no ramp, no tail between steps -- but assigns them statically; 65,536 environments 0.0437 -> 0.0285 ms per
    // step, 524,288: 0.302 -> 0.291, 786,432: 0.434 -> 0.445, 1,048,576: 0.573 -> 0.592: above ~650,000 environments tickets and
    // stealing win more than the launches' ends cost, and step_n issues single-step launches; PCX_FUSE_STEPS=2: always fused)
    const bool force_fused = getenv("PCX_FUSE_STEPS") && atoi(getenv("PCX_FUSE_STEPS")) == 2;
    if (batch_ > 655360 && !force_fused) return 1;
    return shipped_shape && ps_shape(probe) == 3 && !(getenv("PCX_SM_CODES") && atoi(getenv("PCX_SM_CODES")) == 0) ? 64 : 1;
  }
  // include/pcx.h pcx_engine_fuse_croppers: the instances that render from curtain bit vectors + sprite
  // descriptors cut the windows too (pcx_stream.h stream_windows); the owner-code and multi-step instances step aside
  bool fused_window_features() const override { return true; }
  int set_fused_croppers(const crop::FusedCrops* fc) override {
    if (fc && fc->n > 0 && (unoccluded_ || epi_.out))
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: fused croppers need occluded layers and no feature-array epilogue");
    // (round 4: the cooperative shape moves windows that follow a drape after its export of the curtains)
    return fused_.set(fc, false, k_.R, k_.C);
  }
  const int32_t* sprite_track() const override { return track_.ptr; }
  const uint32_t* curtain_bits() const override { return curtains_.ptr; }
  int ensure_curtains() override { return curtains_.ptr ? 0 : curtains_.alloc((size_t)2 * k_.FW * bpad_); }
  int curtain_words() const override { return k_.FW; }
  int64_t batch_pad() const override { return bpad_; }
  void persistent_arrays(std::vector<std::pair<void*, size_t>>& out) override {  // pcx_engine_export_state
    out.push_back({state_.ptr, state_.count * sizeof(uint32_t)});
    out.push_back({track_.ptr, track_.count * sizeof(int32_t)});
  }
  int plane_pitch() const override { return (k_.cells + 3) & ~3; }
  stream::EpilogueArgs* epilogue_args() override { return &epi_; }
  int set_epilogue(const pcx_epilogue_desc* d) override {
    const bool shipped_shape = !unoccluded_ && k_.NS == 4 && k_.R == 10 && k_.C == 30 && k_.L == 8 && k_.ip == 3 && k_.ie == 3;
    if (d && fused_.on) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: release the fused croppers first");
    if (d && !shipped_shape)
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: the feature-array epilogue exists for the shipped 10x30 shape");
    int sc[MAX_NS], dc[2] = {k_.maze_ch, k_.cash_ch}, bc[MAX_L];
    for (int s = 0; s < k_.NS; ++s) sc[s] = k_.sprite_ch[s];
    for (int i = 0; i < k_.n_bchars; ++i) bc[i] = k_.bchar[i];
    if (!stream::fill_epilogue(epi_, d, k_.cells, sc, k_.NS, dc, 2, bc, k_.n_bchars, 64 * 1024 - (size_t)k_.lds_words * 4, 8))
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: the channels-last epilogue needs rows*cols %% 4 == 0 and a stack whose exchange areas fit the LDS left");
    // array-only consumers (skip_board): the value array gets a sweep of its own and the general one is left out
    // (1,048,576 environments: 0.60-0.69 ms against 1.16-1.26 in the general loop; with planes to write as well, one sweep)
    if (epi_.to_array) epi_.two_pass = epi_.skip_board;
    return 0;
  }

 private:
  Consts k_{};
  stream::EpilogueArgs epi_{};
  stream::FusedCropsHolder fused_;
  bool fused_ok_ = false;  // shipped shape and a batch small enough for the four-wave shapes
  int64_t batch_ = 0, bpad_ = 0;
  DevArray<uint32_t> walls_, backdrop4_, state_, curtains_;
  DevArray<uint32_t> coinbits_;
  DevArray<uint16_t> rowbase_;
  DevArray<int32_t> track_;
  DevArray<uint32_t> ps_ctr_, ps_prof_;
  ShapeTuner tuner_;
  int last_shape_ = -1;
  const jit::Loaded* spec_ = nullptr;  // the instances built for this engine's level at run time, when there are any
 public:
  // the phase timers of the last persistent launch (PCX_SM_PROF=1): 16 words per workgroup, see Ptrs::ps_prof
  int read_debug_counters(uint32_t* out_host, int64_t words) override {
    if (!ps_prof_.ptr) return set_error(PCX_E_STATE, "scrolly_maze backend: no phase timers (PCX_SM_PROF)");
    PCX_HIP(hipDeviceSynchronize());
    if (!out_host) {  // (words == -1: clear)
      PCX_HIP(hipMemset(ps_prof_.ptr, 0, ps_prof_.count * sizeof(uint32_t)));
      return 0;
    }
    if ((size_t)words > ps_prof_.count) words = (int64_t)ps_prof_.count;
    PCX_HIP(hipMemcpy(out_host, ps_prof_.ptr, (size_t)words * 4, hipMemcpyDeviceToHost));
    return 0;
  }
 private:
  std::vector<uint8_t> walls_pattern_, coin_pattern_;  // host copies for read_things
  std::vector<uint16_t> h_rowstart_;
  std::vector<uint8_t> h_coincol_;
  int maze_di_ = 0, cash_di_ = 0;
  int num_cus_ = 256;
  int max_lds_ = 64 * 1024;  // per workgroup (hipDeviceProp_t::sharedMemPerBlock)
  bool unoccluded_ = false;
  bool plan_only_ = false;
};

int ScrollyMazeBackend::init(const pcx_template& t, int64_t batch) {
  Consts& k = k_;
  batch_ = batch;
  bpad_ = (batch + WAVE - 1) / WAVE * WAVE;
  unoccluded_ = !t.occlusion_in_layers;
  if (t.n_directives) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: plot directives belong to tabled entities");
  if (t.n_drapes != 2 || t.n_sprites < 1 || t.n_sprites > MAX_NS)
    return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: expects 2 Scrolly drapes and 1..%d sprites", MAX_NS);
  k.R = t.rows; k.C = t.cols; k.cells = t.rows * t.cols; k.L = t.n_chars; k.NS = t.n_sprites;
  k.n_things = t.n_things; k.n_actions = t.n_actions;
  if (k.C > 32 || k.L > MAX_L || k.n_things > MAX_Z || k.cells > 4096)
    return set_error(PCX_E_UNSUPPORTED,
                     "scrolly_maze backend: needs cols <= 32 and <= %d characters", MAX_L);
  k.QW = (k.cells + 3) / 4;
  bool ok1, ok2;
  k.magic_q = magic20(k.QW, WAVE * k.QW, &ok1);
  k.magic_c = magic20(k.C, k.cells, &ok2);
  if (!ok1 || !ok2) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: board too large for 20-bit reciprocal");
  for (int i = 0; i < k.L; ++i) k.chars[i] = t.chars[i];

  maze_di_ = cash_di_ = -1;
  for (int i = 0; i < 2; ++i) {
    if (!t.drapes[i].is_scrolly) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: drapes must be Scrolly");
    if (t.drapes[i].program == PCX_PROG_SM_MAZE) maze_di_ = i;
    if (t.drapes[i].program == PCX_PROG_SM_CASH) cash_di_ = i;
  }
  if (maze_di_ < 0 || cash_di_ < 0) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: need one MazeDrape and one CashDrape");
  const pcx_drape_desc& md = t.drapes[maze_di_];
  const pcx_drape_desc& cd = t.drapes[cash_di_];
  if (md.pattern_rows != cd.pattern_rows || md.pattern_cols != cd.pattern_cols ||
      md.have_margins != cd.have_margins || md.margin_rows != cd.margin_rows || md.margin_cols != cd.margin_cols)
    return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: both Scrolly drapes must share pattern size and margins");
  k.PR = md.pattern_rows; k.PC = md.pattern_cols; k.WPR = (k.PC + 31) / 32 + 1;  // +1: window reads 2 words
  if (k.PR > 1024 || k.PC > 255) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: pattern larger than 1024x255");
  k.lim_r = k.PR - k.R; k.lim_c = k.PC - k.C;
  k.have_margins = md.have_margins;
  k.margin_n = md.margin_rows - 1; k.margin_s = k.R - md.margin_rows;  // drapes.py:355-358
  k.margin_w = md.margin_cols - 1; k.margin_e = k.C - md.margin_cols;
  k.maze_ch = md.ch; k.cash_ch = cd.ch;

  // update schedule must be [maze] [sprites...] [cash]
  if (t.n_groups != 3 || t.n_things != t.n_sprites + 2 || t.schedule[0] != md.ch || t.group_of[0] != 0 ||
      t.schedule[t.n_things - 1] != cd.ch || t.group_of[t.n_things - 1] != 2)
    return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: update schedule must be [[maze],[sprites...],[cash]]");
  // The kernel numbers the sprites in update order (their order inside group
  // 1); the template lists them in engine insertion order, which is the z-order
  // for ascii_art games (ascii_art.py:278-283).  sp[s] = the template's
  // description of sprite s, tmpl_index[s] = its place in the template.
  for (int s = 0; s < t.n_sprites; ++s) if (t.sprites[s].scrolling_group) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: one scrolling group only");
  for (int d = 0; d < t.n_drapes; ++d) if (t.drapes[d].scrolling_group) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: one scrolling group only");
  const pcx_sprite_desc* sp[MAX_NS] = {};
  for (int s = 0; s < t.n_sprites; ++s) {
    k.tmpl_index[s] = -1;
    for (int j = 0; j < t.n_sprites; ++j)
      if (t.sprites[j].ch == t.schedule[1 + s]) k.tmpl_index[s] = j;
    if (k.tmpl_index[s] < 0 || t.group_of[1 + s] != 1)
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: update group 1 must hold exactly the sprites");
    sp[s] = &t.sprites[k.tmpl_index[s]];
  }
  k.ip = k.ie = -1;
  for (int s = 0; s < t.n_sprites; ++s) {
    const pcx_sprite_desc& sd = *sp[s];
    if (!sd.is_walker)
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: sprites must be MazeWalkers");
    k.prog[s] = sd.program; k.confined[s] = sd.confined; k.egocentric[s] = sd.egocentric; k.sprite_ch[s] = sd.ch;
    if (sd.program == PCX_PROG_SM_PLAYER) {
      if (k.ip >= 0) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: one player only");
      k.ip = s;
    } else if (sd.program != PCX_PROG_SM_PATROLLER) {
      return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: unknown sprite program %d", sd.program);
    }
    if (sd.egocentric) {
      if (k.ie >= 0) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: at most one egocentric sprite");
      k.ie = s;
    }
    for (int j = 0; j < 4; ++j) memcpy(&k.imp[s][j], sd.impassable + 4 * j, 4);
  }
  if (k.ip < 0 || sp[k.ip]->ch != 'P')
    return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: the player sprite must paint 'P' (things['P'] lookups)");
  if (md.ch != '#') return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: the maze drape must paint '#' (things['#'] lookups)");

  // z-order tables and, per walker, which things can change a probe's verdict
  auto imp_has = [&](int s, int ch) { return (k.imp[s][ch >> 5] >> (ch & 31)) & 1; };
  for (int z = 0; z < t.n_things; ++z) {
    int ch = t.z_order[z], idx = -1, kind = 0;
    for (int s = 0; s < t.n_sprites; ++s) if (sp[s]->ch == ch) { idx = s; kind = 0; }
    if (ch == md.ch) { idx = 0; kind = 1; }
    if (ch == cd.ch) { idx = 1; kind = 1; }
    if (idx < 0) return set_error(PCX_E_INVALID, "z_order names an unknown character");
    k.z_kind[z] = kind; k.z_idx[z] = idx; k.z_ch[z] = ch;
  }
  for (int z = 0; z < t.n_things; ++z) {
    if (k.z_kind[z] == 0) k.zpos_sprite[k.z_idx[z]] = z;
    else if (k.z_idx[z] == 0) k.zpos_maze = z;
    else k.zpos_cash = z;
  }
  for (int s = 0; s < t.n_sprites; ++s) {
    bool back_imp = false;
    for (int i = 0; i < t.rows * t.cols; ++i) back_imp |= imp_has(s, t.backdrop[i]);
    k.relevant_backdrop[s] = back_imp;
    uint32_t rel = 0, impz = 0;
    bool deeper_matters = back_imp;  // walking back to front
    for (int z = 0; z < t.n_things; ++z) {
      bool mine = imp_has(s, k.z_ch[z]);
      if (mine) impz |= 1u << z;
      if (mine || deeper_matters) rel |= 1u << z;
      deeper_matters |= mine;
    }
    k.relevant[s] = rel;
    k.imp_z[s] = impz;
  }

  // occlusion tables: which things are in front of each thing; layer planes
  {
    int zpos[MAX_NS + 2];
    for (int z = 0; z < t.n_things; ++z) zpos[k.z_kind[z] ? t.n_sprites + k.z_idx[z] : k.z_idx[z]] = z;
    for (int a = 0; a < t.n_sprites + 2; ++a) {
      k.above[a] = 0;
      for (int b = 0; b < t.n_sprites + 2; ++b)
        if (zpos[b] > zpos[a]) k.above[a] |= 1u << b;
    }
    auto layer_of = [&](int ch) { for (int i = 0; i < k.L; ++i) if ((int)k.chars[i] == ch) return i; return -1; };
    for (int s = 0; s < t.n_sprites; ++s) k.lay_sprite[s] = layer_of(sp[s]->ch);
    k.lay_drape[0] = layer_of(md.ch);
    k.lay_drape[1] = layer_of(cd.ch);
    k.n_bchars = 0;
    for (int i = 0; i < k.L; ++i) {
      int ch = (int)k.chars[i];
      bool thing = ch == md.ch || ch == cd.ch;
      for (int s = 0; s < t.n_sprites; ++s) thing |= sp[s]->ch == ch;
      if (!thing) { k.bchar[k.n_bchars] = ch; k.lay_bchar[k.n_bchars] = i; k.n_bchars++; }
    }
    if (k.n_bchars != k.L - t.n_sprites - 2) return set_error(PCX_E_INVALID, "scrolly_maze backend: inconsistent character set");
  }

  // patterns: walls as bit-rows; coins as a row-major list
  walls_pattern_.assign(md.pattern, md.pattern + (size_t)k.PR * k.PC);
  coin_pattern_.assign(cd.pattern, cd.pattern + (size_t)k.PR * k.PC);
  std::vector<uint32_t> wb((size_t)k.PR * k.WPR, 0);
  for (int r = 0; r < k.PR; ++r)
    for (int c = 0; c < k.PC; ++c)
      if (md.pattern[(size_t)r * k.PC + c]) wb[(size_t)r * k.WPR + (c >> 5)] |= 1u << (c & 31);
  h_rowstart_.assign(k.PR + 2, 0);
  h_coincol_.clear();
  for (int r = 0; r < k.PR; ++r) {
    h_rowstart_[r] = (uint16_t)h_coincol_.size();
    for (int c = 0; c < k.PC; ++c)
      if (cd.pattern[(size_t)r * k.PC + c]) h_coincol_.push_back((uint8_t)c);
  }
  h_rowstart_[k.PR] = h_rowstart_[k.PR + 1] = (uint16_t)h_coincol_.size();
  k.n_coins = (int)h_coincol_.size();
  if (k.n_coins > 65000) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: too many coins");
  k.CW = (k.n_coins + 31) / 32;
  k.NW = W_SPOS + k.NS + k.CW;
  // device image: the coin pattern as bit-rows (WPR - 1 words per row: no spare word) and the
  // number of coins before every row; h_rowstart_ / h_coincol_ stay on the host (read_things)
  const int CWPR = k.WPR - 1;
  std::vector<uint32_t> cbits((size_t)k.PR * CWPR, 0);
  for (int r = 0; r < k.PR; ++r)
    for (int c = 0; c < k.PC; ++c)
      if (cd.pattern[(size_t)r * k.PC + c]) cbits[(size_t)r * CWPR + (c >> 5)] |= 1u << (c & 31);
  std::vector<uint16_t> rs = h_rowstart_;
  rs.resize((rs.size() + 3) / 2 * 2, 0);
  std::vector<uint32_t> bd4((size_t)k.QW * (2 + k.n_bchars));
  memcpy(bd4.data(), t.backdrop, k.cells);
  for (int b = 0; b < k.n_bchars; ++b) {
    uint8_t* dst = reinterpret_cast<uint8_t*>(bd4.data() + (size_t)k.QW * (1 + b));
    for (int i = 0; i < k.cells; ++i) dst[i] = t.backdrop[i] == k.bchar[b];
  }
  {  // owner codes of the backdrop (CODES instance): index of each cell's character among the sorted characters
    uint8_t* dst = reinterpret_cast<uint8_t*>(bd4.data() + (size_t)k.QW * (1 + k.n_bchars));
    for (int i = 0; i < k.cells; ++i)
      for (int c = 0; c < k.L; ++c)
        if ((int)k.chars[c] == t.backdrop[i]) dst[i] = (uint8_t)c;
    k.chars_lo = k.chars_hi = 0;
    for (int c = 0; c < k.L && c < 8; ++c) (c < 4 ? k.chars_lo : k.chars_hi) |= (k.chars[c] & 0xFFu) << (8 * (c & 3));
    int n = 0;
    for (int z = 0; z < t.n_things; ++z)
      if (k.z_kind[z] == 0) k.sprite_by_z[n++] = k.z_idx[z];
  }

  // initial state words (what the constructors left: ascii_art.py:247-277)
  memset(k.init, 0, sizeof k.init);
  k.init[W_FRAME] = (uint32_t)-1;  // plot.py: frame starts at -1, play() makes it 0
  k.init[W_FLAGS] = 0;
  k.init[W_PERMIT_FRAME] = 0;
  k.init[W_MAZE] = ((uint32_t)md.corner_row & 0xFFFFu) | ((uint32_t)md.corner_col << 16);
  k.init[W_CASH] = ((uint32_t)cd.corner_row & 0xFFFFu) | ((uint32_t)cd.corner_col << 16);
  k.init[W_STALE] = STALE_NONE;
  uint32_t sf = 0;
  for (int s = 0; s < t.n_sprites; ++s) {
    const pcx_sprite_desc& sd = *sp[s];
    k.init[W_SPOS + s] = ((uint32_t)sd.vrow & 0xFFFFu) | ((uint32_t)sd.vcol << 16);
    uint32_t var = sd.program == PCX_PROG_SM_PATROLLER ? (uint32_t)(sd.param[0] != 0) : 0u;  // _moving_east, scrolly_maze.py:282
    sf |= ((uint32_t)(sd.visible != 0) | ((uint32_t)(sd.prior_visible != 0) << 1) | (var << 2)) << (4 * s);
  }
  k.init[W_SFLAGS] = sf;
  // the initial curtains must be the pattern windows the Scrolly ctor made
  for (int di = 0; di < 2; ++di) {
    const pcx_drape_desc& d = t.drapes[di];
    for (int r = 0; r < k.R; ++r)
      for (int c = 0; c < k.C; ++c)
        if (d.curtain[r * k.C + c] != d.pattern[(size_t)(d.corner_row + r) * k.PC + d.corner_col + c])
          return set_error(PCX_E_INVALID, "scrolly_maze backend: drape curtain is not the pattern window");
  }

  // LDS layout
  int off = 0;
  k.lds_walls = off; off += k.PR * k.WPR;
  k.lds_backdrop = off; off += k.QW;
  k.lds_rowstart = off; off += k.PR * CWPR;      // the coin pattern's bit-rows
  k.lds_coincol = off; off += (int)rs.size() / 2;  // coins before every row
  k.FW = (k.cells + 31) / 32 + 1;
  // per-group render descriptors
  const int buf0 = off;
  k.lds_flat = off; off += 2 * (k.FW | 1) * WAVE;
  off = (off + 1) & ~1;  // uint2 alignment
  k.lds_sdesc = off; off += 2 * k.NS * WAVE;
  k.lds_skip = off; off += WAVE;
  off = (off + 1) & ~1;
  k.lds_buf_words = off - buf0;
  k.lds_cmask = off; off += (k.CW ? k.CW : 1) * WAVE;
  k.lds_bdmask = off; off += k.n_bchars * k.QW;
  k.lds_flatraw = off; if (unoccluded_) off += 2 * (k.FW | 1) * WAVE;
  off = (off + 1) & ~1;
  k.lds_sdescraw = off; if (unoccluded_) off += 2 * k.NS * WAVE;
  k.lds_wcorner = off; off += stream::WCORNER_WORDS;  // fused croppers: the windows' corners
  k.lds_fparams = off; off += (3 + MAX_NS) * WAVE;    // cooperative shape: corners, stale coin, sprite cells
  k.lds_words = off;
  if (off * 4 > 160 * 1024) return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: template needs %d bytes of LDS", off * 4);
  {  // CODES instance: constants, coin masks, the backdrop's owner codes, one code table, the skip flags
    int o = k.lds_coincol + (int)rs.size() / 2;
    k.lds_bdcode = o; o += k.QW;
    k.lds_codes = o; o += WAVE * ((k.QW | 1) + 2);
    k.lds_cmask_c = o; o += (k.CW ? k.CW : 1) * WAVE;
    k.lds_skip_c = o; o += WAVE;
    k.lds_words_codes = o;
    // persistent shapes: the same constants, then inbox, ring, coin masks and one / PS_NB owner-code buffers
    o = k.lds_bdcode + k.QW;
    k.lds_ps_lut = o; o += 256 + (k.QW + 1) / 2;  // (the owner-code instances' bit -> nibble table and nibble backdrop)
    k.lds_ps_ring = o; o += 4;  // [3]: the streaming semaphore
    k.lds_ps_inbox = o; o += PS_IB_ROWS * WAVE;
    k.lds_ps_cmask = o; o += (k.CW ? k.CW : 1) * WAVE;
    k.lds_ps_buf0 = o;
    k.lds_ps_buf_words = WAVE * ((k.QW | 1) + 2) + WAVE;  // code table (CODE_PITCH dwords per environment) + skip flags
    k.lds_ps_words1 = o + k.lds_ps_buf_words;
  }

  if (plan_only_) return 0;  // (pcx_debug_scrolly_consts: the host half only, no device)
  {
    int dev = 0;
    hipDeviceProp_t prop;
    if (hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&prop, dev) == hipSuccess && prop.multiProcessorCount > 0)
      num_cus_ = prop.multiProcessorCount;
    if (hipGetDevice(&dev) == hipSuccess && hipGetDeviceProperties(&prop, dev) == hipSuccess && prop.sharedMemPerBlock >= 64 * 1024) {
      max_lds_ = (int)prop.sharedMemPerBlock;
      if (const char* e = getenv("PCX_SM_TRACE")) if (atoi(e)) fprintf(stderr, "[pcx] sharedMemPerBlock %zu maxSharedMemoryPerMultiProcessor %zu\n", (size_t)prop.sharedMemPerBlock, (size_t)prop.maxSharedMemoryPerMultiProcessor);
    }
  }
  {
    // several steps per launch (pcx_engine_step_n / _step_hashed) pay off where one
    // wave per group cannot fill the chip; PCX_FUSE_STEPS=0 turns them off
    int below = 4;
    if (const char* e = getenv("PCX_COOP_BELOW")) below = atoi(e);
    const char* f = getenv("PCX_FUSE_STEPS");
    fused_ok_ = !(f && atoi(f) == 0) && !unoccluded_ && k.NS == 4 && k.R == 10 && k.C == 30 && k.L == 8 && k.ip == 3 &&
                k.ie == 3 && bpad_ / WAVE < (int64_t)num_cus_ * below;
  }
  set_epilogue(nullptr);
  const bool never_baked = getenv("PCX_SM_BAKED") && atoi(getenv("PCX_SM_BAKED")) == 0;  // (A/B runs and tests of the run-time-constants instances)
  if ((shipped_shape() || other_shape_ok()) && !never_baked && !baked_lv(k_, false)) {
    // A level of one's own on the shipped shape: its own two instances with the constants compiled in (jit above).  Seconds
    // of compile time once per level, then a file read: for the batches this engine is for, not for a unit test's few
    // hundred environments.
    int64_t min_batch = 4096;
    if (const char* e = getenv("PCX_SM_JIT_MIN")) min_batch = atoll(e);
    const char* j = getenv("PCX_SM_JIT");
    const char* dbg = getenv("PCX_DEBUG");
    const bool verbose = dbg && (atoi(dbg) & 16);
    if (j ? atoi(j) != 0 : batch >= min_batch) {
      int dev = 0;
      (void)hipGetDevice(&dev);
      std::string why;
      spec_ = jit::load(spec_text(), dev, why, verbose, shipped_shape() ? std::string() : jit::fn_shape(k_, unoccluded_));
      if (spec_ && spec_->fn) {  // (the persistent shape asks for more dynamic LDS than the default limit: the module function must be told)
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(spec_->fn), hipFuncAttributeMaxDynamicSharedMemorySize, max_lds_);
        if (e != hipSuccess) {
          (void)hipGetLastError();
          why = std::string("hipFuncSetAttribute(MaxDynamicSharedMemorySize) on the module function: ") + hipGetErrorString(e);
          spec_ = nullptr;
        }
      }
      if (!spec_ && verbose) fprintf(stderr, "[pcx scrolly_maze] no run-time build: %s\n", why.c_str());
    }
  }
  int rc;
  if ((rc = walls_.upload(wb))) return rc;
  if ((rc = backdrop4_.upload(bd4))) return rc;
  if ((rc = coinbits_.upload(cbits))) return rc;
  if ((rc = rowbase_.upload(rs))) return rc;
  if ((rc = state_.alloc((size_t)k.NW * bpad_))) return rc;
  if ((rc = track_.alloc((size_t)k.NS * bpad_))) return rc;
  if ((rc = ps_ctr_.alloc(16 * 9))) return rc;  // persistent shapes: eight ticket shards and the workers-done count, 64 bytes apart
  return 0;
}

int ScrollyMazeBackend::launch(const StepArgs& a, const pcx_buffers& out, hipStream_t s) {
  if (a.export_curtains && !curtains_.ptr) {
    int rc = curtains_.alloc((size_t)2 * k_.FW * bpad_);
    if (rc) return rc;
  }
  // Launch shapes (pcx_engine_launch_shape says which one ran):
  //   10 / 12  cooperative: below four groups per CU (and for several steps per launch) a workgroup is four or eight waves
  //            around ONE group of 16-64 environments -- the steps are latency-bound there (profiles/r03_tuning.md);
  //   3 / 5    persistent workers with streaming slots: the shipped shape from 65,536 environments up (5: the instance
  //            with the shipped level's constants compiled in);
  //   0        one single-wave workgroup per group of 64 environments (logic, then render), LDS padded so that about 8
  //            share a CU -- nine interleaved write streams per wave go faster with 7-9 waves per CU than with 15+
  //            (profiles/r01_tuning.md): the shipped shape in between and whenever an epilogue or croppers are fused;
  //   20       the shape-generic instances (other boards, casts, unoccluded layers), launched like 0.
  const int64_t groups = bpad_ / WAVE;
  int waves_per_cu = 8;
  if (const char* e = getenv("PCX_WAVES_PER_CU")) waves_per_cu = atoi(e);
  const dim3 grid((unsigned)groups), block(WAVE);
  size_t lds = (size_t)k_.lds_words * 4;
  if (waves_per_cu > 0) {
    size_t want = (size_t)(160 * 1024) / (size_t)waves_per_cu;
    want &= ~(size_t)255;
    if (want > lds) lds = want;
  }
  if (const char* pad = getenv("PCX_LDS_PAD")) lds += (size_t)atoi(pad);  // occupancy experiments
  if (lds > 64 * 1024) return set_error(PCX_E_INVALID, "scrolly_maze backend: %zu bytes of LDS per workgroup", lds);
  Ptrs P{walls_.ptr, backdrop4_.ptr, coinbits_.ptr, rowbase_.ptr, state_.ptr, track_.ptr, curtains_.ptr, maze_di_, batch_, bpad_,
         ps_ctr_.ptr, WAVE, 1, 1, 1, 16, 0, 0, nullptr};
  // Specialised instances for the shipped scrolly_maze shape (10x30 board, 8 characters, 'abcP' sprites); anything else
  // takes a shape-generic instance.
  const bool shipped_shape = this->shipped_shape();
  bool use_codes = true;  // PCX_SM_CODES=0: the mask-composing render loop of round 1 (A/B; shape 0 only)
  if (const char* e = getenv("PCX_SM_CODES")) use_codes = atoi(e) != 0;
  if (fused_.on) use_codes = false;  // the windows are cut from the curtain bit vectors
  int coop_below = 4;  // groups per CU (measured crossover: profiles/r03_tuning.md; round 1: 5)
  if (const char* e = getenv("PCX_COOP_BELOW")) coop_below = atoi(e);
  const bool coop_steps = a.n_steps > 1 && fused_ok_;  // (several steps of a small batch: the cooperative shape whatever the knobs say)
  if (a.n_steps > 1 && (!shipped_shape || a.mode != 0 || epi_.out || fused_.on || (!fused_ok_ && !(use_codes && ps_shape(a) == 3))))
    return set_error(PCX_E_INVALID, "scrolly_maze backend: %d steps in one launch are not available here", a.n_steps);
  if (shipped_shape && (groups < (int64_t)num_cus_ * coop_below || coop_steps)) {
    int coop_waves = groups <= num_cus_ ? 8 : 4;  // at most one group per CU: split the render loop eight ways
    if (const char* e = getenv("PCX_COOP_WAVES")) coop_waves = atoi(e) == 4 ? 4 : 8;
    // ... and while CUs would still stand empty, halve the environments per workgroup (32, 16): the
    // descriptor tasks and the streaming of a step spread over more CUs (config 2: 4,096 environments
    // = 256 workgroups of 16)
    StepArgs ac = a;
    int epw = WAVE;
    while (epw > 16 && bpad_ / epw < (int64_t)num_cus_) epw >>= 1;
    if (const char* e = getenv("PCX_COOP_EPW")) { const int v = atoi(e); if (v == 8 || v == 16 || v == 32 || v == 64) epw = v; }
    ac.envs_per_group = epw;
    const unsigned coop_groups = (unsigned)(bpad_ / epw);
    last_shape_ = a.n_steps > 1 ? 12 : 10;  // (12: the cooperative shape walking several steps of the launch)
    if (epi_.out) {
      size_t lds_e = (size_t)k_.lds_words * 4;
      const stream::EpilogueArgs ep = stream::with_hwc_scratch(epi_, lds_e, coop_waves);
      hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, true, true>), dim3(coop_groups),
                         dim3(coop_waves * WAVE), lds_e, s, k_, P, ac, out, ep, fused_.ptr());
    } else if (const int lv = fused_.on ? 0 : baked_lv(k_, false)) {  // (round 5: config 2's latency-bound steps with the level's constants compiled in)
#define PCX_SM_COOP_LV(n) hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, true, false, false, 0, n>), dim3(coop_groups), \
                                             dim3(coop_waves * WAVE), (size_t)k_.lds_words * 4, s, k_, P, ac, out, epi_, fused_.ptr())
      if (lv == 2) PCX_SM_COOP_LV(2); else if (lv == 4) PCX_SM_COOP_LV(4); else PCX_SM_COOP_LV(6);
#undef PCX_SM_COOP_LV
    } else if (spec_ && !fused_.on) {  // (round 6: ... and those of a level of one's own, compiled at pcx_engine_create)
      const crop::FusedCrops* fcp = fused_.ptr();
      void* params[] = {const_cast<Consts*>(&k_), &P, &ac, const_cast<pcx_buffers*>(&out), &epi_, &fcp};
      PCX_HIP(hipModuleLaunchKernel(spec_->fn_coop, coop_groups, 1, 1, (unsigned)(coop_waves * WAVE), 1, 1, (unsigned)((size_t)k_.lds_words * 4), s, params, nullptr));
    } else
      hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, true>), dim3(coop_groups),
                         dim3(coop_waves * WAVE), (size_t)k_.lds_words * 4, s, k_, P, ac, out, epi_, fused_.ptr());
  } else if (shipped_shape && use_codes && ps_shape(a) == 3) {
    // persistent workers (see the kernel): workgroups stay on their CU, their waves draw work units
    int unit = WAVE, per_cu = 3, dynamic = 1, waves = 2;
    if (const char* e = getenv("PCX_SM_UNIT")) { const int v = atoi(e); if (v == 16 || v == 32 || v == 64) unit = v; }
    const Consts kk = ps_consts(unit);
    const int baked = baked_lv(kk, true);  // (LV) an instance with the level's constants compiled in steps a unit in ~9 us, the other in ~20
    const bool jitted = !baked && spec_ && spec_->fn;  // ... built at run time
    const int64_t units64 = bpad_ / WAVE;
    if (!baked && !jitted) {
      // (round 4) two workers per workgroup, one of them streaming.  Few units per worker (config 5's shard: 2,048 units): four
      // workgroups per CU, every unit somebody's first, no tickets; up to a few units per worker: three per CU,
      // static round-robin (a drawn ticket commits a worker to one more unit -- the tail -- which costs more than the
      // imbalance it removes until a worker walks four or five units: 262,144 environments 0.178 static / 0.187 tickets,
      // 524,288: 0.330 / 0.323); beyond: three per CU, tickets
      per_cu = units64 <= (int64_t)num_cus_ * 8 ? 4 : 3;
    } else {
      // (round 5) with a 9 us logic phase fewer workers keep the streaming slots busy, and slots SHARED by all workers of a CU
      // (one workgroup of four, two slots) beat private ones (two workgroups of two, one slot each): 1,048,576 environments
      // 0.562 / 0.576 ms, 524,288: 0.300 / 0.303, 262,144: 0.152 / 0.156 on one box, 0.574 / 0.587 (2 x 3: 0.560) on
      // another; config 5's shard (every worker steps ONE unit): two workgroups of four, two slots each -- 0.078 against
      // 0.084-0.087 for 2 x 4 (profiles/r05_ps_sweep_call4_shapes.txt, _call5_steal.txt; the boxes differ by more than
      // the shapes do)
      // ... so the engine measures: the default and three alternatives, on its own first launches (ShapeTuner)
      struct Cand { int waves, per_cu, lock; };
      static const Cand few[ShapeTuner::NC] = {{4, 2, 2}, {8, 1, 3}, {3, 3, 1}, {2, 4, 1}};    // every worker steps one unit
      static const Cand many[ShapeTuner::NC] = {{4, 1, 2}, {2, 3, 1}, {6, 1, 3}, {4, 2, 2}};
      const bool knobs = getenv("PCX_SM_WAVES") || getenv("PCX_SM_PER_CU") || getenv("PCX_SM_LOCK") || getenv("PCX_SM_GRID") ||
                         getenv("PCX_SM_UNIT") || getenv("PCX_SM_PROF") || (getenv("PCX_SM_TUNE") && atoi(getenv("PCX_SM_TUNE")) == 0);
      if (knobs || (a.debug & ~16)) tuner_.off = true;  // (PCX_DEBUG=16: say what was chosen)
      const Cand& c = (units64 <= (int64_t)num_cus_ * 8 ? few : many)[tuner_.pick(a, s)];
      waves = c.waves;
      per_cu = c.per_cu;
      P.ps_lock = c.lock;
    }
    dynamic = units64 >= (int64_t)num_cus_ * 6 * 4;
    if (const char* e = getenv("PCX_SM_PER_CU")) { const int v = atoi(e); if (v >= 1 && v <= 16) per_cu = v; }
    if (const char* e = getenv("PCX_SM_DYNAMIC")) dynamic = atoi(e) != 0;
    if (a.n_steps > 1) dynamic = 0;  // several steps per launch: every worker keeps its own units from step to step
    if (const char* e = getenv("PCX_SM_WAVES")) { const int v = atoi(e); if (v >= 1 && v <= 12) waves = v; }  // workers per workgroup
    if (const char* e = getenv("PCX_SM_LOCK")) P.ps_lock = atoi(e);
    if (const char* e = getenv("PCX_SM_STEAL")) P.ps_steal = atoi(e) != 0;
    P.ps_unit = unit;
    P.ps_dynamic = dynamic;
    const int words3 = kk.lds_ps_inbox + waves * kk.lds_ps_wave_words;  // the staged level, then every worker's {inbox, coin masks, buffer}
    const int64_t n_units = (bpad_ + unit - 1) / unit;
    int64_t resident = (int64_t)num_cus_ * per_cu;
    if (const char* e = getenv("PCX_SM_GRID")) { const int v = atoi(e); if (v >= 1) resident = v; }  // (tests: few workgroups, many units each)
    const size_t lds_p = (size_t)words3 * 4;
    // (no LDS padding here: the grid is sized to what is resident at once, so the occupancy is the grid's)
    if (lds_p > (size_t)max_lds_) return set_error(PCX_E_INVALID, "scrolly_maze backend: %zu bytes of LDS per workgroup", lds_p);
    if (lds_p > 64 * 1024) {
      static bool raised = false;  // (more than 64 KB of dynamic LDS per workgroup has to be asked for, once per kernel)
      if (!raised) {
        PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, false, true, 3>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, max_lds_));
        PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, false, true, 3, 1>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, max_lds_));
        PCX_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, false, true, 3, 3>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, max_lds_));
        raised = true;
      }
    }
    if (!getenv("PCX_SM_GRID")) {  // no more workgroups than are resident at once: a workgroup that starts late would step its first unit late
      const int64_t fit = (int64_t)(160 * 1024) / (int64_t)((lds_p + 511) & ~(size_t)511);
      const int64_t by_regs = waves <= 12 ? 12 / waves : 1;  // (130-170 VGPRs: three waves per SIMD)
      int64_t per = per_cu < fit ? per_cu : fit;
      if (per > by_regs) per = by_regs;
      resident = (int64_t)num_cus_ * (per < 1 ? 1 : per);
    }
    const int64_t want_wgs = (n_units + waves - 1) / waves;  // (no workgroup without a unit)
    const dim3 pgrid((unsigned)(want_wgs < resident ? want_wgs : resident));
    const int64_t workers = (int64_t)pgrid.x * waves;
    if (workers >= n_units) P.ps_dynamic = 0;  // every unit is some worker's first: nothing to draw
    P.ps_n1 = P.ps_n = (uint32_t)n_units;
    {
      // PCX_SM_TAIL=t: with tickets, the last t small units per worker go in units of PCX_SM_TAIL_UNIT environments.  Off by
      // default: measured, every setting loses (1,048,576 environments: 0.614 ms without, 0.617 / 0.631 / 0.642 with
      // t = 1 / 2 / 3 in round 4, 0.569 / 0.572 in round 5 -- a small unit still costs a whole logic phase; profiles/r04_tuning.md)
      int tail = 0, small = 16;
      if (const char* e = getenv("PCX_SM_TAIL")) tail = atoi(e);
      if (const char* e = getenv("PCX_SM_TAIL_UNIT")) { const int v = atoi(e); if (v == 8 || v == 16 || v == 32) small = v; }
      const int64_t tail_envs = ((workers * tail * small + unit - 1) / unit) * unit;
      if (P.ps_dynamic && tail > 0 && small < unit && tail_envs * 4 <= bpad_) {
        const int64_t n1 = (bpad_ - tail_envs) / unit;
        P.ps_tail_unit = small;
        P.ps_n1 = (uint32_t)n1;
        P.ps_n = (uint32_t)(n1 + (bpad_ - n1 * unit + small - 1) / small);
      }
    }
    if (getenv("PCX_SM_PROF")) {
      if (!ps_prof_.ptr) { int rc = ps_prof_.alloc((size_t)16 * 65536); if (rc) return rc; }
      if (workers <= 65536) P.ps_prof = ps_prof_.ptr;
    }
    if (jitted) {
      last_shape_ = a.n_steps > 1 ? 13 : 7;  // (7: the persistent shape on the instance compiled for this engine's level at run time)
      const crop::FusedCrops* fcp = fused_.ptr();
      void* params[] = {const_cast<Consts*>(&kk), &P, const_cast<StepArgs*>(&a), const_cast<pcx_buffers*>(&out), &epi_, &fcp};
      PCX_HIP(hipModuleLaunchKernel(spec_->fn, pgrid.x, 1, 1, (unsigned)(waves * WAVE), 1, 1, (unsigned)lds_p, s, params, nullptr));
      tuner_.launched(s);
    } else if (baked) {
      // the engine's Consts are the shipped level 0's, word for word: the instance that has them as compile-time constants
      last_shape_ = a.n_steps > 1 ? 13 : 5;  // (13: persistent workers walking several steps of the launch)
      if (baked == 1)
        hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, false, true, 3, 1>), pgrid, dim3(waves * WAVE), lds_p, s, kk, P, a, out, epi_, fused_.ptr());
      else
        hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, false, true, 3, 3>), pgrid, dim3(waves * WAVE), lds_p, s, kk, P, a, out, epi_, fused_.ptr());
      tuner_.launched(s);
    } else {
      last_shape_ = a.n_steps > 1 ? 13 : 3;
      hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, false, true, 3>), pgrid, dim3(waves * WAVE), lds_p, s, kk, P, a, out, epi_, fused_.ptr());
    }
  } else if (shipped_shape && use_codes) {
    // owner-code render path: its own, smaller LDS layout, padded to the same workgroups-per-CU target
    last_shape_ = 0;
    size_t lds_c = (size_t)k_.lds_words_codes * 4;
    const stream::EpilogueArgs ep = stream::with_hwc_scratch(epi_, lds_c, 1);  // (channels-last epilogue: its exchange area)
    if (waves_per_cu > 0) {
      size_t want = ((size_t)(160 * 1024) / (size_t)waves_per_cu) & ~(size_t)255;
      if (want > lds_c) lds_c = want;
    }
    if (epi_.out)
      hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, true, true>), grid, block, lds_c, s, k_, P, a, out, ep, fused_.ptr());
    else
      hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, false, true>), grid, block, lds_c, s, k_, P, a, out, epi_, fused_.ptr());
  } else if (shipped_shape) {
    last_shape_ = 0;
    if (epi_.out) {
      size_t lds_e = (size_t)k_.lds_words * 4;
      const stream::EpilogueArgs ep = stream::with_hwc_scratch(epi_, lds_e, 1);
      if (lds > lds_e) lds_e = lds;  // (the padding towards `waves_per_cu` workgroups per CU)
      hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false, false, true>), grid, block, lds_e, s, k_, P, a, out, ep, fused_.ptr());
    } else
      hipLaunchKernelGGL((pcx_scrolly_maze_step<4, 10, 30, 8, 3, 3, false>), grid, block, lds, s, k_, P, a, out, epi_, fused_.ptr());
  } else if (spec_ && spec_->fn_shape && !epi_.out) {
    // (round 6) a level of another shape with its own instance compiled at pcx_engine_create: the shape as template arguments, the constants compiled in
    last_shape_ = 21;
    const crop::FusedCrops* fcp = fused_.ptr();
    void* params[] = {const_cast<Consts*>(&k_), &P, const_cast<StepArgs*>(&a), const_cast<pcx_buffers*>(&out), &epi_, &fcp};
    PCX_HIP(hipModuleLaunchKernel(spec_->fn_shape, grid.x, 1, 1, WAVE, 1, 1, (unsigned)lds, s, params, nullptr));
  } else {
    last_shape_ = 20;
    switch (k_.NS) {
#define PCX_SM_CASE(n)                                                                                          \
  case n:                                                                                                       \
    if (unoccluded_) hipLaunchKernelGGL((pcx_scrolly_maze_step<n, 0, 0, 0, -1, -1, true>), grid, block, lds, s, k_, P, a, out, epi_, fused_.ptr()); \
    else hipLaunchKernelGGL((pcx_scrolly_maze_step<n, 0, 0, 0, -1, -1, false>), grid, block, lds, s, k_, P, a, out, epi_, fused_.ptr());            \
    break;
      PCX_SM_CASE(1) PCX_SM_CASE(2) PCX_SM_CASE(3) PCX_SM_CASE(4) PCX_SM_CASE(5) PCX_SM_CASE(6)
#undef PCX_SM_CASE
      default: return set_error(PCX_E_UNSUPPORTED, "scrolly_maze backend: %d sprites", k_.NS);
    }
  }
  PCX_HIP(hipGetLastError());
  return 0;
}

int ScrollyMazeBackend::read_things(int64_t env0, int64_t n, pcx_sprite_state* sprites, uint8_t* curtains) {
  const Consts& k = k_;
  std::vector<uint32_t> st((size_t)k.NW * n);
  PCX_HIP(hipDeviceSynchronize());
  for (int w = 0; w < k.NW; ++w)
    PCX_HIP(hipMemcpy(st.data() + (size_t)w * n, state_.ptr + (size_t)w * bpad_ + env0, n * 4, hipMemcpyDeviceToHost));
  auto word = [&](int w, int64_t i) { return st[(size_t)w * n + i]; };
  for (int64_t i = 0; i < n; ++i) {
    if (sprites)
      for (int s = 0; s < k.NS; ++s) {
        pcx_sprite_state& o = sprites[i * k.NS + k.tmpl_index[s]];
        memset(&o, 0, sizeof o);
        uint32_t pw = word(W_SPOS + s, i);
        o.vrow = (int16_t)(pw & 0xFFFF); o.vcol = (int16_t)(pw >> 16);
        bool on = o.vrow >= 0 && o.vrow < k.R && o.vcol >= 0 && o.vcol < k.C;
        o.row = on ? o.vrow : 0; o.col = on ? o.vcol : 0;
        o.visible = (word(W_SFLAGS, i) >> (4 * s)) & 1;
      }
    if (curtains) {
      for (int di = 0; di < 2; ++di) {
        bool is_maze = di == maze_di_;
        uint32_t cw = word(is_maze ? W_MAZE : W_CASH, i);
        int cr = (int16_t)(cw & 0xFFFF), cc = (int16_t)(cw >> 16);
        uint8_t* dst = curtains + ((size_t)i * 2 + di) * k.cells;
        uint32_t stale = word(W_STALE, i);
        for (int r = 0; r < k.R; ++r)
          for (int c = 0; c < k.C; ++c) {
            int pr = cr + r, pc = cc + c;
            uint8_t v = 0;
            if (pr >= 0 && pr < k.PR && pc >= 0 && pc < k.PC) {
              if (is_maze) v = walls_pattern_[(size_t)pr * k.PC + pc];
              else
                for (int id = h_rowstart_[pr]; id < h_rowstart_[pr + 1]; ++id)
                  if (h_coincol_[id] == pc)
                    v = ((word(W_SPOS + k.NS + (id >> 5), i) >> (id & 31)) & 1) || (uint32_t)id == stale;
            }
            dst[r * k.C + c] = v;
          }
      }
    }
  }
  return 0;
}

}  // namespace sm

// include/pcx.h pcx_debug_scrolly_consts
int64_t scrolly_maze_consts(const pcx_template& t, int32_t unit, uint32_t* words, int64_t cap) {
  sm::ScrollyMazeBackend b;
  b.set_plan_only();
  const int rc = b.init(t, 64);
  if (rc) return rc;
  if (unit != 0 && unit != 16 && unit != 32 && unit != 64) return set_error(PCX_E_INVALID, "pcx_debug_scrolly_consts: units are 16, 32 or 64 environments (0: the constants as init() leaves them)");
  const sm::Consts kk = unit ? b.ps_consts(unit) : b.consts();
  if (words) {
    if (cap < sm::CONSTS_WORDS) return set_error(PCX_E_INVALID, "pcx_debug_scrolly_consts: room for %d words needed", sm::CONSTS_WORDS);
    memcpy(words, &kk, sizeof kk);
  }
  return sm::CONSTS_WORDS;
}

// include/pcx.h pcx_scrolly_maze_specialise_check
int scrolly_maze_specialise_check(const pcx_template& t, char* log, int64_t log_bytes, int64_t* code_bytes) {
  sm::ScrollyMazeBackend b;
  b.set_plan_only();
  const int rc = b.init(t, 64);
  if (rc) return rc;
  return b.specialise_check(log, log_bytes, code_bytes);
}

Backend* make_scrolly_maze_backend() { return new sm::ScrollyMazeBackend(); }

}  // namespace pcx
