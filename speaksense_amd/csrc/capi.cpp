// extern "C" boundary of libspeaksense_hip.so (include/speaksense.h).  No exceptions cross it.
#include <cstring>
#include <thread>
#include <unordered_set>

#include "engine.h"
#include "ops.h"

using namespace ss;

struct ss_engine { EngineBase* e; };
struct ss_session { Session s; };
struct ss_ticket { Job job; };
struct ss_pool { std::vector<ss_engine*> engines; std::atomic<uint32_t> cursor{0}; };

// Engines that exist.  ss_session_free may have to wait on its engine's condition variable while another thread frees that engine: the waiter
// enters (counted in EngineBase::n_waiters, which stop_worker drains) under this lock, and ss_engine_free leaves the set under it BEFORE teardown
// starts -- so a session either finds its engine alive and is waited for, or finds it gone, in which case every chunk is already complete.
// (heap-allocated and never destroyed: a host may free sessions from its own exit handlers, after this library's static destructors have run)
static std::mutex& g_live_mu = *new std::mutex();
static std::unordered_set<const EngineBase*>& g_live = *new std::unordered_set<const EngineBase*>();

static thread_local std::string g_err;
static int fail(int code, const std::string& msg) { g_err = msg; return code; }
#define SS_TRY try {
#define SS_CATCH                                                          \
    } catch (const ss::Error& e) { return fail(e.code, e.what()); }        \
    catch (const std::exception& e) { return fail(SS_ERR_DEVICE, e.what()); }  \
    catch (...) { return fail(SS_ERR_DEVICE, "unknown exception"); }

// whisper_full_with_state "prepare prompt": initial_prompt is tokenised unless prompt_tokens is given; the job keeps its own copy
static void capture_prompt(Job& j, const EngineBase* e) {
    j.prompt_tokens.clear();
    if (j.P.prompt_tokens && j.P.prompt_n_tokens > 0) j.prompt_tokens.assign(j.P.prompt_tokens, j.P.prompt_tokens + j.P.prompt_n_tokens);
    else if (j.P.initial_prompt && *j.P.initial_prompt) j.prompt_tokens = tokenize(e->hm.vocab, j.P.initial_prompt);
    if (j.prompt_tokens.size() > 1024) j.prompt_tokens.resize(1024);   // whisper.cpp tokenises the initial prompt into a 1024-token buffer
    j.P.prompt_tokens = nullptr; j.P.prompt_n_tokens = 0; j.P.initial_prompt = nullptr;
}
static int bad_prompt(const ss_params& P, const EngineBase* e) {
    if (P.prompt_n_tokens < 0 || (P.prompt_n_tokens > 0 && !P.prompt_tokens)) return 1;
    for (int i = 0; i < P.prompt_n_tokens; i++) if (P.prompt_tokens[i] < 0 || P.prompt_tokens[i] >= e->hm.hp.n_vocab) return 1;
    return 0;
}

extern "C" {

const char* ss_last_error(void) { return g_err.c_str(); }

// Diagnostics (env SS_CRASH_BACKTRACE=1): a SIGSEGV / SIGBUS / SIGABRT inside the process prints the faulting thread's native frames (module + offset;
// resolve with llvm-symbolizer / llvm-objdump on the .so) before the default action runs.  Installed when the library is loaded; off by default --
// a host service owns its signal handlers.
#include <execinfo.h>
#include <signal.h>
#include <unistd.h>
namespace {
void ss_crash_handler(int sig) {
    void* frames[48];
    const int n = backtrace(frames, 48);
    const char msg[] = "\n[speaksense] fatal signal, native frames of the faulting thread:\n";
    (void)!write(2, msg, sizeof msg - 1);
    backtrace_symbols_fd(frames, n, 2);
    signal(sig, SIG_DFL);
    raise(sig);
}
struct CrashHook {
    CrashHook() {
        const char* e = getenv("SS_CRASH_BACKTRACE");
        if (e && *e && *e != '0') { signal(SIGSEGV, ss_crash_handler); signal(SIGBUS, ss_crash_handler); signal(SIGABRT, ss_crash_handler); }
    }
} g_crash_hook;
}  // namespace

void ss_default_params(ss_params* p) {
    // whisper_full_default_params(GREEDY) + build_params (/root/reference/src/asr/whisper.rs:131-173) + stream mode (65-69)
    memset(p, 0, sizeof(*p));
    p->best_of = 5; p->temperature = 0.0f; p->temperature_inc = 0.2f; p->entropy_thold = 2.4f; p->logprob_thold = -1.0f;
    p->max_initial_ts = 1.0f; p->length_penalty = -1.0f; p->no_context = 1; p->single_segment = 0; p->no_timestamps = 0;
    p->suppress_blank = 1; p->tdrz_enable = 0; p->print_special = 0; p->max_tokens = 0; p->audio_ctx = 0; p->translate = 0;
    p->fixed_steps = 0;
    strcpy(p->language, "en");
    p->n_max_text_ctx = 16384; p->offset_ms = 0; p->duration_ms = 0; p->detect_language = 0;
    p->prompt_tokens = nullptr; p->prompt_n_tokens = 0; p->initial_prompt = nullptr;
    p->token_timestamps = 1; p->thold_pt = 0.01f; p->thold_ptsum = 0.01f;   // whisper.rs:160,170-171
    p->suppress_non_speech_tokens = 0; p->max_len = 0; p->split_on_word = 1;   // whisper.rs:156,167,161
}

int ss_engine_create(const char* path, const ss_engine_opts* opts, ss_engine** out) {
    if (!path || !out) return fail(SS_ERR_ARG, "ss_engine_create: null argument");
    *out = nullptr;
    ss_engine_opts o{};
    o.dtype = SS_DTYPE_F16;
    if (opts) o = *opts;
    if (o.max_batch <= 0) o.max_batch = 8;
    if (o.max_decoders <= 0) o.max_decoders = 5;
    if (o.max_batch * o.max_decoders > 128 * 8 || o.max_batch > 128) return fail(SS_ERR_ARG, "ss_engine_create: max_batch*max_decoders too large");
    SS_TRY
    if (o.dtype != SS_DTYPE_F16 && o.dtype != SS_DTYPE_BF16 && o.dtype != SS_DTYPE_FP8) return fail(SS_ERR_ARG, "ss_engine_create: unknown dtype");
    // SS_DTYPE_FP8 = the f16 engine with its encoder and cross-KV projections in e4m3
    EngineBase* e = o.dtype == SS_DTYPE_BF16 ? make_engine_bf16(path, o) : make_engine_f16(path, o);
    *out = new ss_engine{e};
    { std::lock_guard<std::mutex> lk(g_live_mu); g_live.insert(e); }
    if (e->hm.n_quantised > 0) {
        // VERDICT r05 #7, decided: block-quantised ggml files (script/download-ggml-model.sh:28-51, `-q5_0` / `-q5_1` / `-q8_0`) are DE-QUANTISED at load and
        // run the f16 / bf16 kernels.  whisper.cpp multiplies the quantised blocks by q8_0-quantised activations (resources/ggml-metal.metal:918-996 is
        // the Metal analogue): same weights, different arithmetic, so ids can differ on near ties.  Said at every load of such a file, and in INTEGRATION.md.
        fprintf(stderr, "[speaksense_hip] %s: %d block-quantised tensors were de-quantised to 16-bit weights at load; this engine computes in f16/bf16, "
                        "NOT in ggml's quantised-weight x q8_0-activation arithmetic, so results may differ from whisper.cpp on this file in near ties\n",
                path, e->hm.n_quantised);
    }
    return SS_OK;
    SS_CATCH
}
void ss_engine_free(ss_engine* e) {
    if (!e) return;
    { std::lock_guard<std::mutex> lk(g_live_mu); g_live.erase(e->e); }   // no new ss_session_free waiter can enter from here on
    delete e->e;                                                          // ~EngineT -> stop_worker: completes every chunk, lets the counted waiters leave
    delete e;
}
int32_t ss_abi_version(void) { return SS_ABI_VERSION; }
int32_t ss_sizeof_params(void) { return (int32_t)sizeof(ss_params); }
int32_t ss_sizeof_engine_opts(void) { return (int32_t)sizeof(ss_engine_opts); }
int ss_engine_hparams(const ss_engine* e, int32_t out11[11]) {
    if (!e || !out11) return fail(SS_ERR_ARG, "null argument");
    memcpy(out11, &e->e->hm.hp, sizeof(HParams));
    return SS_OK;
}
int ss_engine_special_tokens(const ss_engine* e, int32_t out9[9]) {
    if (!e || !out9) return fail(SS_ERR_ARG, "null argument");
    const Vocab& v = e->e->hm.vocab;
    const int t[9] = {v.token_eot, v.token_sot, v.token_translate, v.token_transcribe, v.token_solm, v.token_prev, v.token_nosp, v.token_not, v.token_beg};
    memcpy(out9, t, sizeof(t));
    return SS_OK;
}
const char* ss_engine_token_str(const ss_engine* e, int32_t id) {
    if (!e || id < 0 || id >= (int)e->e->hm.vocab.id_to_token.size()) return nullptr;
    return e->e->hm.vocab.id_to_token[id].c_str();
}

int ss_engine_tokenize(const ss_engine* e, const char* text, int32_t* ids, int32_t n_max) {
    if (!e || !text || (n_max > 0 && !ids)) return fail(SS_ERR_ARG, "ss_engine_tokenize: bad argument");
    const std::vector<int> t = tokenize(e->e->hm.vocab, text);
    if (!ids && n_max == 0) return (int)t.size();       // size query
    if ((int)t.size() > n_max) return fail(SS_ERR_BUFFER, "ss_engine_tokenize: buffer too small: " + std::to_string(t.size()) + " tokens needed");
    for (size_t i = 0; i < t.size(); i++) ids[i] = t[i];
    return (int)t.size();
}

int ss_model_tokenize(const char* path, const char* text, int32_t* ids, int32_t n_max) {
    if (!path || !text || (n_max > 0 && !ids)) return fail(SS_ERR_ARG, "ss_model_tokenize: bad argument");
    SS_TRY
    HostModel m;
    load_ggml_model(path, m, true);
    const std::vector<int> t = tokenize(m.vocab, text);
    if (!ids && n_max == 0) return (int)t.size();       // size query
    if ((int)t.size() > n_max) return fail(SS_ERR_BUFFER, "ss_model_tokenize: buffer too small: " + std::to_string(t.size()) + " tokens needed");
    for (size_t i = 0; i < t.size(); i++) ids[i] = t[i];
    return (int)t.size();
    SS_CATCH
}

ss_session* ss_session_create(ss_engine* e) {
    if (!e) return nullptr;
    ss_session* s = new ss_session();
    s->s.eng = e->e;
    return s;
}
// A session with chunks still queued or running must outlive them (the worker writes the results into it): wait until the engine has completed
// them.  Completion does not need ss_wait -- an abandoned ticket only leaks its own memory -- and after ss_engine_free every chunk is complete.
void ss_session_free(ss_session* s) {
    if (!s) return;
    if (s->s.in_flight.load() > 0) {
        EngineBase* e = s->s.eng;          // while in_flight > 0 the session stays on this engine (ss_pool_submit)
        std::unique_lock<std::mutex> live(g_live_mu);
        if (g_live.count(e)) e->wait_session_idle(s->s, live);     // releases `live` once it is counted as a waiter
        // else: the engine is being (or has been) freed -- teardown completes every chunk before it returns; spin on the counter, never touch `e`
        else { live.unlock(); while (s->s.in_flight.load() > 0) std::this_thread::yield(); }
    }
    {   // the stage hooks' decoder context may still name this session: a later session allocated at the same address must not inherit it
        std::lock_guard<std::mutex> live(g_live_mu);
        if (g_live.count(s->s.eng)) { const void* me = &s->s; s->s.eng->hook_owner.compare_exchange_strong(me, nullptr); }
    }
    delete s;
}

int32_t ss_pool_pick(const int32_t* load, int32_t n, uint32_t cursor) {
    if (!load || n <= 0) return -1;
    int best = (int)(cursor % (uint32_t)n);
    for (int k = 1; k < n; k++) {                       // scan from the cursor: among equally loaded engines the next in turn wins
        const int i = (int)((cursor + (uint32_t)k) % (uint32_t)n);
        if (load[i] < load[best]) best = i;
    }
    return best;
}
int ss_pool_create(const char* path, const int32_t* device_ids, int32_t n, const ss_engine_opts* opts, ss_pool** out) {
    if (!path || !device_ids || n <= 0 || n > 64 || !out) return fail(SS_ERR_ARG, "ss_pool_create: bad argument");
    *out = nullptr;
    ss_pool* p = new ss_pool();
    for (int i = 0; i < n; i++) {
        ss_engine_opts o{};
        o.dtype = SS_DTYPE_F16;
        if (opts) o = *opts;
        o.device = device_ids[i];
        ss_engine* e = nullptr;
        const int rc = ss_engine_create(path, &o, &e);
        if (rc != SS_OK) { ss_pool_free(p); return rc; }     // message already set by ss_engine_create
        p->engines.push_back(e);
    }
    *out = p;
    return SS_OK;
}
void ss_pool_free(ss_pool* p) {
    if (!p) return;
    for (ss_engine* e : p->engines) ss_engine_free(e);
    delete p;
}
int32_t ss_pool_n_engines(const ss_pool* p) { return p ? (int32_t)p->engines.size() : 0; }
ss_engine* ss_pool_engine(ss_pool* p, int32_t i) { return (!p || i < 0 || i >= (int)p->engines.size()) ? nullptr : p->engines[i]; }
ss_session* ss_pool_session_create(ss_pool* p) { return (!p || p->engines.empty()) ? nullptr : ss_session_create(p->engines[0]); }
int32_t ss_pool_last_engine(const ss_session* s) { return s ? s->s.pool_engine : -1; }
int ss_pool_submit(ss_pool* p, ss_session* s, const float* pcm, int32_t n_samples, const ss_params* params, ss_ticket** out) {
    if (!p || p->engines.empty() || !s) return fail(SS_ERR_ARG, "ss_pool_submit: bad argument");
    const int n = (int)p->engines.size();
    std::vector<int32_t> load(n);
    for (int i = 0; i < n; i++) load[i] = p->engines[i]->e->load.load();
    int k = ss_pool_pick(load.data(), n, p->cursor.fetch_add(1));
    // A session with a ticket outstanding stays on the engine that holds it: the one-chunk-per-session-at-a-time guard (`running` in
    // start_worker / admit_more) is per engine, so a second chunk routed elsewhere would run concurrently on the same Session state.
    if (s->s.in_flight.load() > 0 && s->s.pool_engine >= 0 && s->s.pool_engine < n) k = s->s.pool_engine;
    s->s.eng = p->engines[k]->e;       // the session's state is host-side only: this chunk runs on engine k
    s->s.pool_engine = k;
    return ss_submit(s, pcm, n_samples, params, out);
}

int ss_transcribe_batch(ss_engine* e, ss_session* const* sessions, const float* const* pcm, const int32_t* n_samples, int32_t n,
                        const ss_params* params, int32_t pcm_on_device) {
    if (!e || !sessions || !pcm || !n_samples || n <= 0) return fail(SS_ERR_ARG, "ss_transcribe_batch: bad argument");
    ss_params P;
    if (params) P = *params; else ss_default_params(&P);
    if (bad_prompt(P, e->e)) return fail(SS_ERR_ARG, "ss_transcribe_batch: bad prompt_tokens");
    std::vector<Job> jobs(n);
    std::vector<Job*> jp(n);
    for (int i = 0; i < n; i++) {
        if (!sessions[i] || (n_samples[i] > 0 && !pcm[i]) || n_samples[i] < 0) return fail(SS_ERR_ARG, "ss_transcribe_batch: bad chunk");
        for (int k = 0; k < i; k++) if (sessions[k] == sessions[i]) return fail(SS_ERR_ARG, "ss_transcribe_batch: sessions must be distinct");
        jobs[i].sess = &sessions[i]->s; jobs[i].pcm = pcm[i]; jobs[i].n_samples = n_samples[i]; jobs[i].pcm_on_device = pcm_on_device != 0;
        jobs[i].P = P;
        capture_prompt(jobs[i], e->e);
        jp[i] = &jobs[i];
    }
    SS_TRY
    e->e->run_jobs_parallel(jp);
    for (int i = 0; i < n; i++)
        if (jobs[i].status != 0) return fail(jobs[i].status, "chunk " + std::to_string(i) + " failed" + (jobs[i].err.empty() ? "" : ": " + jobs[i].err));
    return SS_OK;
    SS_CATCH
}
int ss_transcribe(ss_session* s, const float* pcm, int32_t n_samples, const ss_params* params) {
    if (!s) return fail(SS_ERR_ARG, "ss_transcribe: null session");
    ss_engine tmp{s->s.eng};
    ss_session* ss1[1] = {s};
    const float* p1[1] = {pcm};
    int32_t n1[1] = {n_samples};
    return ss_transcribe_batch(&tmp, ss1, p1, n1, 1, params, 0);
}
int ss_submit(ss_session* s, const float* pcm, int32_t n_samples, const ss_params* params, ss_ticket** out) {
    return ss_submit_ex(s, pcm, n_samples, params, 0, out);
}
int ss_submit_ex(ss_session* s, const float* pcm, int32_t n_samples, const ss_params* params, int32_t pcm_on_device, ss_ticket** out) {
    if (!s || !out || n_samples < 0 || (n_samples > 0 && !pcm)) return fail(SS_ERR_ARG, "ss_submit: bad argument");
    ss_ticket* t = new ss_ticket();
    t->job.sess = &s->s;
    if (pcm_on_device) { t->job.pcm = pcm; t->job.pcm_on_device = true; }      // device buffer: the caller keeps it alive until ss_wait
    else { t->job.owned.assign(pcm, pcm + n_samples); t->job.pcm = t->job.owned.data(); }
    t->job.n_samples = n_samples;
    if (params) t->job.P = *params; else ss_default_params(&t->job.P);
    if (bad_prompt(t->job.P, s->s.eng)) { delete t; return fail(SS_ERR_ARG, "ss_submit: bad prompt_tokens"); }
    capture_prompt(t->job, s->s.eng);
    t->job.eng = s->s.eng;             // the ticket remembers the engine that owns it (a pool session may be re-pointed before ss_wait)
    s->s.in_flight.fetch_add(1);
    s->s.eng->submit(&t->job);
    *out = t;
    return SS_OK;
}
int ss_ticket_ready(const ss_ticket* t) { return t && t->job.done.load(std::memory_order_acquire) ? 1 : 0; }
int ss_wait(ss_ticket* t) {
    if (!t) return fail(SS_ERR_ARG, "ss_wait: null ticket");
    // done already (also: the engine has been freed since, or the session has): neither is touched
    if (!t->job.done.load(std::memory_order_acquire)) t->job.eng->wait(&t->job);
    const int st = t->job.status;
    const std::string why = t->job.err.empty() ? std::string("chunk failed") : t->job.err;
    delete t;
    return st == 0 ? SS_OK : fail(st, why);
}

int32_t ss_result_n_segments(const ss_session* s) { return s ? (int32_t)s->s.segments.size() : 0; }
const char* ss_result_segment_text(const ss_session* s, int32_t i) {
    if (!s || i < 0 || i >= (int)s->s.segments.size()) return nullptr;
    return s->s.segments[i].text.c_str();
}
int64_t ss_result_segment_t0(const ss_session* s, int32_t i) { return (!s || i < 0 || i >= (int)s->s.segments.size()) ? 0 : s->s.segments[i].t0; }
int64_t ss_result_segment_t1(const ss_session* s, int32_t i) { return (!s || i < 0 || i >= (int)s->s.segments.size()) ? 0 : s->s.segments[i].t1; }
int32_t ss_result_segment_speaker_turn_next(const ss_session* s, int32_t i) {
    return (!s || i < 0 || i >= (int)s->s.segments.size()) ? 0 : (int32_t)s->s.segments[i].speaker_turn_next;
}
int32_t ss_result_segment_n_tokens(const ss_session* s, int32_t i) {
    return (!s || i < 0 || i >= (int)s->s.segments.size()) ? 0 : (int32_t)s->s.segments[i].tokens.size();
}
int ss_result_segment_token(const ss_session* s, int32_t i, int32_t k, int32_t* id, int32_t* tid, float out4[4]) {
    if (!s || i < 0 || i >= (int)s->s.segments.size() || k < 0 || k >= (int)s->s.segments[i].tokens.size()) return fail(SS_ERR_ARG, "segment token: out of range");
    const TokenData& t = s->s.segments[i].tokens[k];
    if (id) *id = t.id;
    if (tid) *tid = t.tid;
    if (out4) { out4[0] = t.p; out4[1] = t.plog; out4[2] = t.pt; out4[3] = t.ptsum; }
    return SS_OK;
}
int ss_result_segment_token_times(const ss_session* s, int32_t i, int32_t k, int64_t* t0, int64_t* t1, float* vlen) {
    if (!s || i < 0 || i >= (int)s->s.segments.size() || k < 0 || k >= (int)s->s.segments[i].tokens.size()) return fail(SS_ERR_ARG, "segment token times: out of range");
    const TokenData& t = s->s.segments[i].tokens[k];
    if (t0) *t0 = t.t0;
    if (t1) *t1 = t.t1;
    if (vlen) *vlen = t.vlen;
    return SS_OK;
}
// whisper_full_parallel's merge: append src's segments to dst shifted by t_offset centiseconds, "make sure that segments are not overlapping"
int ss_result_append(ss_session* dst, const ss_session* src, int64_t t_offset) {
    if (!dst || !src || dst == src) return fail(SS_ERR_ARG, "ss_result_append: bad argument");
    for (const Segment& g : src->s.segments) {
        Segment r = g;
        r.t0 += t_offset; r.t1 += t_offset;
        if (!dst->s.segments.empty()) r.t0 = std::max(r.t0, dst->s.segments.back().t1);
        dst->s.segments.push_back(r);
    }
    dst->s.tokens.insert(dst->s.tokens.end(), src->s.tokens.begin(), src->s.tokens.end());
    return SS_OK;
}
int32_t ss_result_n_tokens(const ss_session* s) { return s ? (int32_t)s->s.tokens.size() : 0; }
int ss_result_tokens(const ss_session* s, int32_t* ids, float* plog) {
    if (!s || !ids) return fail(SS_ERR_ARG, "null argument");
    for (size_t i = 0; i < s->s.tokens.size(); i++) { ids[i] = s->s.tokens[i].id; if (plog) plog[i] = s->s.tokens[i].plog; }
    return SS_OK;
}
int32_t ss_result_n_sampled_tokens(const ss_session* s) { return s ? (int32_t)s->s.sampled.size() : 0; }
int ss_result_sampled_tokens(const ss_session* s, int32_t* ids) {
    if (!s || !ids) return fail(SS_ERR_ARG, "null argument");
    for (size_t i = 0; i < s->s.sampled.size(); i++) ids[i] = s->s.sampled[i];
    return SS_OK;
}
int32_t ss_result_n_trace_tokens(const ss_session* s) { return s ? (int32_t)s->s.trace.size() : 0; }
int ss_result_trace_tokens(const ss_session* s, int32_t* ids) {
    if (!s || !ids) return fail(SS_ERR_ARG, "null argument");
    for (size_t i = 0; i < s->s.trace.size(); i++) ids[i] = s->s.trace[i];
    return SS_OK;
}
int32_t ss_result_lang_id(const ss_session* s) { return s ? s->s.lang_id : -1; }
int ss_result_counters(const ss_session* s, int32_t out4[4]) {
    if (!s || !out4) return fail(SS_ERR_ARG, "null argument");
    out4[0] = s->s.n_encode; out4[1] = s->s.n_decode; out4[2] = s->s.n_fail; out4[3] = s->s.n_windows;
    return SS_OK;
}

int64_t ss_session_rng_draws(const ss_session* s) { return s ? (int64_t)s->s.rng.n : 0; }
int64_t ss_session_rng_draws_decoder(const ss_session* s, int32_t decoder) {
    if (!s || decoder < 0) return 0;
    if (decoder == 0) return (int64_t)s->s.rng.n;
    return (size_t)decoder - 1 < s->s.rng_dec.size() ? (int64_t)s->s.rng_dec[(size_t)decoder - 1].n : 0;
}
int ss_session_rng_discard(ss_session* s, int64_t n) {
    if (!s || n < 0) return fail(SS_ERR_ARG, "ss_session_rng_discard: bad argument");
    s->s.rng.discard((uint64_t)n);
    return SS_OK;
}

int32_t ss_mel_n_len(int32_t n_samples) { return mel_n_len(n_samples); }
int64_t ss_dec_weight_offset(int64_t n, int32_t k, int32_t K) {
    if (n < 0 || k < 0 || K <= 0 || k >= K || K % 32) return -1;
    return dec_wpack_off(n, k, K);
}
int ss_signal_energy(ss_engine* e, const float* pcm, int32_t n, float* out) {
    if (!e || !pcm || !out || n <= 0) return fail(SS_ERR_ARG, "ss_signal_energy: bad argument");
    SS_TRY e->e->signal_energy_host(pcm, n, out); return SS_OK; SS_CATCH
}
int ss_log_mel(ss_engine* e, const float* pcm, int32_t n, float* out, int32_t n_len) {
    if (!e || !pcm || !out || n <= 0) return fail(SS_ERR_ARG, "ss_log_mel: bad argument");
    SS_TRY e->e->log_mel_host(pcm, n, out, n_len); return SS_OK; SS_CATCH
}
int ss_encode(ss_engine* e, const float* mel, int32_t n_len, int32_t seek, float* enc_out) {
    if (!e || !mel || !enc_out || n_len <= 0 || seek < 0) return fail(SS_ERR_ARG, "ss_encode: bad argument");
    SS_TRY e->e->encode_host(mel, n_len, seek, enc_out); return SS_OK; SS_CATCH
}
int ss_encode_ctx(ss_engine* e, const float* mel, int32_t n_len, int32_t seek, int32_t audio_ctx, float* enc_out) {
    if (!e || !mel || !enc_out || n_len <= 0 || seek < 0) return fail(SS_ERR_ARG, "ss_encode_ctx: bad argument");
    SS_TRY e->e->encode_host(mel, n_len, seek, enc_out, audio_ctx); return SS_OK; SS_CATCH
}
int ss_session_set_encoder(ss_session* s, const float* enc) {
    if (!s || !enc) return fail(SS_ERR_ARG, "ss_session_set_encoder: bad argument");
    SS_TRY s->s.eng->set_encoder_host(enc, 0, &s->s); return SS_OK; SS_CATCH
}
int ss_session_set_encoder_ctx(ss_session* s, const float* enc, int32_t audio_ctx) {
    if (!s || !enc) return fail(SS_ERR_ARG, "ss_session_set_encoder_ctx: bad argument");
    SS_TRY s->s.eng->set_encoder_host(enc, audio_ctx, &s->s); return SS_OK; SS_CATCH
}
int ss_engine_set_encoder_window(ss_engine* e, int32_t window, const float* enc) {
    if (!e || !enc) return fail(SS_ERR_ARG, "ss_engine_set_encoder_window: bad argument");
    SS_TRY e->e->set_encoder_window_host(enc, window); return SS_OK; SS_CATCH
}
int ss_engine_fp8_first_quant(ss_engine* e, const float* mel, int32_t n_len, int32_t seek, uint8_t* codes, uint8_t* exps) {
    if (!e || !mel || !codes || !exps || n_len <= 0 || seek < 0) return fail(SS_ERR_ARG, "ss_engine_fp8_first_quant: bad argument");
    SS_TRY e->e->fp8_first_quant_host(mel, n_len, seek, codes, exps); return SS_OK; SS_CATCH
}
int ss_engine_decode_rows(ss_engine* e, const int32_t* token, const int32_t* pos, const int32_t* slot, const int32_t* cross, int32_t n_rows,
                          const int32_t* sample_rows, int32_t n_sample_rows, float* logits_out) {
    if (!e || !token || !pos || !slot || !cross || !sample_rows || !logits_out) return fail(SS_ERR_ARG, "ss_engine_decode_rows: null argument");
    SS_TRY e->e->decode_rows_host(token, pos, slot, cross, n_rows, sample_rows, n_sample_rows, logits_out); return SS_OK; SS_CATCH
}
int ss_session_decode(ss_session* s, const int32_t* tokens, int32_t n, int32_t n_past, float* logits_out) {
    if (!s || !tokens || !logits_out || n <= 0 || n_past < 0 || n_past + n > s->s.eng->hm.hp.n_text_ctx) return fail(SS_ERR_ARG, "ss_session_decode: bad argument");
    for (int i = 0; i < n; i++) if (tokens[i] < 0 || tokens[i] >= s->s.eng->hm.hp.n_vocab) return fail(SS_ERR_ARG, "ss_session_decode: token out of range");
    SS_TRY s->s.eng->decode_host(tokens, n, n_past, logits_out, &s->s); return SS_OK; SS_CATCH
}
int ss_process_logits(ss_engine* e, const float* raw, const int32_t* hist, int32_t n_hist, int32_t has_ts, int32_t seek_delta, const ss_params* params,
                      float out6[6]) {
    if (!e || !raw || !out6 || n_hist < 0 || (n_hist > 0 && !hist)) return fail(SS_ERR_ARG, "ss_process_logits: bad argument");
    ss_params P;
    if (params) P = *params; else ss_default_params(&P);
    SS_TRY e->e->process_logits_host(raw, hist, n_hist, has_ts, seek_delta, P, out6); return SS_OK; SS_CATCH
}
int ss_process_logits_row(ss_engine* e, const float* raw, const int32_t* hist, int32_t n_hist, int32_t has_ts, int32_t seek_delta, const ss_params* params,
                          float out6[6], float* logprobs_out) {
    if (!e || !raw || !out6 || !logprobs_out || n_hist < 0 || (n_hist > 0 && !hist)) return fail(SS_ERR_ARG, "ss_process_logits_row: bad argument");
    ss_params P;
    if (params) P = *params; else ss_default_params(&P);
    SS_TRY e->e->process_logits_host(raw, hist, n_hist, has_ts, seek_delta, P, out6, logprobs_out); return SS_OK; SS_CATCH
}
// last_ms / last_cnt describe the group that most recently FINISHED on any lane (a blocking call may have run on a lane other than 0);
// each lane writes its own under its `mu`, the engine keeps which lane was last
int ss_engine_last_timing(const ss_engine* e, float out_ms[4]) {
    if (!e || !out_ms) return fail(SS_ERR_ARG, "null argument");
    EngineBase* L = e->e->lane(std::min(std::max(e->e->last_lane.load(), 0), e->e->n_lanes() - 1));
    std::lock_guard<std::mutex> lk(L->stat_mu);   // never the device-work mutex: a worker holds that for a whole (possibly unbounded) group
    memcpy(out_ms, L->last_ms, 16);
    return SS_OK;
}
int ss_engine_totals(const ss_engine* e, double out_ms[4], int64_t out_cnt[6], int32_t* n_lanes) {
    if (!e || !out_ms || !out_cnt) return fail(SS_ERR_ARG, "null argument");
    for (int i = 0; i < 4; i++) out_ms[i] = 0;
    for (int i = 0; i < 6; i++) out_cnt[i] = 0;
    const int n = e->e->n_lanes();
    for (int l = 0; l < n; l++) {
        EngineBase* L = e->e->lane(l);
        std::lock_guard<std::mutex> lk(L->stat_mu);    // a lane updates its totals at the end of a group, under this lock
        for (int i = 0; i < 4; i++) out_ms[i] += L->tot_ms[i];
        for (int i = 0; i < 6; i++) out_cnt[i] += L->tot_cnt[i];
    }
    if (n_lanes) *n_lanes = n;
    return SS_OK;
}
int ss_engine_lane_counters(const ss_engine* e, int32_t lane, int64_t out_cnt[6]) {
    if (!e || !out_cnt || lane < 0 || lane >= e->e->n_lanes()) return fail(SS_ERR_ARG, "ss_engine_lane_counters: bad argument");
    EngineBase* L = e->e->lane(lane);
    std::lock_guard<std::mutex> lk(L->stat_mu);
    for (int i = 0; i < 6; i++) out_cnt[i] = L->tot_cnt[i];
    return SS_OK;
}
int ss_engine_mem_info(const ss_engine* e, int64_t* free_bytes, int64_t* total_bytes) {
    if (!e || !free_bytes || !total_bytes) return fail(SS_ERR_ARG, "null argument");
    SS_TRY
    SS_HIP(hipSetDevice(e->e->opts.device));
    size_t f = 0, t = 0;
    SS_HIP(hipMemGetInfo(&f, &t));
    *free_bytes = (int64_t)f; *total_bytes = (int64_t)t;
    return SS_OK;
    SS_CATCH
}
int ss_engine_last_counters(const ss_engine* e, int64_t out4[4]) {
    if (!e || !out4) return fail(SS_ERR_ARG, "null argument");
    EngineBase* L = e->e->lane(std::min(std::max(e->e->last_lane.load(), 0), e->e->n_lanes() - 1));
    std::lock_guard<std::mutex> lk(L->stat_mu);
    for (int i = 0; i < 4; i++) out4[i] = L->last_cnt[i];
    return SS_OK;
}
void ss_default_denoise_config(ss_denoise_config* c) {
    // DenoiseConfig::default (/root/reference/src/audio/mod.rs:50-61)
    c->frame_size = 2048; c->overlap = 0.75f; c->strength = 0.2f; c->noise_gate = 0.003f; c->enable_noise_reduction = 1; c->threshold = 0.002f;
}
int ss_denoise_audio(ss_engine* e, const float* pcm, int32_t n, const ss_denoise_config* cfg, int32_t force_type, float* out, int32_t* noise_type,
                     float* norm_var, float* device_ms) {
    if (!e || !pcm || !out || n <= 0) return fail(SS_ERR_ARG, "ss_denoise_audio: bad argument");
    ss_denoise_config c;
    if (cfg) c = *cfg; else ss_default_denoise_config(&c);
    SS_TRY
    int nt = 0;
    e->e->denoise_host(pcm, n, c, force_type, out, &nt, norm_var, device_ms);
    if (noise_type) *noise_type = nt;
    return SS_OK;
    SS_CATCH
}
int64_t ss_resample_max_out(int64_t n, int32_t from_rate) {
    if (n <= 0 || from_rate <= 0) return 0;
    return (int64_t)((double)(n / 4096) * (4096.0 * 16000.0 / (double)from_rate + 2.0)) + 16;
}
int ss_resample_stream(ss_engine* e, const float* pcm, int64_t n, int32_t from_rate, float* out, int64_t out_cap, int64_t* n_out, int32_t* chunk_lens,
                       float* device_ms) {
    if (!e || !pcm || !out || n <= 0 || out_cap <= 0) return fail(SS_ERR_ARG, "ss_resample_stream: bad argument");
    SS_TRY e->e->resample_stream_host(pcm, n, from_rate, out, out_cap, n_out, chunk_lens, device_ms); return SS_OK; SS_CATCH
}
int64_t ss_preprocess_n_out(int64_t n_samples) { return n_samples <= 0 ? 0 : (n_samples + 2047) / 2048 * 2048; }
int ss_preprocess_stream(ss_engine* e, const float* pcm, int64_t n, const int32_t* chunk_lens, int32_t n_chunks, int32_t chunk_len,
                         const ss_denoise_config* cfg, float* out, float* gains_out, float* device_ms) {
    if (!e || !pcm || !out || n <= 0 || (chunk_lens && n_chunks <= 0)) return fail(SS_ERR_ARG, "ss_preprocess_stream: bad argument");
    ss_denoise_config c;
    if (cfg) c = *cfg; else ss_default_denoise_config(&c);
    SS_TRY e->e->preprocess_stream_host(pcm, n, chunk_lens, n_chunks, chunk_len, c, out, gains_out, device_ms); return SS_OK; SS_CATCH
}
int ss_engine_selftest_gemm(ss_engine* e, int32_t M, int32_t N, int32_t K, int32_t kind, float* max_err, float* max_ref) {
    if (!e || !max_err || !max_ref) return fail(SS_ERR_ARG, "bad argument");
    SS_TRY e->e->selftest_gemm(M, N, K, kind, max_err, max_ref); return SS_OK; SS_CATCH
}
int ss_e4m3_from_f32(const float* x, uint8_t* codes, int64_t n) {
    if (!x || !codes || n < 0) return fail(SS_ERR_ARG, "ss_e4m3_from_f32: bad argument");
    for (int64_t i = 0; i < n; i++) codes[i] = f32_to_e4m3(x[i]);
    return SS_OK;
}
int ss_engine_selftest_gemm_ex(ss_engine* e, int32_t M, int32_t N, int32_t K, int32_t kind, int32_t fp8, int32_t reps, float* max_err, float* max_ref, float* avg_ms) {
    if (!e || !max_err || !max_ref || reps < 0) return fail(SS_ERR_ARG, "bad argument");
    SS_TRY e->e->selftest_gemm_ex(M, N, K, kind, fp8, reps, max_err, max_ref, avg_ms); return SS_OK; SS_CATCH
}
int ss_engine_probe_gemm(ss_engine* e, int32_t batch, int32_t reps, float* avg_ms, double* flops) {
    if (!e || !avg_ms || !flops || reps <= 0) return fail(SS_ERR_ARG, "bad argument");
    SS_TRY e->e->probe_gemm(batch, reps, avg_ms, flops); return SS_OK; SS_CATCH
}

// ---- decoder operators on the caller's device buffers ----
}  // extern "C"

namespace {
struct OnDevice {            // the caller's device for the time of a call; the thread's current one afterwards
    int before = 0;
    bool moved = false;
    explicit OnDevice(int device) {
        SS_HIP(hipGetDevice(&before));
        if (device == before) return;
        int n = 0;
        SS_HIP(hipGetDeviceCount(&n));      // asked first: a failing hipSetDevice leaves an error that the next launch check would report as its own
        if (device < 0 || device >= n) throw Error(SS_ERR_DEVICE, "no HIP device " + std::to_string(device));
        SS_HIP(hipSetDevice(device));
        moved = true;
    }
    ~OnDevice() { if (moved) (void)hipSetDevice(before); }
};
bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// null = fine, else what is wrong
const char* bad_cache(const ss_kv_cache& c) {
    if (c.kind != SS_KV_SAME && c.kind != SS_KV_E4M3 && c.kind != SS_KV_INT8) return "unknown kind";
    if (c.dtype != SS_DTYPE_F16 && c.dtype != SS_DTYPE_BF16) return "dtype must be SS_DTYPE_F16 or SS_DTYPE_BF16";
    if (c.head_dim != 64 && c.head_dim != 128) return "head_dim must be 64 or 128";
    if (c.page_size < 16 || c.page_size > 256 || (c.page_size & (c.page_size - 1))) return "page_size must be a power of two from 16 to 256";
    if (c.n_pages <= 0 || c.n_kv_heads <= 0 || c.n_kv_heads > 4096) return "n_pages and n_kv_heads must be positive (at most 4096 heads)";
    const int64_t rows = (int64_t)c.n_kv_heads * c.page_size;
    if (c.page_stride < rows * c.head_dim || c.page_stride % 16 || c.page_stride >= (int64_t)1 << 31) return "page_stride must hold a page, be a multiple of 16 and less than 2^31";
    if (!c.k || !c.v || !aligned(c.k, 16) || !aligned(c.v, 16)) return "k and v must be 16-byte aligned device pointers";
    if (c.kind != SS_KV_SAME) {
        if (!c.k_scale || !c.v_scale || !aligned(c.k_scale, 16) || !aligned(c.v_scale, 16)) return "an 8-bit cache needs 16-byte aligned k_scale and v_scale";
        if (c.scale_stride < rows || c.scale_stride % 16 || c.scale_stride >= (int64_t)1 << 31) return "scale_stride must hold a page's rows, be a multiple of 16 and less than 2^31";
    }
    return nullptr;
}
const char* bad_batch(const ss_kv_batch& b, const ss_kv_cache& c) {
    if (b.n_seqs < 0 || b.n_tokens < 0 || b.max_new < 0 || b.min_new < 0 || b.max_len < 0) return "negative size";
    if (b.n_seqs > 1 << 20 || b.n_tokens > 1 << 24) return "too many sequences or tokens";
    if (b.max_pages <= 0 || (int64_t)b.max_pages * c.page_size >= (int64_t)1 << 30) return "max_pages * page_size must lie in (0, 2^30)";
    if (b.table_stride < b.max_pages) return "table_stride is smaller than max_pages";
    if (b.n_seqs > 0 && (!b.page_table || !b.q_start || !b.kv_len)) return "null page_table, q_start or kv_len";
    if (!aligned(b.page_table, 4) || !aligned(b.q_start, 4) || !aligned(b.kv_len, 4)) return "page_table, q_start and kv_len must be 4-byte aligned";
    if (b.min_new > b.max_new) return "min_new is larger than max_new";
    return nullptr;
}
const char* bad_rows(const ss_kv_rows* r, int n_tokens, int heads, int dim, bool written) {
    if (!r) return "null rows";
    if (n_tokens == 0) return nullptr;
    if (!r->p || !aligned(r->p, 16)) return "token rows must be 16-byte aligned device pointers";
    if (r->row_stride % 8 || r->head_stride % 8 || r->row_stride < 0 || r->head_stride < 0) return "row_stride and head_stride must be non-negative multiples of 8";
    if (r->row_stride > (int64_t)1 << 32 || r->head_stride > (int64_t)1 << 32) return "stride too large";
    if (written) {
        const bool head_inside = (heads == 1 || r->head_stride >= dim) && (n_tokens == 1 || r->row_stride >= (int64_t)(heads - 1) * r->head_stride + dim);
        const bool row_inside = (n_tokens == 1 || r->row_stride >= dim) && (heads == 1 || r->head_stride >= (int64_t)(n_tokens - 1) * r->row_stride + dim);
        if (!head_inside && !row_inside) return "rows that are written must not overlap";
    }
    return nullptr;
}
const char* bad_heads(const ss_kv_cache& c, const ss_kv_batch& b, int n_heads) {
    if (n_heads <= 0 || n_heads % c.n_kv_heads || n_heads > 1 << 16) return "n_heads must be a multiple of n_kv_heads (at most 65536)";
    if ((int64_t)b.max_new * (n_heads / c.n_kv_heads) >= (int64_t)1 << 30 || (int64_t)b.n_tokens * n_heads >= (int64_t)1 << 31) return "too many query rows";
    // workgroups of either kernel (at most 64 key ranges each)
    if ((int64_t)b.n_seqs * c.n_kv_heads * (((int64_t)b.max_new * (n_heads / c.n_kv_heads) + 63) / 64) >= (int64_t)1 << 24) return "too many sequences x heads x query tiles";
    return nullptr;
}
int refuse(const char* who, const char* why) { return fail(SS_ERR_ARG, std::string(who) + ": " + why); }
}  // namespace

extern "C" {

int32_t ss_sizeof_kv_cache(void) { return (int32_t)sizeof(ss_kv_cache); }
int32_t ss_sizeof_kv_batch(void) { return (int32_t)sizeof(ss_kv_batch); }
int32_t ss_sizeof_kv_rows(void) { return (int32_t)sizeof(ss_kv_rows); }
int32_t ss_sizeof_sample_rows_args(void) { return (int32_t)sizeof(ss_sample_rows_args); }

int ss_kv_append(const ss_kv_cache* c, const ss_kv_batch* b, const ss_kv_rows* k, const ss_kv_rows* v, int32_t device, void* stream) {
    SS_TRY
    if (!c || !b) return refuse("ss_kv_append", "null argument");
    const char* why = bad_cache(*c);
    if (!why) why = bad_batch(*b, *c);
    if (!why) why = bad_rows(k, b->n_tokens, c->n_kv_heads, c->head_dim, false);
    if (!why) why = bad_rows(v, b->n_tokens, c->n_kv_heads, c->head_dim, false);
    if (why) return refuse("ss_kv_append", why);
    OnDevice on(device);
    launch_kv_append(*c, *b, *k, *v, (hipStream_t)stream);
    return SS_OK;
    SS_CATCH
}
int ss_kv_read(const ss_kv_cache* c, const ss_kv_batch* b, const ss_kv_rows* k, const ss_kv_rows* v, int32_t device, void* stream) {
    SS_TRY
    if (!c || !b) return refuse("ss_kv_read", "null argument");
    const char* why = bad_cache(*c);
    if (!why) why = bad_batch(*b, *c);
    if (!why) why = bad_rows(k, b->n_tokens, c->n_kv_heads, c->head_dim, true);
    if (!why) why = bad_rows(v, b->n_tokens, c->n_kv_heads, c->head_dim, true);
    if (why) return refuse("ss_kv_read", why);
    OnDevice on(device);
    launch_kv_read(*c, *b, *k, *v, (hipStream_t)stream);
    return SS_OK;
    SS_CATCH
}
int64_t ss_kv_attention_workspace(const ss_kv_cache* c, const ss_kv_batch* b, int32_t n_heads) {
    SS_TRY
    if (!c || !b) return refuse("ss_kv_attention_workspace", "null argument");
    const char* why = bad_cache(*c);
    if (!why) why = bad_batch(*b, *c);
    if (!why) why = bad_heads(*c, *b, n_heads);
    if (why) return refuse("ss_kv_attention_workspace", why);
    return kv_attention_plan(*c, *b, n_heads).workspace;
    SS_CATCH
}
int ss_kv_attention(const ss_kv_cache* c, const ss_kv_batch* b, const ss_kv_rows* q, int32_t n_heads, float scale, int32_t causal, const ss_kv_rows* out, float* lse,
                    void* workspace, int64_t workspace_bytes, int32_t device, void* stream) {
    SS_TRY
    if (!c || !b) return refuse("ss_kv_attention", "null argument");
    const char* why = bad_cache(*c);
    if (!why) why = bad_batch(*b, *c);
    if (!why) why = bad_heads(*c, *b, n_heads);
    if (!why) why = bad_rows(q, b->n_tokens, n_heads, c->head_dim, false);
    if (!why) why = bad_rows(out, b->n_tokens, n_heads, c->head_dim, true);
    if (!why && !(scale == scale && scale - scale == 0.0f)) why = "scale must be finite";
    if (!why && !aligned(lse, 4)) why = "lse must be 4-byte aligned";
    if (why) return refuse("ss_kv_attention", why);
    const int64_t need = kv_attention_plan(*c, *b, n_heads).workspace;
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return fail(workspace && aligned(workspace, 16) ? SS_ERR_BUFFER : SS_ERR_ARG,
                    "ss_kv_attention: needs " + std::to_string(need) + " bytes of 16-byte aligned workspace, got " + std::to_string(workspace ? workspace_bytes : 0));
    OnDevice on(device);
    launch_kv_attention(*c, *b, *q, n_heads, scale, causal != 0, *out, lse, workspace, (hipStream_t)stream);
    return SS_OK;
    SS_CATCH
}
int ss_sample_rows(const ss_sample_rows_args* a, int32_t device, void* stream) {
    SS_TRY
    if (!a) return refuse("ss_sample_rows", "null argument");
    const int size = a->dtype == SS_DTYPE_F32 ? 4 : 2;
    const char* why = nullptr;
    if (a->dtype != SS_DTYPE_F32 && a->dtype != SS_DTYPE_F16 && a->dtype != SS_DTYPE_BF16) why = "dtype must be SS_DTYPE_F32, SS_DTYPE_F16 or SS_DTYPE_BF16";
    else if (a->n_rows < 0 || a->n_rows > 1 << 21) why = "n_rows must lie in [0, 2^21]";
    else if (a->n_vocab <= 0 || a->n_vocab > 1 << 20) why = "n_vocab must lie in [1, 2^20]";
    else if (a->row_stride < a->n_vocab || a->row_stride > (int64_t)1 << 40) why = "row_stride is smaller than n_vocab";
    else if (a->n_rows > 0 && (!a->logits || !a->u || !a->id)) why = "null logits, u or id";
    else if (!aligned(a->logits, size) || !aligned(a->u, 8) || !aligned(a->temperature, 4) || !aligned(a->top_k, 4) || !aligned(a->top_p, 4) || !aligned(a->min_p, 4) ||
             !aligned(a->id, 4) || !aligned(a->p, 4) || !aligned(a->logprob, 4) || !aligned(a->n_kept, 4)) why = "misaligned pointer";
    if (why) return refuse("ss_sample_rows", why);
    OnDevice on(device);
    launch_sample_rows(*a, (hipStream_t)stream);
    return SS_OK;
    SS_CATCH
}

}  // extern "C"
